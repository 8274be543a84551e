// Paged key-value cache on MI355X (gfx950): block tables and slot maps from request lengths, and the
// norms, rotation and store of new tokens. The attention over the pages is in qtts_paged_attn.hip.
//
// A layer's cache is pages of page_size tokens; block_table[r][i] is the page of request r's tokens
// i * page_size .. , and a token's slot is page * page_size + its place in the page. No counterpart in the
// reference, whose cache is one contiguous block for one stream (megakernel_backbone.py:156-159).
#include "qtts_paged.h"
#include <algorithm>
#include <climits>

namespace qtts {
namespace pg {

// ---- plan ------------------------------------------------------------------------------------
// Request b holds L_b tokens and gets n_b more. With page size P, table width W, F free pages:
//   need_b = ceil((L_b + n_b) / P) - ceil(L_b / P), 0 where the tokens do not fit the table or the arrays
//   granted iff it fits and (need_b = 0 or need_0 + .. + need_b <= F): pages are given in request order,
//   and a request that finds too few ends the giving (those behind it do not overtake it)
//   table[b][ceil(L_b / P) + j] = free_pages[F - 1 - (need_0 + .. + need_{b-1}) - j]
//   token i of b: position L_b + i, slot table[b][(L_b + i) / P] P + (L_b + i) % P, or -1 if not granted
// One workgroup: the prefix sums of tokens and pages over the requests, NT at a time, then the new pages and the
// tokens as flat lists, each element finding its request by a search in LDS. It is bound by latency: the chain is
// lengths -> sums -> free pages -> slots; 256 threads for up to 256 requests, whose sums cross 4 waves and not 16
// (64 requests of one token 4.1 us, 7.1 on 16 waves). Measured: 64 requests 6.1 us a call, of which an empty launch is
// 2 to 3; 400 requests with 60 prompts up to 1500 tokens 10.9 (this kernel 7.2, the tokens 4.0).
constexpr int PT = 1024;

// Inclusive prefix sums of N values over the workgroup of NT threads; total[] receives the sums. `part`: N * NT / 64
// words of LDS.
template <int NT, int N>
__device__ __forceinline__ void block_scan(long long (&x)[N], long long* part, long long (&total)[N]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long long y = __shfl_up(x[k], o, 64);
      if (lane >= o) x[k] += y;
    }
  __syncthreads();                      // the words' readers of an earlier scan are done
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < N; ++k) part[k * (NT / 64) + w] = x[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    long long before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
      const long long p = part[k * (NT / 64) + i];
      before += i < w ? p : 0;
      all += p;
    }
    total[k] = all;
    x[k] += before;
  }
}

// The first i < n with cum[i] > x (cum non-decreasing, x below its last entry).
template <class T>
__device__ __forceinline__ int first_above(const T* cum, int n, T x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

struct PlanArgs {
  int n, width, shift, total;
  long long table_stride;
  const int* new_tokens;
  const int* lengths;
  int* table;
  const int* free_pages;
  int capacity;
  const int* free_count;
  int* slots;
  int* positions;
  int* cu;
  int* kv_lens;
  int* lengths_out;
  int* free_out;
  int* status;
  int fill;              // this launch writes the tokens too
};

__device__ __forceinline__ int slot_of(int page, int pos, int shift) {
  const long long s = ((long long)page << shift) + (pos & ((1 << shift) - 1));
  return page < 0 || s > INT_MAX ? -1 : (int)s;
}

template <int NT>
__global__ void __launch_bounds__(NT) plan_kernel(const PlanArgs g) {
  __shared__ long long part[2 * NT / 64];
  __shared__ long long s_taken[NT];   // pages asked up to and with the request
  __shared__ int s_cu[NT];            // tokens up to and with the request
  __shared__ int s_len[NT], s_have[NT];   // s_have: -1 where the request is refused
  __shared__ long long s_given;
  const int t = threadIdx.x;
  const long long page = 1ll << g.shift, keys = (long long)g.width << g.shift;
  const long long free_n = min(max(*g.free_count, 0), g.capacity);
  long long carry_n = 0, carry_taken = 0;
  if (t == 0) {
    g.cu[0] = 0;
    s_given = 0;
  }
  for (int base = 0; base < g.n; base += NT) {
    const int b = base + t;
    const bool in = b < g.n;
    const long long add = in ? max(g.new_tokens[b], 0) : 0, len = in ? max(g.lengths[b], 0) : 0;
    const bool full = len + add > keys;
    const long long have = (len + page - 1) >> g.shift, want = ((len + add + page - 1) >> g.shift) - have;
    long long x[2] = {add, full ? 0 : want}, sum[2];
    block_scan<NT>(x, part, sum);
    const long long end = carry_n + x[0];
    const bool room = end <= g.total, fits = in && room && !full;
    if (carry_n + sum[0] > g.total) {     // tokens past the arrays: their pages are not asked for
      long long y[1] = {fits ? want : 0}, ysum[1];
      block_scan<NT>(y, part, ysum);
      x[1] = y[0];
      sum[1] = ysum[0];
    }
    const long long need = fits ? want : 0, taken = carry_taken + x[1], sum_n = sum[0], sum_taken = sum[1];
    const bool ok = fits && (need == 0 || taken <= free_n);
    s_taken[t] = taken;
    s_cu[t] = (int)min(end, (long long)INT_MAX);
    s_len[t] = (int)len;
    s_have[t] = ok ? (int)have : -1;
    if (in) {
      g.cu[b + 1] = s_cu[t];
      g.kv_lens[b] = ok ? (int)(len + add) : 0;
      g.lengths_out[b] = (int)(ok ? len + add : len);
      g.status[b] = !room ? 3 : (full ? 2 : (ok ? 0 : 1));
    }
    __syncthreads();
    const int m = min(NT, g.n - base);
    // pages given: the last sum that the free ones cover
    if (t < m && taken <= free_n && (t + 1 == m || s_taken[t + 1] > free_n)) s_given = taken;
    // new pages: page q of the chunk's that the free ones cover, asked by request r
    const long long most = min(sum_taken, free_n - carry_taken);
    for (long long q = t; q < most; q += NT) {
      const int r = first_above(s_taken, m, carry_taken + q);
      if (s_have[r] < 0) continue;
      const long long at = s_have[r] + carry_taken + q - (r ? s_taken[r - 1] : carry_taken);
      g.table[(long long)(base + r) * g.table_stride + at] = g.free_pages[free_n - 1 - carry_taken - q];
    }
    if (g.fill) {
      const int last = (int)min(carry_n + sum_n, (long long)g.total);
      for (int q = (int)min(carry_n, (long long)g.total) + t; q < last; q += NT) {
        const int r = first_above(s_cu, m, q);
        const int pos = s_len[r] + q - (r ? s_cu[r - 1] : (int)carry_n);
        int slot = -1;
        if (s_have[r] >= 0) {
          const int i = pos >> g.shift;
          const long long before = r ? s_taken[r - 1] : carry_taken;
          const int p = i < s_have[r] ? g.table[(long long)(base + r) * g.table_stride + i]
                                      : g.free_pages[free_n - 1 - before - (i - s_have[r])];
          slot = slot_of(p, pos, g.shift);
        }
        g.slots[q] = slot;
        g.positions[q] = pos;
      }
    }
    carry_n += sum_n;
    carry_taken += sum_taken;
    __syncthreads();                    // the chunk's LDS has been read
  }
  if (g.fill)
    for (long long q = min(carry_n, (long long)g.total) + t; q < g.total; q += NT) {
      g.slots[q] = -1;
      g.positions[q] = 0;
    }
  __syncthreads();                      // every thread has read the count
  if (t == 0) *g.free_out = (int)(free_n - s_given);
}

// The tokens of a large plan, from what plan_kernel left: one thread a token over the whole GPU. Its chain is the search,
// a step a load; up to 2048 requests' sums come into LDS first, two loads deep (400 requests: a call 10.9 us, 11.8 when
// it searched them in memory).
constexpr int PL = 2048;
__global__ void __launch_bounds__(256) plan_tokens_kernel(const PlanArgs g) {
  __shared__ int s_cu[PL];
  const int q = blockIdx.x * 256 + threadIdx.x;
  const bool in_lds = g.n <= PL;
  if (in_lds) {
    for (int i = threadIdx.x; i < g.n; i += 256) s_cu[i] = g.cu[i + 1];
    __syncthreads();
  }
  if (q >= g.total) return;
  int slot = -1, pos = 0;
  if (q < (in_lds ? s_cu[g.n - 1] : g.cu[g.n])) {
    const int r = in_lds ? first_above(s_cu, g.n, q) : first_above(g.cu + 1, g.n, q);
    const int i = q - g.cu[r];
    if (g.status[r] == 0) {
      pos = g.lengths_out[r] - (g.cu[r + 1] - g.cu[r]) + i;
      slot = slot_of(g.table[(long long)r * g.table_stride + (pos >> g.shift)], pos, g.shift);
    } else {
      pos = g.lengths_out[r] + i;
    }
  }
  g.slots[q] = slot;
  g.positions[q] = pos;
}

// Pages of the flagged requests back onto the stack of free pages, in request and table order; their
// lengths become 0 and their table entries -1. Entries that hold no page are passed over.
__global__ void __launch_bounds__(PT) release_kernel(int n, int width, int shift, long long table_stride, const int* release,
                                                     int* lengths, int* table, int* free_pages, int capacity,
                                                     int* free_count) {
  __shared__ long long part[PT / 64];
  __shared__ long long s_cum[PT];
  const int t = threadIdx.x;
  const long long page = 1ll << shift;
  long long top = min(max(*free_count, 0), capacity);
  for (int base = 0; base < n; base += PT) {
    const int b = base + t;
    const long long len = b < n && release[b] != 0 ? max(lengths[b], 0) : 0;
    long long x[1] = {min((len + page - 1) >> shift, (long long)width)}, sum[1];
    block_scan<PT>(x, part, sum);
    s_cum[t] = x[0];
    const long long pages = sum[0];
    if (b < n && release[b] != 0) lengths[b] = 0;
    __syncthreads();
    const int m = min(PT, n - base);
    for (long long q0 = 0; q0 < pages; q0 += PT) {
      const long long q = q0 + t;
      int id = -1;
      if (q < pages) {
        const int r = first_above(s_cum, m, q);
        int* e = table + (long long)(base + r) * table_stride + (q - (r ? s_cum[r - 1] : 0));
        id = *e;
        *e = -1;
      }
      long long y[1] = {id >= 0 ? 1 : 0}, kept[1];
      block_scan<PT>(y, part, kept);
      const long long at = top + y[0] - 1;
      if (id >= 0 && at < capacity) free_pages[at] = id;
      top = min(top + kept[0], (long long)capacity);
    }
    __syncthreads();                    // the chunk's LDS has been read
  }
  if (t == 0) *free_count = (int)top;   // (after the scans' barriers: every thread has read the count)
}

// ---- norms, rotation, store ----------------------------------------------------------------
// Per head of q and k: y = x / sqrt(mean(x^2) + eps) * gain, then with the token's table row, d < D / 2:
//   out[d] = y[d] cos[d] - y[d + D/2] sin[d],  out[d + D/2] = y[d + D/2] cos[d] + y[d] sin[d]
// in f32, rounded once to the element type (a query row, or K at the token's slot); V goes to its slot as
// it is. Both halves of a table row hold the same values; the first is read. The work is moving bytes: a
// token's heads in and out once, 16 bytes a lane on each side, D / 16 lanes a head row, so that a wave
// takes 1024 / D rows at a time and the sum of squares stays within D / 16 lanes. Measured: 6001 tokens of 16 / 8 heads of
// 128 in bf16 20.0 us, 5.0 TB/s of the 99.9 MB that it must move (a large copy reaches 4.8); 1777 of 24 / 4 heads of 64
// in fp16 6.4 us; 40 tokens 4.4, the latency of token -> slot and position -> table row -> stores.
struct StoreArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  long long q_token, k_token, v_token, o_token;   // strides in elements
  long long q_head, k_head, v_head, o_head;
  const uint16_t* wq;
  const uint16_t* wk;
  const void* cos_t;
  const void* sin_t;
  const int* pos;
  const int* slots;
  long long pos_stride;                           // between the (t, h, w) rows; 0: one row
  int rows, tokens, hq, hkv, h_end, w_end;        // channels below h_end / w_end take h / w by d % 3
  float eps;
  int parts;                                      // waves a token
  Pages pages;
};

template <class E, bool F32>
__device__ __forceinline__ void table8(const void* t, long long at, float (&f)[8]) {
  if constexpr (F32) {
    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(t) + at);
    const f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
  } else {
    const u32x4 v = ldw(static_cast<const uint16_t*>(t) + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[2 * e] = E::lo(v[e]); f[2 * e + 1] = E::hi(v[e]); }
  }
}

template <class E, int D, bool F32>
__global__ void __launch_bounds__(256) store_kernel(const StoreArgs g) {
  constexpr int LPR = D / 16, RPW = 64 / LPR, H = D / 2;
  const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int tok = (int)(id / g.parts), part = (int)(id % g.parts);
  if (tok >= g.tokens) return;
  const int slot = g.slots[tok];
  if (slot < 0 || (slot >> g.pages.shift) >= g.pages.num_pages) return;
  const int lane = threadIdx.x & 63, d0 = 8 * (lane & (LPR - 1)), sub = lane / LPR;
  const int heads = g.hq + 2 * g.hkv;
  const long long row_at = (long long)(slot >> g.pages.shift) * g.pages.page_stride +
                           (long long)(slot & ((1 << g.pages.shift) - 1)) * g.pages.slot_stride;
  float c[8], s[8];
  auto row = [&](int j) QTTS_PG_INLINE { return (long long)min(max(g.pos[j * g.pos_stride + tok], 0), g.rows - 1) * D + d0; };
  {
    const long long r = row(0);
    table8<E, F32>(g.cos_t, r, c);
    table8<E, F32>(g.sin_t, r, s);
  }
  if (g.pos_stride != 0) {
#pragma unroll
    for (int j = 1; j < 3; ++j) {
      const long long r = row(j);
      float cj[8], sj[8];
      table8<E, F32>(g.cos_t, r, cj);
      table8<E, F32>(g.sin_t, r, sj);
      const int end = j == 1 ? g.h_end : g.w_end;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool take = (d0 + e) % 3 == j && d0 + e < end;
        c[e] = take ? cj[e] : c[e];
        s[e] = take ? sj[e] : s[e];
      }
    }
  }
  for (int h0 = part * RPW; h0 < heads; h0 += g.parts * RPW) {
    const int h = h0 + sub;
    const bool in = h < heads, isq = h < g.hq, isv = h >= g.hq + g.hkv;
    const int hh = isq ? h : (isv ? h - g.hq - g.hkv : h - g.hq);
    const uint16_t* src = isq ? g.q + tok * g.q_token + hh * g.q_head
                              : (isv ? g.v + tok * g.v_token + hh * g.v_head : g.k + tok * g.k_token + hh * g.k_head);
    u32x4 a{}, b{};
    if (in) {
      a = ldw(src + d0);
      b = ldw(src + d0 + H);
    }
    uint16_t* dst = isq ? g.out + tok * g.o_token + hh * g.o_head
                        : const_cast<uint16_t*>(isv ? g.pages.v : g.pages.k) + row_at + (long long)hh * g.pages.head_stride;
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = E::lo(a[e]);
      x[2 * e + 1] = E::hi(a[e]);
      y[2 * e] = E::lo(b[e]);
      y[2 * e + 1] = E::hi(b[e]);
    }
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
    ss += xlane_f<0>(ss);
    ss += xlane_f<1>(ss);
    if constexpr (LPR == 8) ss += xlane_f<2>(ss);
    const uint16_t* gain = isq ? g.wq : g.wk;
    if (!isv) {
      float rs = 1.0f, ga[8], gb[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) ga[e] = gb[e] = 1.0f;
      if (gain != nullptr) {
        rs = 1.0f / sqrtf(ss / (float)D + g.eps);
        table8<E, false>(gain, d0, ga);
        table8<E, false>(gain, d0 + H, gb);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int k = 2 * e + i;
          const float p = x[k] * rs * ga[k], r = y[k] * rs * gb[k];
          lo[i] = p * c[k] - r * s[k];
          hi[i] = r * c[k] + p * s[k];
        }
        a[e] = E::pack(lo[0], lo[1]);
        b[e] = E::pack(hi[0], hi[1]);
      }
    }
    if (in) {
      *reinterpret_cast<u32x4*>(dst + d0) = a;
      *reinterpret_cast<u32x4*>(dst + d0 + H) = b;
    }
  }
}

template <class E, int D>
void launch_store(const StoreArgs& g, bool f32_tables, hipStream_t st) {
  const dim3 grid((unsigned)(((long long)g.tokens * g.parts + 3) / 4));
  if (f32_tables) hipLaunchKernelGGL((store_kernel<E, D, true>), grid, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((store_kernel<E, D, false>), grid, dim3(256), 0, st, g);
}

}  // namespace pg
}  // namespace qtts

using namespace qtts;
using namespace qtts::pg;

extern "C" {

hipError_t qtts_paged_plan(int n_requests, int table_width, long long table_stride, int page_size, int total_tokens,
                           const int* new_tokens, const int* lengths, int* block_table, const int* free_pages,
                           int free_capacity, const int* free_count, int* slots, int* positions, int* cu_tokens,
                           int* kv_lens, int* lengths_out, int* free_count_out, int* status, hipStream_t stream) {
  if (n_requests < 1 || n_requests > (1 << 24) || table_width < 1 || table_stride < table_width || total_tokens < 0 ||
      total_tokens > (1 << 30) || free_capacity < 0)
    return hipErrorInvalidValue;
  if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)) != 0) return hipErrorInvalidValue;
  if ((long long)table_width * page_size > (1ll << 30)) return hipErrorInvalidValue;
  if (new_tokens == nullptr || lengths == nullptr || block_table == nullptr || free_count == nullptr || cu_tokens == nullptr ||
      kv_lens == nullptr || lengths_out == nullptr || free_count_out == nullptr || status == nullptr ||
      (free_capacity > 0 && free_pages == nullptr) || (total_tokens > 0 && (slots == nullptr || positions == nullptr)))
    return hipErrorInvalidValue;
  PlanArgs g{n_requests, table_width, __builtin_ctz((unsigned)page_size), total_tokens, table_stride, new_tokens, lengths,
             block_table, free_pages, free_capacity, free_count, slots, positions, cu_tokens, kv_lens, lengths_out,
             free_count_out, status, 0};
  // the tokens in the same launch while they are two for a thread; past that a second one over the whole GPU (us, one
  // launch : two: 64 requests of one token 3.7 : 4.9, 200 of 10 9.3 : 6.8, 64 of 64 14.3 : 7.1, 60 of 700 113 : 12.8)
  g.fill = total_tokens <= 2 * (n_requests <= 256 ? 256 : PT);
  if (n_requests <= 256) hipLaunchKernelGGL(plan_kernel<256>, dim3(1), dim3(256), 0, stream, g);
  else hipLaunchKernelGGL(plan_kernel<PT>, dim3(1), dim3(PT), 0, stream, g);
  if (!g.fill) hipLaunchKernelGGL(plan_tokens_kernel, dim3((unsigned)((total_tokens + 255) / 256)), dim3(256), 0, stream, g);
  return hipGetLastError();
}

hipError_t qtts_paged_release(int n_requests, int table_width, long long table_stride, int page_size, const int* release,
                              int* lengths, int* block_table, int* free_pages, int free_capacity, int* free_count,
                              hipStream_t stream) {
  if (n_requests < 1 || n_requests > (1 << 24) || table_width < 1 || table_stride < table_width || free_capacity < 1)
    return hipErrorInvalidValue;
  if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1)) != 0) return hipErrorInvalidValue;
  if (release == nullptr || lengths == nullptr || block_table == nullptr || free_pages == nullptr || free_count == nullptr)
    return hipErrorInvalidValue;
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(PT), 0, stream, n_requests, table_width, __builtin_ctz((unsigned)page_size),
                     table_stride, release, lengths, block_table, free_pages, free_capacity, free_count);
  return hipGetLastError();
}

hipError_t qtts_qk_norm_rope_store(const QttsPagedCache* cache, int n_tokens, int num_q_heads, const void* q,
                                   long long q_token_stride, long long q_head_stride, const void* k,
                                   long long k_token_stride, long long k_head_stride, const void* v,
                                   long long v_token_stride, long long v_head_stride, void* q_out,
                                   long long out_token_stride, long long out_head_stride, const void* q_weight,
                                   const void* k_weight, float eps, const void* cos_table, const void* sin_table,
                                   int table_f32, int table_rows, const int* positions, long long position_stride,
                                   int h_channels, int w_channels, const int* slots, hipStream_t stream) {
  if (!cache_ok(cache) || n_tokens < 0 || num_q_heads < 1 || table_rows < 1) return hipErrorInvalidValue;
  if (n_tokens == 0) return hipSuccess;
  if (q == nullptr || k == nullptr || v == nullptr || q_out == nullptr || cos_table == nullptr || sin_table == nullptr ||
      positions == nullptr || slots == nullptr)
    return hipErrorInvalidValue;
  const int half = cache->head_dim / 2;
  if (position_stride < 0 || h_channels < 0 || w_channels < 0 || h_channels > half || w_channels > half || !(eps >= 0.0f))
    return hipErrorInvalidValue;
  const long long strides[] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride,
                               v_token_stride, v_head_stride, out_token_stride, out_head_stride};
  for (long long s : strides)
    if ((s & 7) != 0) return hipErrorInvalidValue;
  const void* aligned[] = {q, k, v, q_out, q_weight, k_weight, cos_table, sin_table};
  for (const void* p : aligned)
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return hipErrorInvalidValue;
  StoreArgs g{};
  g.q = static_cast<const uint16_t*>(q);
  g.k = static_cast<const uint16_t*>(k);
  g.v = static_cast<const uint16_t*>(v);
  g.out = static_cast<uint16_t*>(q_out);
  g.q_token = q_token_stride; g.k_token = k_token_stride; g.v_token = v_token_stride; g.o_token = out_token_stride;
  g.q_head = q_head_stride; g.k_head = k_head_stride; g.v_head = v_head_stride; g.o_head = out_head_stride;
  g.wq = static_cast<const uint16_t*>(q_weight);
  g.wk = static_cast<const uint16_t*>(k_weight);
  g.cos_t = cos_table;
  g.sin_t = sin_table;
  g.pos = positions;
  g.pos_stride = position_stride;
  g.slots = slots;
  g.rows = table_rows;
  g.tokens = n_tokens;
  g.hq = num_q_heads;
  g.hkv = cache->num_kv_heads;
  g.h_end = h_channels;
  g.w_end = w_channels;
  g.eps = eps;
  g.pages = pages_of(cache);
  // a wave a token (its table row read once) from 2048 tokens on, 8 waves a CU; below, a wave for each group of head
  // rows (us, a wave a token : a group, 16 / 8 heads of 128: 40 tokens 4.9 : 3.4, 1024 6.1 : 5.1, 2048 8.5 : 8.4,
  // 3000 11.3 : 12.3, 6001 18.1 : 20.2)
  const int rpw = 1024 / cache->head_dim, groups = (num_q_heads + 2 * cache->num_kv_heads + rpw - 1) / rpw;
  g.parts = n_tokens >= 2048 ? 1 : groups;
  if (((long long)n_tokens * g.parts + 3) / 4 > INT_MAX) return hipErrorInvalidValue;
  if (cache->dtype == QTTS_BF16) {
    if (cache->head_dim == 128) launch_store<Bf16, 128>(g, table_f32 != 0, stream);
    else launch_store<Bf16, 64>(g, table_f32 != 0, stream);
  } else {
    if (cache->head_dim == 128) launch_store<F16, 128>(g, table_f32 != 0, stream);
    else launch_store<F16, 64>(g, table_f32 != 0, stream);
  }
  return hipGetLastError();
}

}  // extern "C"
