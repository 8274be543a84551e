// Attention over a paged key-value cache on MI355X (gfx950): one new token per request (decode), and the
// new tokens of prompts (prefill). The cache's layout is in qtts_paged.hip.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = e^(scale q . k_j - max),  over the keys j that the query sees:
//   j <= p (its position) and, under a window of w keys, j > p - w or j < sinks.
// A query that sees no key (or no finite score) gets zeros. Keys that no query of a workgroup sees are
// never loaded as numbers: their rows come as zeros, so what unused slots hold (NaN included) does not
// matter. A key on a page outside the cache (an entry of -1) is not seen.
#include "qtts_paged.h"
#include <algorithm>
#include <climits>
#include <cmath>

namespace qtts {
namespace pg {

typedef __attribute__((address_space(3))) void lvoid_t;

// Wait until at most N of this wave's vector-memory instructions and none of its LDS reads are in flight.
template <int N>
__device__ __forceinline__ void wait_vm_lds() {
  static_assert(N >= 0 && N <= 63, "vmcnt field");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
}

struct AttnArgs {
  const uint16_t* q;
  uint16_t* out;
  long long q_token, q_head, o_token, o_head;    // strides in elements
  Pages pages;
  const int* table;
  long long table_stride;
  int width;                                     // table entries of a request
  const int* lens;
  const int* cu;                                 // prefill: first token of each request
  int requests, tokens, hq, hkv, group;          // group: query heads of a KV head
  float scale_log2;                              // scale * log2(e)
  int window, sinks;                             // window 0: none
  int merged;                                    // prefill: tiles of all requests in one order (find_tile)
  int splits, blocks;                            // decode: most units of a request, blocks a unit
  float* part;                                   // [requests][hq][splits][D] sums
  float* part_ml;                                // [requests][hq][splits][2] running max and sum
};

// A request's keys, clamped to what its table can hold.
__device__ __forceinline__ int request_len(const AttnArgs& g, int b) {
  const long long most = (long long)g.width << g.pages.shift;
  return (int)min((long long)max(ld_const(g.lens + b), 0), most);
}

// The blocks of KB keys that a range of queries reads: those of the first `sinks` keys, then those from the
// first key of the lowest window (lo) to the last key. t-th block: t < ns ? t : t + skip.
struct Blocks {
  int ns, skip, n;
};
template <int KB>
__device__ __forceinline__ Blocks blocks_of(int lo, int end, int sinks) {
  Blocks r;
  const int first = lo / KB;
  r.ns = (int)min((long long)first, ((long long)min(sinks, lo) + KB - 1) / KB);
  r.skip = first - r.ns;
  r.n = (end + KB - 1) / KB - r.skip;
  return r;
}

// Staged rows: row r of a block at r * 2 D bytes, its 16-byte chunk c at position c ^ swz(r). LDS serves 256 bytes
// a cycle from 64 banks; with this permutation the 16 rows of an operand read (one chunk each) and the 4 rows x
// 64 bytes of a transpose read of the prefill fall on different banks (with c ^ (r & 7) the transpose reads of 4 rows
// fell on the same 64 bytes: two thirds of the LDS cycles were conflicts; now none are). The decode's transpose reads, 8
// rows x 32 bytes, meet two at a time; a permutation for them changed no time (its LDS is busy 15% of the cycles).
template <int D>
__device__ __forceinline__ int swz(int r) {
  if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return ((r << 1) & 4) | ((r >> 1) & 2) | ((r >> 3) & 1);
}

// 16-key pieces of K or V into LDS by DMA. The descriptor begins at the piece's first row and ends with its last.
// A piece whose rows are not all seen asks for the others past the end: they come as zeros. The lane's offsets
// inside a piece are the same for all of them.
template <int D>
struct PieceCopy {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, N = 16 / RPI;   // chunks a row, rows an instruction, instructions
  int off[N];
  __device__ __forceinline__ PieceCopy(int slot_stride, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = RPI * i + lane / CPR;
      off[i] = r * slot_stride * 2 + ((lane % CPR) ^ swz<D>(r)) * 16;
    }
  }
  // the piece's descriptor; `head`: the KV head's channels in page 0
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t piece(const uint16_t* head, const Pages& pg, int page, int key0) const {
    const long long at = (long long)page * pg.page_stride + (long long)((key0 & ((1 << pg.shift) - 1)) * (long long)pg.slot_stride);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(head + at), (short)0, (15 * pg.slot_stride + D) * 2, 0x00020000);
  }
  // the lane's offsets in a piece of which only the rows that seen(key) says are wanted
  template <class Seen>
  __device__ __forceinline__ void some(int key0, int lane, int (&o)[N], Seen&& seen) const {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = seen(key0 + RPI * i + lane / CPR) ? off[i] : 0x7fffff00;
  }
  // ONCE: the bytes are read once and need no place in the caches
  template <bool ONCE = false>
  __device__ __forceinline__ static void one(__amdgpu_buffer_rsrc_t rs, char* dst, int o) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lvoid_t*)dst, 16, o, 0, 0, ONCE ? 2 : 0);
  }
};

// ---- decode --------------------------------------------------------------------------------
// One workgroup of W waves per (request, KV head, up to 16 of its query heads, part of its keys: a unit). Bound by
// reading K and V: every wave streams its own 32-key blocks (blocks w, w + W, .. of the unit) through LDS rows of its
// own, so the loop has no barrier. The next block's K goes out as soon as this one's scores are taken, its V after
// the products, so that 16 KB a wave (128 channels) are in flight nearly always; two workgroups of 4 waves fit a CU,
// and one's beginning and end run under the other's stream.
//   S^T = K Q^T on MFMA 16x16x32 (A: 16 keys x 32 channels from LDS, B: Q^T in registers): lane (g, c) holds
//     head c's scores of keys 4 g + r and 16 + 4 g + r, r < 4; the max over a head's keys is in-lane and two
//     exchanges.
//   O^T += V^T P^T: P^T is the score registers as they are (k-index 8 g + j is key 4 g + j for j < 4 and
//     16 + 4 g + j - 4 above), V^T comes through LDS transpose reads of 4 keys each. P goes in as two 16-bit
//     numbers, the rounded value and the rounded rest, so that its rounding is that of 16 bits or more: the
//     matrix units are idle otherwise.
// Measured (us, and of K and V read): 64 requests of 129 to 4090 keys, 16 / 8 heads of 128, bf16 97 with the join (5.65
// TB/s; reading that much does 7.0), 24 under a window of 1024 20.3 (5.0), 3 of 40000 to 60000 keys, 32 / 4 heads of
// 64, fp16 32 (5.0); one of 700 keys 10.0: two launches and the chain lengths -> table -> K -> scores -> V -> join. What
// the long ones lose against a plain read is each unit's beginning and end, where its 64 KB are not in flight.
// The heads of a group share every K and V byte; a group over 16 is several workgroups. The waves join through
// LDS, the units of a request through part / part_ml and decode_join_kernel, both in key order, so results do not
// depend on timing. A request of one unit writes its output here.
constexpr int DKB = 32;               // keys of a block

// The transpose reads of an MFMA step: 4 keys at LDS addresses a[..] + A and 4 more at b[..] + B, of each channel
// block. In assembly with their wait: before the builtin the compiler waits for every DMA in flight, the next
// block's among them.
template <int A, int B>
__device__ __forceinline__ void tr_read8(const uint32_t (&a)[4], const uint32_t (&b)[4], u32x2 (&lo)[4], u32x2 (&hi)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%c16\n\tds_read_b64_tr_b16 %4, %12 offset:%c17\n\t"
      "ds_read_b64_tr_b16 %1, %9 offset:%c16\n\tds_read_b64_tr_b16 %5, %13 offset:%c17\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%c16\n\tds_read_b64_tr_b16 %6, %14 offset:%c17\n\t"
      "ds_read_b64_tr_b16 %3, %11 offset:%c16\n\tds_read_b64_tr_b16 %7, %15 offset:%c17\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]), "i"(A), "i"(B)
      : "memory");
}
// two MFMA steps (the second S bytes further)
template <int A, int B, int S>
__device__ __forceinline__ void tr_read16(const uint32_t (&a)[4], const uint32_t (&b)[4], u32x2 (&lo)[8], u32x2 (&hi)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16 offset:%c24\n\tds_read_b64_tr_b16 %8, %20 offset:%c25\n\t"
      "ds_read_b64_tr_b16 %1, %17 offset:%c24\n\tds_read_b64_tr_b16 %9, %21 offset:%c25\n\t"
      "ds_read_b64_tr_b16 %2, %18 offset:%c24\n\tds_read_b64_tr_b16 %10, %22 offset:%c25\n\t"
      "ds_read_b64_tr_b16 %3, %19 offset:%c24\n\tds_read_b64_tr_b16 %11, %23 offset:%c25\n\t"
      "ds_read_b64_tr_b16 %4, %16 offset:%c26\n\tds_read_b64_tr_b16 %12, %20 offset:%c27\n\t"
      "ds_read_b64_tr_b16 %5, %17 offset:%c26\n\tds_read_b64_tr_b16 %13, %21 offset:%c27\n\t"
      "ds_read_b64_tr_b16 %6, %18 offset:%c26\n\tds_read_b64_tr_b16 %14, %22 offset:%c27\n\t"
      "ds_read_b64_tr_b16 %7, %19 offset:%c26\n\tds_read_b64_tr_b16 %15, %23 offset:%c27\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(lo[4]), "=&v"(lo[5]), "=&v"(lo[6]), "=&v"(lo[7]),
        "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3]), "=&v"(hi[4]), "=&v"(hi[5]), "=&v"(hi[6]), "=&v"(hi[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]), "i"(A), "i"(B), "i"(A + S), "i"(B + S)
      : "memory");
}
template <class E, int D, int W>
__global__ void __launch_bounds__(64 * W, 2) decode_kernel(const AttnArgs g) {
  constexpr int BLK = DKB * D * 2;               // bytes of a K or V block
  constexpr int MB = D / 16, KS = D / 32;        // 16-channel blocks of O^T, MFMA steps of a score
  constexpr int NL = BLK / 1024;                 // DMA instructions of a K or V block
  __shared__ __attribute__((aligned(1024))) char smem[W * 2 * BLK + (2 * W + 2) * 16 * 4];   // (K, V) a wave; (m, l) of the join
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int c = lane & 15, gr = lane >> 4;
  int id = blockIdx.x;
  const int kvh = id % g.hkv; id /= g.hkv;
  const int unit = id % g.splits; id /= g.splits;
  const int tiles = (g.group + 15) / 16, tile = id % tiles, b = id / tiles;
  const int head0 = kvh * g.group + 16 * tile, nh = min(16, g.group - 16 * tile);

  const int len = request_len(g, b);
  const int lo = g.window > 0 ? max(len - g.window, 0) : 0;
  const Blocks bl = blocks_of<DKB>(lo, len, g.sinks);
  // a unit is g.blocks blocks, or more where the request is longer than the caller said
  const int per = max(g.blocks, (bl.n + g.splits - 1) / g.splits);
  const int units = max(1, (bl.n + per - 1) / per);
  if (unit >= units) return;
  const int t1 = min(bl.n, (unit + 1) * per), t0 = unit * per + w;
  const int nt = t0 < t1 ? (t1 - t0 + W - 1) / W : 0;   // this wave's blocks

  // Q^T: head c, channels 32 s + 8 gr ..
  u32x4 q[KS];
  const uint16_t* qp = g.q + (long long)b * g.q_token + (long long)(head0 + min(c, nh - 1)) * g.q_head + 8 * gr;
#pragma unroll
  for (int s = 0; s < KS; ++s) q[s] = ldw(qp + 32 * s);

  char* const buf = smem + w * 2 * BLK;
  const int* row = g.table + (long long)b * g.table_stride;
  auto key_of = [&](int i) QTTS_PG_INLINE { const int t = t0 + W * i; return (t < bl.ns ? t : t + bl.skip) * DKB; };
  // the table entries of a block's two pieces, piece lane & 1 a lane, loaded a block before they are used
  struct Entries {
    int e;
    uint32_t in;                                 // pieces that have keys, as bits
  };
  auto entries = [&](int i) QTTS_PG_INLINE {
    const int key = key_of(i) + 16 * (lane & 1);
    const bool in = (i < nt) & (key < len);
    return Entries{*gmem(row + (in ? key >> g.pages.shift : 0)), (uint32_t)__builtin_amdgcn_ballot_w64(in) & 3u};
  };
  // a block as it is copied: pages of its pieces (bits of `has`), and the lane's offsets where only a part is seen
  const PieceCopy<D> copy(g.pages.slot_stride, lane);
  const uint16_t* const k_head = g.pages.k + (long long)kvh * g.pages.head_stride;
  const uint16_t* const v_head = g.pages.v + (long long)kvh * g.pages.head_stride;
  struct Block {
    int key0, page[2];
    uint32_t has;
    bool whole;
  };
  auto block = [&](const Entries& x, int i) QTTS_PG_INLINE {
    Block r;
    r.key0 = key_of(i);
    r.has = (uint32_t)__builtin_amdgcn_ballot_w64((unsigned)x.e < (unsigned)g.pages.num_pages) & x.in;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int page = __builtin_amdgcn_readlane(x.e, u);
      r.page[u] = (r.has >> u) & 1 ? page : 0;
    }
    r.whole = (r.has == 3u) & (r.key0 + DKB <= len) & ((r.key0 >= lo) | (r.key0 + DKB <= g.sinks));
    return r;
  };
  auto sees = [&](const Block& r, int key, int u) QTTS_PG_INLINE {
    return (((r.has >> u) & 1) != 0) & (key < len) & ((key >= lo) | (key < g.sinks));
  };
  auto issue = [&](const Block& r, const uint16_t* head, char* dst) QTTS_PG_INLINE {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const auto rs = copy.piece(head, g.pages, r.page[u], r.key0 + 16 * u);
      int off[copy.N];
#pragma unroll
      for (int j = 0; j < copy.N; ++j) off[j] = copy.off[j];
      if (!r.whole) copy.some(r.key0 + 16 * u, lane, off, [&](int key) QTTS_PG_INLINE { return sees(r, key, u); });
#pragma unroll
      for (int j = 0; j < copy.N; ++j) copy.template one<true>(rs, dst + u * 16 * D * 2 + j * 1024, off[j]);
    }
  };

  const float SL = g.scale_log2;
  float m = -INFINITY, l = 0.0f;
  f32x4 o[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) o[mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // transpose reads of V: row 4 gr + (c >> 2), chunk 2 mb + ((c & 3) >> 1), 8 bytes at 8 (c & 1)
  const int vrow = 4 * gr + (c >> 2);
  uint32_t va[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
    va[mb] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)buf + BLK + vrow * D * 2 +
             ((2 * mb + ((c & 3) >> 1)) ^ swz<D>(vrow)) * 16 + 8 * (c & 1);

  if (nt > 0) {
    Entries ahead = entries(1);
    Block now = block(entries(0), 0);
    issue(now, k_head, buf);
    issue(now, v_head, buf + BLK);
#pragma unroll 1
    for (int i = 0; i < nt; ++i) {
      const Block next = block(ahead, i + 1);
      ahead = entries(i + 2);
      wait_vm_lds<NL + 1>();                     // K is here: V's copies and the entries may be under way
      asm volatile("" ::: "memory");
      f32x4 sc[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const u32x4 k = *reinterpret_cast<const u32x4*>(buf + (16 * u + c) * D * 2 + ((4 * s + gr) ^ swz<D>(c)) * 16);
          sc[u] = E::mma16(k, q[s], sc[u]);
        }
      }
      asm volatile("" : "+v"(sc[0]), "+v"(sc[1]) :: "memory");   // K has been read
      if (i + 1 < nt) issue(next, k_head, buf);
      if (!now.whole) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[u][r] = sees(now, now.key0 + 16 * u + 4 * gr + r, u) ? sc[u][r] : -INFINITY;
      }
      float bm = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                       fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
      bm = fmaxf(bm, xlane_f<4>(bm));
      bm = fmaxf(bm, xlane_f<5>(bm));
      if (__builtin_amdgcn_ballot_w64(bm > m) != 0ull) {
        const float mn = fmaxf(m, bm);
        if (__builtin_amdgcn_ballot_w64(m > -INFINITY) != 0ull) {   // (else the sums are zeros)
          const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * SL);
          l *= al;
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[mb][r] *= al;
        }
        m = mn;
      }
      const float nm = m == -INFINITY ? 0.0f : -m * SL;
      u32x4 ph, pl;
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[u][2 * h], SL, nm)), e1 = __builtin_amdgcn_exp2f(fmaf(sc[u][2 * h + 1], SL, nm));
          sum += e0 + e1;
          const uint32_t p = E::pack(e0, e1);
          ph[2 * u + h] = p;
          pl[2 * u + h] = E::pack(e0 - E::lo(p), e1 - E::hi(p));
        }
      l += sum;
      if (i + 1 < nt) wait_vm_lds<NL + 1>();     // V is here: the next K's copies and the entries may be under way
      else wait_vm_lds<1>();
      auto pv = [&](int half, const u32x2 (&a)[4], const u32x2 (&bq)[4]) QTTS_PG_INLINE {
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          const u32x4 v = {a[mb][0], a[mb][1], bq[mb][0], bq[mb][1]};
          o[4 * half + mb] = E::mma16(v, ph, o[4 * half + mb]);
          o[4 * half + mb] = E::mma16(v, pl, o[4 * half + mb]);
        }
      };
      u32x2 a[4], bq[4];
      tr_read8<0, 16 * D * 2>(va, va, a, bq);
      if constexpr (D == 128) {
        uint32_t vb[4];
        u32x2 a2[4], bq2[4];
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) vb[mb] = va[mb] ^ 128;   // channels 64 ..
        tr_read8<0, 16 * D * 2>(vb, vb, a2, bq2);
        if (i + 1 < nt) issue(next, v_head, buf + BLK);
        pv(0, a, bq);
        pv(1, a2, bq2);
      } else {
        if (i + 1 < nt) issue(next, v_head, buf + BLK);
        pv(0, a, bq);
      }
      now = next;
    }
  }
  // A seen v_j that is infinite makes its channel's sum infinite, but 0 or a negative rest times it a NaN. Sums that are
  // not finite are taken again in 32 bits, key by key (a sum of weights that is NaN makes NaN of them anyway). The rests
  // in sums of their own, dropped there, were 3% slower.
  l += xlane_f<4>(l);
  l += xlane_f<5>(l);
  float odd = 0.0f;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int r = 0; r < 4; ++r) odd = fmaf(o[mb][r], 0.0f, odd);
  if (__builtin_amdgcn_ballot_w64((odd != 0.0f) & (l == l)) != 0ull) {
    f32x4 again[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) again[mb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float nm = m == -INFINITY ? 0.0f : -m * SL;
#pragma unroll 1
    for (int i = 0; i < nt; ++i) {
      const Block x = block(entries(i), i);
#pragma unroll 1
      for (int j = 0; j < DKB; ++j) {
        const int key = x.key0 + j, u = j >> 4;
        if (!sees(x, key, u)) continue;
        const long long at = (long long)(u ? x.page[1] : x.page[0]) * g.pages.page_stride +
                             (long long)(key & ((1 << g.pages.shift) - 1)) * g.pages.slot_stride;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x4 kk = ldw(k_head + at + 32 * k + 8 * gr);
#pragma unroll
          for (int h = 0; h < 4; ++h) s = fmaf(E::lo(q[k][h]), E::lo(kk[h]), fmaf(E::hi(q[k][h]), E::hi(kk[h]), s));
        }
        s += xlane_f<4>(s);
        s += xlane_f<5>(s);
        const float p = __builtin_amdgcn_exp2f(fmaf(s, SL, nm));
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const u32x2 v = *gmem(reinterpret_cast<const u32x2*>(v_head + at + 16 * mb + 4 * gr));
          again[mb][0] = fmaf(p, E::lo(v[0]), again[mb][0]);
          again[mb][1] = fmaf(p, E::hi(v[0]), again[mb][1]);
          again[mb][2] = fmaf(p, E::lo(v[1]), again[mb][2]);
          again[mb][3] = fmaf(p, E::hi(v[1]), again[mb][3]);
        }
      }
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[mb][r] = (__float_as_uint(o[mb][r]) & 0x7fffffffu) < 0x7f800000u ? o[mb][r] : again[mb][r];
  }

  // join the waves: M = max m_w, L = sum l_w e^(m_w - M), O = sum O_w e^(m_w - M)
  static_assert(D * 16 * 4 <= 2 * BLK, "the join's sums");
  wait_vm_lds<0>();
  __syncthreads();                               // every buffer is dead
  float* sml = reinterpret_cast<float*>(smem + W * 2 * BLK);
  if (gr == 0) {
    sml[(2 * w) * 16 + c] = m;
    sml[(2 * w + 1) * 16 + c] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.0f;
#pragma unroll
  for (int v = 0; v < W; ++v) M = fmaxf(M, sml[2 * v * 16 + c]);
#pragma unroll
  for (int v = 0; v < W; ++v) {
    const float mv = sml[2 * v * 16 + c];
    L += mv == -INFINITY ? sml[(2 * v + 1) * 16 + c] : sml[(2 * v + 1) * 16 + c] * __builtin_amdgcn_exp2f((mv - M) * SL);
  }
  const float sw = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * SL);
  float* so = reinterpret_cast<float*>(smem);    // [wave][head][channel]
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = o[mb][r] * sw;
    *reinterpret_cast<f32x4*>(so + (w * 16 + c) * D + 16 * mb + 4 * gr) = x;
  }
  if (w == 0 && gr == 0) {
    sml[W * 2 * 16 + c] = M;
    sml[W * 2 * 16 + 16 + c] = L;
  }
  __syncthreads();
  const bool whole = units == 1;
  for (int e = threadIdx.x; e < nh * D / 4; e += 64 * W) {
    const int h = e / (D / 4), d = 4 * (e % (D / 4));
    f32x4 x = *reinterpret_cast<const f32x4*>(so + h * D + d);
#pragma unroll
    for (int v = 1; v < W; ++v) x += *reinterpret_cast<const f32x4*>(so + (v * 16 + h) * D + d);
    if (whole) {
      const float Lh = sml[W * 2 * 16 + 16 + h];
      const float rl = Lh == 0.0f ? 0.0f : 1.0f / Lh;
      u32x2 p;
      p[0] = E::pack(x[0] * rl, x[1] * rl);
      p[1] = E::pack(x[2] * rl, x[3] * rl);
      *reinterpret_cast<u32x2*>(g.out + (long long)b * g.o_token + (long long)(head0 + h) * g.o_head + d) = p;
    } else {
      const long long at = ((long long)b * g.hq + head0 + h) * g.splits + unit;
      *reinterpret_cast<f32x4*>(g.part + at * D + d) = x;
      if (d == 0) {
        g.part_ml[2 * at] = sml[W * 2 * 16 + h];
        g.part_ml[2 * at + 1] = sml[W * 2 * 16 + 16 + h];
      }
    }
  }
}

// The units of a request's head joined (3 to 5 us, a dependent launch): one workgroup per (request, query head), its
// D / 4 lanes a unit taking 4 channels each and its groups of lanes units u, u + groups, ..; the groups' sums add
// through LDS in order. Loads do not wait for the request's length (what a unit past its last has in its place is
// passed over), so the chain is one read, not three.
template <class E, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(const AttnArgs g) {
  constexpr int LU = D / 4, GR = 256 / LU, AT = 4;   // lanes a unit, groups, units of a group read at once
  __shared__ float sums[GR][D + 4];
  const int t = threadIdx.x, gq = t / LU, d = 4 * (t % LU);
  const int b = blockIdx.x / g.hq, h = blockIdx.x % g.hq;
  const long long id = blockIdx.x;
  const float* ml = g.part_ml + 2 * id * g.splits;
  const float* po = g.part + id * g.splits * D + d;
  f32x4 x[AT];
  float mu[AT], lu[AT];
  auto read = [&](int u0) QTTS_PG_INLINE {
#pragma unroll
    for (int k = 0; k < AT; ++k) {
      const int u = min(u0 + gq + GR * k, g.splits - 1);
      x[k] = *reinterpret_cast<const f32x4*>(po + (long long)u * D);
      mu[k] = ml[2 * u];
      lu[k] = ml[2 * u + 1];
    }
  };
  read(0);
  const int len = request_len(g, b);
  const Blocks bl = blocks_of<DKB>(g.window > 0 ? max(len - g.window, 0) : 0, len, g.sinks);
  const int per = max(g.blocks, (bl.n + g.splits - 1) / g.splits), units = (bl.n + per - 1) / per;
  if (units <= 1) return;
  float M = -INFINITY, L = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  auto take = [&](float m2, float l2, const f32x4& x2) QTTS_PG_INLINE {
    const float mn = fmaxf(M, m2);
    const float a = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((M - mn) * g.scale_log2);   // (-inf: sums are 0, or NaN)
    const float e = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m2 - mn) * g.scale_log2);
    L = L * a + l2 * e;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * a + x2[i] * e;
    M = mn;
  };
  for (int u0 = 0;;) {
#pragma unroll
    for (int k = 0; k < AT; ++k)
      if (u0 + gq + GR * k < units) take(mu[k], lu[k], x[k]);
    u0 += GR * AT;
    if (u0 >= units) break;
    read(u0);
  }
  *reinterpret_cast<f32x4*>(&sums[gq][d]) = o;
  if (d == 0) {
    sums[gq][D] = M;
    sums[gq][D + 1] = L;
  }
  __syncthreads();
  if (gq != 0) return;
#pragma unroll
  for (int k = 1; k < GR; ++k) take(sums[k][D], sums[k][D + 1], *reinterpret_cast<const f32x4*>(&sums[k][d]));
  const float rl = L == 0.0f ? 0.0f : 1.0f / L;
  u32x2 p;
  p[0] = E::pack(o[0] * rl, o[1] * rl);
  p[1] = E::pack(o[2] * rl, o[3] * rl);
  *reinterpret_cast<u32x2*>(g.out + (long long)b * g.o_token + (long long)h * g.o_head + d) = p;
}

// ---- prefill -------------------------------------------------------------------------------
// The query rows of a request and KV head are its tokens times the group's heads, row r = token r / group,
// head r % group, so that any group size fills the tiles. One workgroup of 8 waves takes a tile of 32 NR rows
// and walks the keys that any of them sees 128 at a time: wave (ks, wr) takes rows 32 wr .. and the key
// block ks of each step (NS blocks of 128 / NS keys, NR = 8 / NS). K and V of a step come by DMA, a 16-key piece
// a wave, into one of two LDS buffers, one step ahead. The key splits halve (NS = 2) or quarter (NS = 4) the
// chain of steps of a tile, which is what a causal launch waits for: its last tiles see all the keys.
//   S^T = K Q^T on MFMA 32x32x16 (A: 32 keys from LDS, B: the rows in registers): lane (hf, c) holds row c's
//     scores of keys 8 (r >> 2) + 4 hf + (r & 3), so a row's max and sum are in-lane and one exchange.
//   O^T += V^T P^T with the score registers as P^T (k-index 8 hf + j of step kk is key 16 kk + 8 (j >> 2) +
//     4 hf + (j & 3)) and V^T by LDS transpose reads. P is rounded to the element type, as V is (in two
//     parts, as in decode, it would cost half as many matrix products again); its sum is of the unrounded values in f32.
// Bound by the issue of matrix products (34% of the SIMDs' cycles) and vector instructions (40%), with two waves a SIMD to
// run one under the other; with 64 channels the exponentials and masks take 65%. Measured: a prompt of 4096 tokens, 16 / 8
// heads of 128, bf16 82 us (840 TFLOP/s; a large library product does 1208), 3 of 1111 to 3500 under a window of 777,
// 32 / 4 heads of 64, fp16 86 (580), 12 of 5 to 300 tokens after up to 900 25.7, two rounds of tiles.
// The running max moves only when a row's block max passes it by more than a factor 2^8 of the weights. The
// splits of a row join through LDS in key order.
// A weight that is masked is 0, but 0 times an infinite or NaN v_j is NaN, and a key may be hidden from one
// row of a tile and seen by another: rows that end with a number that is not finite are summed again over
// the keys that they see, one by one (exact_row); not those whose sum of weights is NaN: a score that they see is.
constexpr int PWV = 8;                // waves

// Row `r` of (request b, KV head kvh) again, key by key: the wave's lanes take D / 64 channels each.
template <class E, int D>
__device__ __forceinline__ void exact_row(const AttnArgs& g, int b, int kvh, int token, int head, int pos) {
  constexpr int DL = D / 64;
  const int lane = threadIdx.x & 63;
  const int* row = g.table + (long long)b * g.table_stride;
  auto at2 = [&](const uint16_t* p) QTTS_PG_INLINE {
    float2 f;
    if constexpr (DL == 2) {
      const uint32_t v = *gmem(reinterpret_cast<const uint32_t*>(p + 2 * lane));
      f.x = E::lo(v);
      f.y = E::hi(v);
    } else {
      f.x = E::lo((uint32_t)*gmem(p + lane));
      f.y = 0.0f;
    }
    return f;
  };
  const float2 q = at2(g.q + (long long)token * g.q_token + (long long)head * g.q_head);
  const int lo = g.window > 0 ? max(pos - g.window + 1, 0) : 0;
  float m = -INFINITY, l = 0.0f, x = 0.0f, y = 0.0f;
  for (int key = 0; key <= pos; ++key) {
    if (key < lo && key >= g.sinks) {
      key = lo - 1;
      continue;
    }
    const int page = *gmem(row + (key >> g.pages.shift));
    if ((unsigned)page >= (unsigned)g.pages.num_pages) continue;
    const long long at = (long long)page * g.pages.page_stride + (long long)kvh * g.pages.head_stride +
                         (long long)(key & ((1 << g.pages.shift) - 1)) * g.pages.slot_stride;
    const float2 k = at2(g.pages.k + at), v = at2(g.pages.v + at);
    const float s = group_sum<64>(q.x * k.x + q.y * k.y);
    if (s == -INFINITY) continue;
    const float mn = fmaxf(m, s);
    const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * g.scale_log2);
    const float e = __builtin_amdgcn_exp2f((s - mn) * g.scale_log2);
    l = (m == -INFINITY ? l : l * al) + e;       // (m is -inf still after a NaN score: keep it)
    x = (m == -INFINITY ? x : x * al) + e * v.x;
    y = (m == -INFINITY ? y : y * al) + e * v.y;
    m = mn;
  }
  const float rl = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* op = g.out + (long long)token * g.o_token + (long long)head * g.o_head + DL * lane;
  if constexpr (DL == 2) *reinterpret_cast<uint32_t*>(op) = E::pack(x * rl, y * rl);
  else *op = (uint16_t)E::pack(x * rl, 0.0f);
}

// Tile number `back` of PM rows, the longest keys first: its request and its place in it; request -1 past the last
// one. Either request by request from the last, every lane taking a request, 64 at a time; or (merged, up to 64
// requests) over all of them: a request's tiles lie at the places ceil(len group / PM) and downwards, one each, and the
// place of number `back` is found by halving on how many tiles lie past it.
struct TilePlace {
  int b, tile, first, n;              // request, tile in it, first token, tokens
};
template <int PM>
__device__ __forceinline__ int tiles_of(const AttnArgs& g, int b, int* first, int* n) {
  int f = 0, k = 0;
  if (b < g.requests) {
    f = min(max(g.cu[b], 0), g.tokens);
    k = max(min(max(g.cu[b + 1], 0), g.tokens) - f, 0);
  }
  *first = f;
  *n = k;
  return (int)(((long long)k * g.group + PM - 1) / PM);
}
template <int PM>
__device__ __forceinline__ TilePlace find_tile(const AttnArgs& g, int back) {
  const int lane = threadIdx.x & 63;
  if (g.merged) {
    int first, n;
    const int own = tiles_of<PM>(g, lane, &first, &n);
    const int len = request_len(g, min(lane, g.requests - 1));
    const int top = (int)min(((long long)len * g.group + PM - 1) / PM, 1ll << 29);   // place of the request's last tile
    auto most = [](int x) QTTS_PG_INLINE {
      x = max(x, (int)xlane<0>((uint32_t)x));
      x = max(x, (int)xlane<1>((uint32_t)x));
      x = max(x, (int)xlane<2>((uint32_t)x));
      x = max(x, (int)xlane<3>((uint32_t)x));
      x = max(x, (int)xlane<4>((uint32_t)x));
      return __builtin_amdgcn_readfirstlane(max(x, (int)xlane<5>((uint32_t)x)));
    };
    auto behind = [&](int place) QTTS_PG_INLINE {        // tiles of all requests past a place
      int x = min(max(top - place, 0), own);
      x += (int)xlane<0>((uint32_t)x);
      x += (int)xlane<1>((uint32_t)x);
      x += (int)xlane<2>((uint32_t)x);
      x += (int)xlane<3>((uint32_t)x);
      x += (int)xlane<4>((uint32_t)x);
      return __builtin_amdgcn_readfirstlane(x + (int)xlane<5>((uint32_t)x));
    };
    int lo = -most(own > 0 ? own - top : -(1 << 30)), up = most(own > 0 ? top : -(1 << 30));   // lo: before every tile
    if (up < lo || back >= behind(lo)) return TilePlace{-1, 0, 0, 0};
    while (lo < up) {                                    // the least place with at most `back` tiles past it
      const int mid = lo + ((up - lo) >> 1);
      if (behind(mid) <= back) up = mid;
      else lo = mid + 1;
    }
    const uint64_t here = __builtin_amdgcn_ballot_w64((top >= lo) & (top - lo < own));
    const int rank = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(here >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)here, 0u));
    const int src = __builtin_ctzll(here & __builtin_amdgcn_ballot_w64(rank == back - behind(lo)));
    TilePlace p;
    p.b = src;
    p.tile = __builtin_amdgcn_readlane(own, src) - 1 - (__builtin_amdgcn_readlane(top, src) - lo);
    p.first = __builtin_amdgcn_readlane(first, src);
    p.n = __builtin_amdgcn_readlane(n, src);
    return p;
  }
  for (int b0 = (g.requests - 1) & ~63; b0 >= 0; b0 -= 64) {
    int first, n;
    const int own = tiles_of<PM>(g, b0 + lane, &first, &n);
    int after = own;                  // tiles of the lane's request and those behind it
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_down(after, o, 64);
      if (lane + o < 64) after += y;
    }
    const int all = __builtin_amdgcn_readfirstlane(after);
    if (back < all) {
      const int src = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(after > back));   // the last such lane
      TilePlace p;
      p.b = b0 + src;
      p.tile = __builtin_amdgcn_readlane(after, src) - 1 - back;   // those of later requests come first
      p.first = __builtin_amdgcn_readlane(first, src);
      p.n = __builtin_amdgcn_readlane(n, src);
      return p;
    }
    back -= all;
  }
  return TilePlace{-1, 0, 0, 0};
}

template <class E, int D, int NS>
__global__ void __launch_bounds__(64 * PWV, D == 128 ? 2 : 4) prefill_kernel(const AttnArgs g) {
  constexpr int NR = PWV / NS, PM = 32 * NR, KB = NS == 4 ? 32 : 64;   // row groups, rows of a tile, keys of a wave's block
  constexpr int STEP = NS * KB, NP = STEP / 16;                        // keys of a step, its pieces (8, or 4)
  constexpr int NU = KB / 32, PPB = KB / 16;                           // 32-key score blocks, pieces of a block
  constexpr int BUF = STEP * D * 2;                                    // bytes of a step's K or V
  constexpr int PAIR = NP / 4;                                         // pieces that a wave copies: K and V, or one of them
  constexpr int MB = D / 32, KS = D / 16;
  constexpr int JOIN = PWV * D * 32 * 4;                               // bytes of the join's sums (one split needs none)
  constexpr int ROOM = NS > 1 && JOIN > 4 * BUF ? JOIN : 4 * BUF;
  __shared__ __attribute__((aligned(1024))) char smem[ROOM + PWV * 2 * 32 * 4];   // (K, V) x 2 buffers; (m, l) of the join
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int hf = lane >> 5, c = lane & 31, wr = w % NR, ks = w / NR;
  const int kvh = blockIdx.x % g.hkv;
  const TilePlace at = find_tile<PM>(g, blockIdx.x / g.hkv);
  if (at.b < 0) return;
  const int len = request_len(g, at.b), p0 = len - at.n;   // (p0 < 0: more tokens than keys; those before key 0 see none)
  const int rows = at.n * g.group;                          // (the host bounds tokens * group)
  const int r0 = at.tile * PM, i0 = r0 / g.group, i1 = (min(r0 + PM, rows) - 1) / g.group;
  const int end = max(p0 + i1 + 1, 0);                      // keys that the tile's last token sees
  const int lo = g.window > 0 ? max(p0 + i0 + 1 - g.window, 0) : 0;
  const Blocks bl = blocks_of<KB>(lo, end, g.sinks);
  const int steps = (bl.n + NS - 1) / NS;

  // this lane's row, and the first and last position of the wave's
  const int r = min(r0 + 32 * wr + c, rows - 1), ti = r / g.group, head = kvh * g.group + (r - ti * g.group);
  const bool stored = r0 + 32 * wr + c < rows;
  const int pos = p0 + ti;
  const int wlo = p0 + min(r0 + 32 * wr, rows - 1) / g.group, whi = p0 + min(r0 + 32 * wr + 31, rows - 1) / g.group;
  const int first_key = g.window > 0 ? pos - g.window + 1 : 0;   // of the row's window

  u32x4 q[KS];
  const uint16_t* qp = g.q + (long long)(at.first + ti) * g.q_token + (long long)head * g.q_head + 8 * hf;
#pragma unroll
  for (int s = 0; s < KS; ++s) q[s] = ldw(qp + 16 * s);

  const int* row = g.table + (long long)at.b * g.table_stride;
  auto key_of = [&](int t) QTTS_PG_INLINE { return (t < bl.ns ? t : t + bl.skip) * KB; };   // first key of block t
  // The table entries of a step's pieces, piece lane & (NP - 1) a lane, loaded a step before they are used; in: the pieces
  // that have keys, as bits.
  struct Entries {
    int e;
    uint32_t in;
  };
  auto entries = [&](int i) QTTS_PG_INLINE {
    const int t = i * NS + (lane & (NP - 1)) / PPB, key = key_of(t) + 16 * (lane & (PPB - 1));
    const bool in = (t < bl.n) & (key < end);
    return Entries{*gmem(row + (in ? key >> g.pages.shift : 0)), (uint32_t)__builtin_amdgcn_ballot_w64(in) & ((1u << NP) - 1)};
  };
  // pieces with a page of the cache, as bits; and the page of this wave's (-1: none)
  auto found = [&](const Entries& x) QTTS_PG_INLINE {
    return (uint32_t)__builtin_amdgcn_ballot_w64((unsigned)x.e < (unsigned)g.pages.num_pages) & x.in;
  };
  auto own = [&](const Entries& x, uint32_t has) QTTS_PG_INLINE {
    const int page = __builtin_amdgcn_readlane(x.e, w % NP), none = (int)((has >> (w % NP)) & 1) - 1;   // -1: none
    return page | none;
  };
  // steps whose wave's block is seen whole by all its rows, and whose copies (of the next step's K
  // and V) are whole: no mask, no partial piece
  int fs, fe;
  {
    const int see0 = g.window > 0 ? max(bl.ns, (max(whi - g.window + 1, 0) + KB - 1) / KB - bl.skip) : 0;
    const int see1 = (max(wlo, -1) + 1) / KB - bl.skip, copy1 = end / KB - bl.skip;
    const int copy0 = g.window > 0 ? max(bl.ns, (lo + KB - 1) / KB - bl.skip) : 0;
    fs = (max(max(see0, copy0) - ks, 0) + NS - 1) / NS;
    fe = (max(min(see1, copy1 - NS) - ks, 0) + NS - 1) / NS;
  }
  const PieceCopy<D> copy(g.pages.slot_stride, lane);
  const uint16_t* const k_head = g.pages.k + (long long)kvh * g.pages.head_stride;
  const uint16_t* const v_head = g.pages.v + (long long)kvh * g.pages.head_stride;
  // The copy of a piece of step i by wave w, of K into half 0 of its buffer or of V into half 1: piece w of both, or, of
  // a step of 4 pieces, piece w % 4 of K (waves 0 .. 3) or V.
  struct Piece {
    __amdgpu_buffer_rsrc_t rs;
    char* dst;
    int key0, page;
    int off[PieceCopy<D>::N];
  };
  auto piece = [&](const uint16_t* head, int page, int i, int half) QTTS_PG_INLINE {
    Piece p;
    p.page = page;
    p.key0 = key_of(i * NS + w % NP / PPB) + 16 * (w % PPB);
    p.rs = copy.piece(head, g.pages, max(page, 0), p.key0);
    p.dst = smem + (i & 1) * 2 * BUF + half * BUF + (w % NP) * 16 * D * 2;
#pragma unroll
    for (int j = 0; j < copy.N; ++j) p.off[j] = copy.off[j];
    return p;
  };
  auto part = [&](Piece& p) QTTS_PG_INLINE {             // only the rows that are seen
    copy.some(p.key0, lane, p.off,
              [&](int key) QTTS_PG_INLINE { return (p.page >= 0) & (key < end) & ((key >= lo) | (key < g.sinks)); });
  };
  auto issue = [&](Piece p) QTTS_PG_INLINE {
    part(p);
#pragma unroll
    for (int j = 0; j < copy.N; ++j) copy.one(p.rs, p.dst + j * 1024, p.off[j]);
  };

  const float SL = g.scale_log2;
  float m = -INFINITY, l = 0.0f;
  f32x16 o[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[mb][e] = 0.0f;
  // transpose reads of V: row vrow, chunk 4 mb + vch, 8 bytes at 8 (gi & 1)
  const int gi = lane & 15, gg = lane >> 4;
  const int vrow = 4 * (gg >> 1) + (gi >> 2), vch = 2 * (gg & 1) + ((gi & 3) >> 1);
  uint32_t vaddr[4];
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
    vaddr[mb] = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + BUF + (ks * KB + vrow) * D * 2 +
                ((4 * (mb % MB) + vch) ^ swz<D>(vrow)) * 16 + 8 * (gi & 1);

  float sc[16 * NU];
  u32x4 p[2 * NU];
  // K fragments of half of the channel steps, of the block's NU score blocks: h = 0, 1
  u32x4 kf[2][NU][KS / 2];
  auto read_k = [&](int i, int h) QTTS_PG_INLINE {
    const char* K = smem + (i & 1) * 2 * BUF + (ks * KB + c) * D * 2;
#pragma unroll
    for (int s = 0; s < KS / 2; ++s)
#pragma unroll
      for (int u = 0; u < NU; ++u)
        kf[h][u][s] = *reinterpret_cast<const u32x4*>(K + 32 * u * D * 2 + ((KS * h + 2 * s + hf) ^ swz<D>(c)) * 16);
  };
  // scores of step i, the first half of K's fragments read before; the blocks' sums run as chains of their own
  auto scores = [&](int i) QTTS_PG_INLINE {
    f32x16 a[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) a[u][e] = 0.0f;
    read_k(i, 1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < KS / 2; ++s)
#pragma unroll
        for (int u = 0; u < NU; ++u) a[u] = E::mma32(kf[h][u][s], q[h * KS / 2 + s], a[u]);
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[16 * u + e] = a[u][e];
  };
  // O^T += V^T P^T of MFMA steps kk and kk + 1 of step i
  auto products = [&](int i, auto kk_) QTTS_PG_INLINE {
    constexpr int kk = decltype(kk_)::value;
    uint32_t va[4], vb[4];
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
      va[mb] = vaddr[mb] + (i & 1) * 2 * BUF;
      vb[mb] = va[mb] ^ (swz<D>(8) * 16);       // rows 8 further: their chunks' positions
    }
    if constexpr (D == 128) {
      u32x2 a[8], bq[8];
      tr_read16<16 * kk * D * 2, 16 * kk * D * 2 + 8 * D * 2, 16 * D * 2>(va, vb, a, bq);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const u32x4 v = {a[4 * j + mb][0], a[4 * j + mb][1], bq[4 * j + mb][0], bq[4 * j + mb][1]};
          o[mb] = E::mma32(v, p[kk + j], o[mb]);
        }
    } else {
      u32x2 a[4], bq[4];
      const uint32_t xa[4] = {va[0], va[1], va[0] + 16 * D * 2, va[1] + 16 * D * 2};
      const uint32_t xb[4] = {vb[0], vb[1], vb[0] + 16 * D * 2, vb[1] + 16 * D * 2};
      tr_read8<16 * kk * D * 2, 16 * kk * D * 2 + 8 * D * 2>(xa, xb, a, bq);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const u32x4 v = {a[2 * j + mb][0], a[2 * j + mb][1], bq[2 * j + mb][0], bq[2 * j + mb][1]};
          o[mb] = E::mma32(v, p[kk + j], o[mb]);
        }
    }
  };
  auto mask = [&](int i, int has_i) QTTS_PG_INLINE {
    const int key0 = key_of(i * NS + ks);
#pragma unroll
    for (int e = 0; e < 16 * NU; ++e) {
      const int in = 32 * (e >> 4) + 8 * ((e >> 2) & 3) + 4 * hf + (e & 3), key = key0 + in;
      const bool seen = (((has_i >> (in >> 4)) & 1) != 0) & (key <= pos) & ((key >= first_key) | (key < g.sinks));
      sc[e] = seen ? sc[e] : -INFINITY;
    }
  };
  auto softmax = [&](const Piece& kp, const Piece& vp) QTTS_PG_INLINE {   // (vp: steps of 8 pieces)
    float bm = sc[0];
#pragma unroll
    for (int e = 1; e < 16 * NU; ++e) bm = fmaxf(bm, sc[e]);
    bm = fmaxf(bm, xlane_f<5>(bm));
    if (__builtin_amdgcn_ballot_w64(bm > m + 8.0f / SL) != 0ull) {
      const float mn = fmaxf(m, bm);
      const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * SL);
      l *= al;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[mb][e] *= al;
      m = mn;
    }
    const float nm = m == -INFINITY ? 0.0f : -m * SL;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8 * NU; ++j) {
      const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[2 * j], SL, nm)), e1 = __builtin_amdgcn_exp2f(fmaf(sc[2 * j + 1], SL, nm));
      sum += e0;
      sum += e1;
      p[j >> 2][j & 3] = E::pack(e0, e1);
      // one copy at a time between the exponentials: issued together each holds the wave for 130 cycles
      constexpr int every = 8 * NU / (PAIR * copy.N);
      if (j % every == every - 1) {
        const int n = j / every;
        if (n < copy.N) copy.one(kp.rs, kp.dst + n * 1024, kp.off[n]);
        else copy.one(vp.rs, vp.dst + (n - copy.N) * 1024, vp.off[n - copy.N]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    l += sum;
  };
  auto barrier = [&]() QTTS_PG_INLINE {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // what step i copies (step i + 1's pieces) and whether it needs masks or partial pieces
  const Entries first = entries(0);
  Entries second = entries(1);
  uint32_t has = found(first);                            // of the step computed
  const int half = PAIR == 2 ? 0 : w >> 2;
  const uint16_t* const head_a = half == 0 ? k_head : v_head;
  issue(piece(head_a, own(first, has), 0, half));
  if constexpr (PAIR == 2) issue(piece(v_head, own(first, has), 0, 1));
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    wait_vm_lds<0>();                 // this wave's copies have landed, its reads of the other buffer are done
    barrier();
    read_k(i, 0);
    const uint32_t has_n = found(second);                 // of step i + 1
    const int page = own(second, has_n);
    Piece kp = piece(head_a, page, i + 1, half), vp = PAIR == 2 ? piece(v_head, page, i + 1, 1) : kp;
    second = entries(i + 2);
    const int has_i = (int)(has >> (ks * PPB)) & ((1 << PPB) - 1);
    has = has_n;
    const bool whole = (i >= fs) & (i < fe) & (has_i == (1 << PPB) - 1) & (page >= 0);
    scores(i);
    if (!whole) {
      part(kp);
      if constexpr (PAIR == 2) part(vp);
      mask(i, has_i);
    }
    softmax(kp, vp);
    products(i, std::integral_constant<int, 0>{});
    if constexpr (NU == 2) products(i, std::integral_constant<int, 2>{});
  }
  wait_vm_lds<0>();
  l += xlane_f<5>(l);

  // join the splits: M = max m_s, L = sum l_s e^(m_s - M), O = sum O_s e^(m_s - M), in key order; wave (ks, wr)
  // finishes channels ks D / NS .. of its rows
  float* sml = reinterpret_cast<float*>(smem + ROOM) + wr * NS * 2 * 32;
  float* so = reinterpret_cast<float*>(smem) + wr * NS * MB * 1024;
  float L = l;
  if constexpr (NS > 1) {
    if (hf == 0) {
      sml[(2 * ks) * 32 + c] = m;
      sml[(2 * ks + 1) * 32 + c] = l;
    }
    __syncthreads();                    // every buffer is dead
    float M = -INFINITY;
    L = 0.0f;
#pragma unroll
    for (int v = 0; v < NS; ++v) M = fmaxf(M, sml[2 * v * 32 + c]);
#pragma unroll
    for (int v = 0; v < NS; ++v) {
      const float mv = sml[2 * v * 32 + c], lv = sml[(2 * v + 1) * 32 + c];
      L += mv == -INFINITY ? lv : lv * __builtin_amdgcn_exp2f((mv - M) * SL);   // (-inf: 0, or NaN after NaN scores)
    }
    const float sw = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * SL);
    // [row group][split][channel block][register quad][lane][4]; O^T: column = row c, register e of block mb =
    // channel 32 mb + 8 (e >> 2) + 4 hf + (e & 3)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f32x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = o[mb][4 * e + k] * sw;
        *reinterpret_cast<f32x4*>(so + ((ks * MB + mb) * 4 + e) * 256 + lane * 4) = x;
      }
    __syncthreads();
  }
  const float rl = L == 0.0f ? 0.0f : 1.0f / L;
  uint16_t* op = g.out + (long long)(at.first + ti) * g.o_token + (long long)head * g.o_head + 4 * hf;
  constexpr int NQ = MB * 4 / NS;     // register quads that this wave finishes
  f32x4 y[NQ];
  uint32_t worst = 0u;                // largest magnitude by its bits (x - x would be contracted with the product)
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    if constexpr (NS > 1) {
      const int e = ks * NQ + j;
      y[j] = *reinterpret_cast<const f32x4*>(so + e * 256 + lane * 4);
#pragma unroll
      for (int v = 1; v < NS; ++v) y[j] += *reinterpret_cast<const f32x4*>(so + (v * MB * 4 + e) * 256 + lane * 4);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) y[j][k] = o[j >> 2][4 * (j & 3) + k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      y[j][k] *= rl;
      worst = max(worst, __float_as_uint(y[j][k]) & 0x7fffffffu);
    }
  }
  worst = max(worst, xlane<5>(worst));
  if constexpr (NS > 1) {   // rows that are to be summed again, known to every split
    __syncthreads();        // (all have read the words)
    if (hf == 0) sml[2 * ks * 32 + c] = __uint_as_float(worst);
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NS; ++v) worst = max(worst, __float_as_uint(sml[2 * v * 32 + c]));
  }
  const bool redo = (worst >= 0x7f800000u) & (L == L);
  if (stored && !redo) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int e = ks * NQ + j;
      u32x2 p;
      p[0] = E::pack(y[j][0], y[j][1]);
      p[1] = E::pack(y[j][2], y[j][3]);
      *reinterpret_cast<u32x2*>(op + 8 * e) = p;
    }
  }
  uint64_t again = __builtin_amdgcn_ballot_w64(stored & redo) & 0xffffffffull;
  for (int n = 0; again != 0ull; ++n) {        // the splits take them in turn
    const int src = __builtin_ctzll(again);
    again &= again - 1;
    if (n % NS == ks)
      exact_row<E, D>(g, at.b, kvh, at.first + __builtin_amdgcn_readlane(ti, src), __builtin_amdgcn_readlane(head, src),
                      __builtin_amdgcn_readlane(pos, src));
  }
}

// ---- host ----------------------------------------------------------------------------------

constexpr long long kMostKeys = 1ll << 30;   // of a table row: positions and windows stay inside int

bool attn_ok(const QttsPagedCache* cache, int n_tokens, int hq, const void* q, long long q_token, long long q_head, const void* out,
             long long o_token, long long o_head, const int* table, int width, long long table_stride, const int* lens,
             int requests, float scale, int window, int sinks) {
  if (!cache_ok(cache) || requests < 1 || n_tokens < 0 || hq < 1 || hq % cache->num_kv_heads != 0) return false;
  if (q == nullptr || out == nullptr || table == nullptr || lens == nullptr) return false;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u) != 0) return false;
  if (((q_token | q_head | o_token | o_head) & 7) != 0) return false;
  if (width < 1 || table_stride < width || (long long)width * cache->page_size > kMostKeys) return false;
  if (!(scale > 0.0f) || !std::isfinite(scale) || window < 0 || sinks < 0) return false;
  return (long long)n_tokens * hq <= INT_MAX / 2;
}

AttnArgs attn_args(const QttsPagedCache* cache, int hq, const void* q, long long q_token, long long q_head, void* out,
                   long long o_token, long long o_head, const int* table, int width, long long table_stride,
                   const int* lens, int requests, float scale, int window, int sinks) {
  AttnArgs g{};
  g.q = static_cast<const uint16_t*>(q);
  g.out = static_cast<uint16_t*>(out);
  g.q_token = q_token; g.q_head = q_head; g.o_token = o_token; g.o_head = o_head;
  g.pages = pages_of(cache);
  g.table = table;
  g.table_stride = table_stride;
  g.width = width;
  g.lens = lens;
  g.requests = requests;
  g.hq = hq;
  g.group = hq / cache->num_kv_heads;
  g.hkv = cache->num_kv_heads;
  g.scale_log2 = scale * 1.4426950408889634f;
  g.window = (int)std::min<long long>(window, kMostKeys);   // (as good as none)
  g.sinks = window > 0 ? sinks : 0;
  return g;
}

// How decode splits requests into units. Pairs of a request and a KV head that fill the GPU by themselves (128 on) are
// split only where they are long: a second launch joins the units, and short units are mostly their own beginning
// and end (us, unsplit against units of 512 keys: 200 requests of 100 to 700 keys 59.5 : 88.9, 64 of 50 to 300
// 13.3 : 22.7 (256 keys); 24 under a window of 1024 21.6 : 26.5), but 64 ragged ones up to 4090 keys leave a shorter last
// round (101.8 : 108.8, 16 up to 4000 31.0 : 33.5). Fewer pairs are split down to 256 keys a unit, until there
// are 512 units (one request of 1000 keys 10.0 : 11.5 unsplit, of 2000 10.7 : 21.7, of 60000 in 512 units 46.7, in 1024
// 49.8). Up to 512 keys 8 waves take them unsplit (one of 300 to 512 9.0 : 10.0, 4 10.3 : 10.8), up to 768 those of 64
// channels (700 keys 8.6 to 9.0 : 9.7, 300 6.3 to 6.8 : 9.4) or of 64 pairs (12 requests of 700 14.7 : 16.4, but of 1000
// 19.0 : 17.5); up to 256 keys 4 waves do (6.5, 8 waves 7.1).
struct Split {
  int splits, blocks;      // most units, blocks a unit
  bool wide;               // 8 waves a workgroup, where a CU has one
};
Split decode_split(int requests, int hkv, int group, int head_dim, int width, int page_size, int max_len, int window, int sinks) {
  long long keys = std::min<long long>((long long)width * page_size, max_len);
  if (window > 0) keys = std::min<long long>(keys, (long long)window + std::min<long long>(sinks, keys) + 2 * DKB);
  const long long blocks = std::max<long long>(1, (keys + DKB - 1) / DKB);
  const long long pairs = (long long)requests * hkv * ((group + 15) / 16);
  if (pairs >= 128 && blocks < 64) return Split{1, (int)blocks, pairs <= 256};
  if (pairs < 128 && blocks <= (head_dim == 64 || pairs >= 64 ? 24 : 16)) return Split{1, (int)blocks, blocks > 8};
  const long long units = pairs >= 128 ? 4096 : 512, least = pairs > 256 ? 16 : 8;
  long long per = std::max(least, (blocks * pairs + units - 1) / units);
  per = std::min((per + 3) / 4 * 4, blocks);
  return Split{(int)((blocks + per - 1) / per), (int)per, false};
}

template <class E, int D>
void launch_decode(const AttnArgs& g, bool wide, hipStream_t st) {
  const int tiles = (g.group + 15) / 16;
  const dim3 grid((unsigned)((long long)g.requests * g.hkv * tiles * g.splits));
  if (wide) hipLaunchKernelGGL((decode_kernel<E, D, 8>), grid, dim3(512), 0, st, g);
  else hipLaunchKernelGGL((decode_kernel<E, D, 4>), grid, dim3(256), 0, st, g);
  if (g.splits > 1) hipLaunchKernelGGL((decode_join_kernel<E, D>), dim3((unsigned)(g.requests * g.hq)), dim3(256), 0, st, g);
}

template <class E, int D, int NS>
hipError_t launch_prefill(const AttnArgs& g, hipStream_t st) {
  constexpr int PM = 32 * PWV / NS;
  // every request ends with a tile that may be part empty; no more tiles than rows
  const long long n = (long long)g.tokens * g.group, tiles = std::min(n / PM + g.requests, n);
  if (tiles * g.hkv > INT_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL((prefill_kernel<E, D, NS>), dim3((unsigned)(tiles * g.hkv)), dim3(64 * PWV), 0, st, g);
  return hipGetLastError();
}

// Which tiles: 256 rows unsplit (NS = 1) take the fewest key steps for all the rows together, 64 rows in 4 key splits
// the shortest chain for one tile. A launch takes the longer of the longest tile's chain and all tiles' steps over
// the tiles that run at once (one a CU with 128 channels, two with 64), estimated with 2 to 2.5 us a tile and
// 1.6, 2.4 and 1.6 us a step (loaded and unloaded CUs: 1.4 to 2.2). Measured us, NS = 1 : 2 : 4, of 16 / 8 heads of 128:
// a prompt of 300 tokens 16.4 : 14.4 : 11.6, 1000 35.6 : 23.7 : 18.0, 2000 61.3 : 39.4 : 37.5, 4096 117.8 : 89.5 : 114.5,
// 8192 278.8 : 294.8 : 366; 64 prompts of 20 to 100 25.5 : 36.1 : 40.9; 8 of 50 to 100 after 4000 104 : 57 : 44; 8192 under
// a window of 512 77 : 81 : 107.
// Merged order (find_tile): where a tile's keys grow with its place and the longest tile is more than half of what all take;
// its start costs 0.5 us, and it reads more requests' keys at once (us, merged : not: 4 prompts of 2000 91 : 117, 16 of 500
// 43.5 : 51.8, 6 of 100 to 3000 115 : 130, 16 of 100 to 200, 32 / 4 heads of 64, 15.2 : 16.5; but 40 of 300 67 : 62, 3 under a
// window 100 : 95, 8 pieces of up to 512 after 4000 60.5 : 58.7).
struct Tiles {
  int splits;
  bool merged;
};
template <int D>
Tiles prefill_tiles(const AttnArgs& g, int max_len) {
  const double each = (double)g.tokens / g.requests, slots = D == 128 ? 256 : 512;
  Tiles pick{1, false};
  double best = 1e30;
  for (int ns = 1; ns <= 4; ns *= 2) {
    const int pm = 32 * PWV / ns, step = ns == 4 ? 128 : 64 * ns;
    const double tile = ns == 2 ? 2.5 : 2.0, cost = ns == 2 ? 2.4 : 1.6, span = (double)g.window + (double)g.sinks + (double)pm / g.group;
    const double rows = each * g.group, n = (g.requests == 1 ? std::ceil(rows / pm) : std::max(1.0, rows / pm + 0.5)) * g.requests * g.hkv;
    double longest = max_len, mean = std::max(max_len - each / 2, max_len / 2.0);
    if (g.window > 0) {
      longest = std::min(longest, span);
      mean = std::min(mean, span);
    }
    const double chain = tile + std::ceil(longest / step) * cost, all = n / slots * (tile + std::ceil(mean / step) * cost);
    if (std::max(chain, all) < best) {
      best = std::max(chain, all);
      pick = Tiles{ns, g.requests > 1 && g.requests <= 64 && longest > 1.25 * mean && 2 * chain > all};
    }
  }
  return pick;
}
template <class E, int D>
hipError_t launch_prefill_any(AttnArgs& g, int max_len, hipStream_t st) {
  const Tiles t = prefill_tiles<D>(g, max_len);
  g.merged = t.merged ? 1 : 0;
  switch (t.splits) {
    case 1: return launch_prefill<E, D, 1>(g, st);
    case 2: return launch_prefill<E, D, 2>(g, st);
    default: return launch_prefill<E, D, 4>(g, st);
  }
}

}  // namespace pg
}  // namespace qtts

using namespace qtts;
using namespace qtts::pg;

extern "C" {

size_t qtts_paged_decode_workspace_bytes(int n_requests, int num_q_heads, int num_kv_heads, int head_dim, int table_width,
                                         int page_size, int max_len, int window, int sinks) {
  if (n_requests < 1 || num_kv_heads < 1 || num_q_heads < 1 || num_q_heads % num_kv_heads != 0 || head_dim < 1 ||
      table_width < 1 || page_size < 1 || max_len < 1 || window < 0 || sinks < 0)
    return 0;
  const Split s = decode_split(n_requests, num_kv_heads, num_q_heads / num_kv_heads, head_dim, table_width, page_size, max_len, window, sinks);
  return s.splits == 1 ? 0 : (size_t)n_requests * num_q_heads * s.splits * (head_dim + 2) * 4;
}

hipError_t qtts_paged_attention_decode(const QttsPagedCache* cache, int n_requests, int num_q_heads, const void* q,
                                       long long q_token_stride, long long q_head_stride, void* out,
                                       long long out_token_stride, long long out_head_stride, const int* block_table,
                                       int table_width, long long table_stride, const int* kv_lens, int max_len,
                                       float scale, int window, int sinks, void* workspace, size_t workspace_bytes,
                                       hipStream_t stream) {
  if (!attn_ok(cache, n_requests, num_q_heads, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
               block_table, table_width, table_stride, kv_lens, n_requests, scale, window, sinks) || max_len < 1)
    return hipErrorInvalidValue;
  AttnArgs g = attn_args(cache, num_q_heads, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
                         block_table, table_width, table_stride, kv_lens, n_requests, scale, window, sinks);
  const Split s = decode_split(n_requests, g.hkv, g.group, cache->head_dim, table_width, cache->page_size, max_len, window, sinks);
  g.splits = s.splits;
  g.blocks = s.blocks;
  if (s.splits > 1) {
    const size_t sums = (size_t)n_requests * num_q_heads * s.splits * cache->head_dim * 4;
    const size_t need = qtts_paged_decode_workspace_bytes(n_requests, num_q_heads, g.hkv, cache->head_dim, table_width,
                                                          cache->page_size, max_len, window, sinks);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
      return hipErrorInvalidValue;
    g.part = static_cast<float*>(workspace);
    g.part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums);
  }
  if ((long long)n_requests * g.hkv * ((g.group + 15) / 16) * g.splits > INT_MAX) return hipErrorInvalidValue;
  if (cache->dtype == QTTS_BF16) {
    if (cache->head_dim == 128) launch_decode<Bf16, 128>(g, s.wide, stream);
    else launch_decode<Bf16, 64>(g, s.wide, stream);
  } else {
    if (cache->head_dim == 128) launch_decode<F16, 128>(g, s.wide, stream);
    else launch_decode<F16, 64>(g, s.wide, stream);
  }
  return hipGetLastError();
}

hipError_t qtts_paged_attention_prefill(const QttsPagedCache* cache, int n_requests, int n_tokens, int num_q_heads,
                                        const void* q, long long q_token_stride, long long q_head_stride, void* out,
                                        long long out_token_stride, long long out_head_stride, const int* block_table,
                                        int table_width, long long table_stride, const int* kv_lens, const int* cu_tokens,
                                        int max_len, float scale, int window, int sinks, hipStream_t stream) {
  if (!attn_ok(cache, n_tokens, num_q_heads, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
               block_table, table_width, table_stride, kv_lens, n_requests, scale, window, sinks) || cu_tokens == nullptr || max_len < 1)
    return hipErrorInvalidValue;
  if (n_tokens == 0) return hipSuccess;
  AttnArgs g = attn_args(cache, num_q_heads, q, q_token_stride, q_head_stride, out, out_token_stride, out_head_stride,
                         block_table, table_width, table_stride, kv_lens, n_requests, scale, window, sinks);
  g.cu = cu_tokens;
  g.tokens = n_tokens;
  const int most = (int)std::min<long long>(max_len, (long long)table_width * cache->page_size);
  if (cache->dtype == QTTS_BF16)
    return cache->head_dim == 128 ? launch_prefill_any<Bf16, 128>(g, most, stream) : launch_prefill_any<Bf16, 64>(g, most, stream);
  return cache->head_dim == 128 ? launch_prefill_any<F16, 128>(g, most, stream) : launch_prefill_any<F16, 64>(g, most, stream);
}

}  // extern "C"
