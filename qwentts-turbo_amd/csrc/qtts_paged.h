// What the paged-cache kernels share: the two 16-bit element types and the cache as kernels see it.
#pragma once
#include <hip/hip_runtime.h>
#include "qwentts_amd.h"
#include "qtts_common.h"

namespace qtts {
namespace pg {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define QTTS_PG_INLINE __attribute__((always_inline))

// 16-bit elements held as bits: unpacking to f32, packing with one rounding to nearest even, and the
// matrix products of each type (operands are 8 elements a lane).
struct Bf16 {
  __device__ static __forceinline__ float lo(uint32_t w) { return bflo(w); }
  __device__ static __forceinline__ float hi(uint32_t w) { return bfhi(w); }
  __device__ static __forceinline__ uint32_t pack(float a, float b) { return f2bf2(a, b); }
  __device__ static __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct F16 {
  __device__ static __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
  __device__ static __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
  __device__ static __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// One layer's pages; strides in elements, shared by K and V.
struct Pages {
  const uint16_t* k;
  const uint16_t* v;
  int page_stride, head_stride, slot_stride;
  int num_pages, shift;      // page size = 1 << shift
};

// A cache that the kernels can address: a page size that is a power of two of at least 16 (a 16-row copy
// stays inside a page), 64 or 128 channels, 16-byte rows (alignment and strides), and a page's 16-row
// copies inside 31-bit offsets.
inline bool cache_ok(const QttsPagedCache* c) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->num_pages < 1 || c->num_kv_heads < 1) return false;
  if (c->dtype != QTTS_BF16 && c->dtype != QTTS_F16) return false;
  if (c->head_dim != 64 && c->head_dim != 128) return false;
  if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)) != 0) return false;
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u) != 0) return false;
  if (((c->page_stride | c->head_stride | c->slot_stride) & 7) != 0) return false;
  if (c->page_stride < 0 || c->page_stride > 0x7fffffffLL || c->head_stride < 0 || c->head_stride > 0x7fffffffLL) return false;
  return c->slot_stride >= c->head_dim && c->slot_stride <= (1 << 24);
}
inline Pages pages_of(const QttsPagedCache* c) {
  return Pages{static_cast<const uint16_t*>(c->k), static_cast<const uint16_t*>(c->v), (int)c->page_stride,
               (int)c->head_stride, (int)c->slot_stride, c->num_pages, __builtin_ctz((unsigned)c->page_size)};
}

}  // namespace pg
}  // namespace qtts
