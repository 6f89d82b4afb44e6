// kv8.cuh -- what the kernels of the 8-bit paged KV cache share: the cache's
// device view, the code types and the block scale.
//
// A page holds 32 rows of every KV head in 8-bit codes.  One (page, K or V,
// head) block of 32 x 128 values X has one scale,
//   scale = 2^e, e the smallest integer with max|X| <= Q 2^e
//   (Q = 448 for e4m3, 127 for int8; scale 1 for a block of zeros),
//   code = X / scale rounded to nearest, ties to even.
// A power of two makes the division and the later multiplication exact, so
// the code's own rounding is the only one a value ever gets (half a code step:
// 2^-4 of an e4m3 value, scale / 2 of an int8 one) and the codes do not depend
// on how a block's rows arrived.  A block that holds a NaN or an infinity gets
// scale NaN and codes 0: whatever attends to it reads NaN.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "pvlc_common.cuh"
#include "pvlc_internal.h"

namespace pvlc {
namespace kv8 {

constexpr int PAGE = 32;
constexpr int HD = 128;
constexpr uint32_t BLOCK_CODES = PAGE * HD;      // one (page, K/V, head) block

// Further fault bits of a workspace's word (0..3 are in pvlc_common.cuh).
constexpr uint32_t kFlagPage = 1u << 4;        // a page id outside the pool
constexpr uint32_t kFlagSlot = 1u << 5;        // a slot or parent out of range, or named twice
constexpr uint32_t kFlagExhausted = 1u << 6;   // no free page or slot left
constexpr uint32_t kFlagRows = 1u << 7;        // input rows out of range

struct View {
  uint8_t* codes;     // this layer's
  float* scales;
  __half* tails;
  const int32_t* table;
  const int32_t* tokens;
  uint32_t pages, slots, max_pages, heads;
};

inline View view_of(const pvlc_kv8_cache& c, uint32_t layer) {
  View v;
  v.codes = static_cast<uint8_t*>(c.codes) + (size_t)layer * c.pages * 2 * c.kv_heads * BLOCK_CODES;
  v.scales = c.scales + (size_t)layer * c.pages * c.kv_heads * 2;
  v.tails = reinterpret_cast<__half*>(c.tails) +
            (size_t)layer * c.slots * 2 * c.kv_heads * BLOCK_CODES;
  v.table = c.table;
  v.tokens = c.tokens;
  v.pages = c.pages;
  v.slots = c.slots;
  v.max_pages = c.max_pages;
  v.heads = c.kv_heads;
  return v;
}

// Rows [0, n) fit a slot when every full block has a table entry.
__host__ __device__ __forceinline__ bool rows_fit(uint64_t n, uint32_t max_pages) {
  return n / PAGE <= max_pages;
}

// A block's codes and its tail rows: [.., K or V, head].
__device__ __forceinline__ uint8_t* block_codes(const View& v, uint32_t page, uint32_t kv,
                                                uint32_t h) {
  return v.codes + (((size_t)page * 2 + kv) * v.heads + h) * BLOCK_CODES;
}
__device__ __forceinline__ __half* tail_rows(const View& v, uint32_t slot, uint32_t kv,
                                             uint32_t h) {
  return v.tails + (((size_t)slot * 2 + kv) * v.heads + h) * BLOCK_CODES;
}

// The exponent e of a block's scale; `amax` is finite and positive.  With
// amax = m 2^x, 0.5 <= m < 1, and Q = qm 2^qe likewise: e = x - qe + (m > qm).
template <int CODE>
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int x = static_cast<int>(bits >> 23) - 126;
  const uint32_t mant = bits & 0x7fffffu;
  // 448 = 0.875 * 2^9, 127 = 0.9921875 * 2^7
  return CODE == PVLC_KV8_E4M3 ? x - 9 + (mant > 0x600000u ? 1 : 0)
                               : x - 7 + (mant > 0x7e0000u ? 1 : 0);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four values, already divided by the scale, as four code bytes.
template <int CODE>
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  if (CODE == PVLC_KV8_E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  const uint32_t ab = __byte_perm(__float2int_rn(a), __float2int_rn(b), 0x0040);
  const uint32_t cd = __byte_perm(__float2int_rn(c), __float2int_rn(d), 0x0040);
  return (ab & 0xffffu) | (cd << 16);
}

// One warp quantises a [32, 128] block held in registers: lane l's x[2 i],
// x[2 i + 1] are dims 16 (l % 8) .. + 15 of row 4 i + l / 8.
template <int CODE>
__device__ __forceinline__ void quantise_block(const uint4 (&x)[16], uint8_t* codes, float* scale,
                                               int lane) {
  __half2 top = __float2half2_rn(0.f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(&w[e])));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    uint32_t t = *reinterpret_cast<uint32_t*>(&top);
    t = __shfl_xor_sync(0xffffffffu, t, o);
    top = __hmax2_nan(top, *reinterpret_cast<__half2*>(&t));
  }
  const float amax = __half2float(__hmax_nan(__low2half(top), __high2half(top)));
  const bool finite = amax <= 65504.f;   // false for NaN and infinity
  const int e = finite && amax > 0.f ? scale_exponent<CODE>(amax) : 0;
  const float inv = pow2f(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 q = x[2 * i + j];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * p]));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w[2 * p + 1]));
        out[2 * j + p] = finite ? pack_codes<CODE>(a.x * inv, a.y * inv, b.x * inv, b.y * inv) : 0u;
      }
    }
    *reinterpret_cast<uint4*>(codes + (4 * i + (lane >> 3)) * HD + (lane & 7) * 16) =
        make_uint4(out[0], out[1], out[2], out[3]);
  }
  if (lane == 0) *scale = finite ? pow2f(e) : __uint_as_float(0x7fc00000u);
}

}  // namespace kv8
}  // namespace pvlc
