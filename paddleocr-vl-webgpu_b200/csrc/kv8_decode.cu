// kv8_decode.cu -- one token of every sequence against the 8-bit paged cache,
// with the decode M-RoPE and the append fused.
//
// Per sequence with n rows before the append: q and the new key are rotated
// at rope_row; the rotated key and the value become row n % 32 of the tail;
// attention runs over the n / 32 full pages (8 bits) and the 1 .. 32 tail rows
// (fp16); a tail that is now full is quantised into page table[slot][n / 32].
//   s_r = scale_K(r) (q . k_r) / sqrt(128),   out = sum_r softmax(s)_r scale_V(r) v_r
//
// The rotation multiplies and adds with a rounding each (no fused
// multiply-add), so a cached key row is the plain f32 formula's, bit for bit.
#include <cuda_runtime.h>
#include <math_constants.h>

#include "kv8.cuh"

namespace pvlc {
namespace kv8 {

constexpr int MAX_GROUP = 16;

struct DecodeParams {
  View c;
  const __half* q;
  const __half* k_new;
  const __half* v_new;
  const float* rope_cos;
  const float* rope_sin;
  const int32_t* rope_row;
  const int32_t* slot;
  __half* out;
  uint32_t q_stride, kv_stride, rope_rows, batch, group;
  uint32_t* flags;
};

// What is wrong with sequence b (0: nothing); its slot, rows and table row.
__device__ __forceinline__ uint32_t check_sequence(const DecodeParams& p, uint32_t b, int32_t slot,
                                                   int32_t* rows, uint32_t* rope) {
  if (slot < 0 || (uint32_t)slot >= p.c.slots) return kFlagSlot;
  const int32_t n = p.c.tokens[slot];
  const int32_t r = p.rope_row ? p.rope_row[b] : n;
  uint32_t bad = 0;
  if (n < 0 || !rows_fit((uint64_t)n + 1, p.c.max_pages)) bad |= kFlagCacheRow;
  if (r < 0 || (uint32_t)r >= p.rope_rows) bad |= kFlagRopeRow;
  *rows = n;
  *rope = (uint32_t)r;
  return bad;
}

// Dim d of a head row rotated: x cos - y sin below 64 (y = dim d + 64),
// x cos + y sin above (y = dim d - 64).
__device__ __forceinline__ float rotated(const __half* row, uint32_t d, const DecodeParams& p,
                                         uint32_t r) {
  const size_t at = ((size_t)mrope_axis(d) * p.rope_rows + r) * HD + d;
  const float x = __half2float(row[d]), y = __half2float(row[d ^ 64]);
  return __fadd_rn(__fmul_rn(x, p.rope_cos[at]), __fmul_rn(d < 64 ? -y : y, p.rope_sin[at]));
}

// One block per (KV head, sequence), thread d = dim d.
template <int CODE>
__global__ void __launch_bounds__(HD) kv8_decode_kernel(const DecodeParams p) {
  __shared__ float q[MAX_GROUP][HD];
  __shared__ float w[MAX_GROUP][PAGE];
  __shared__ float m[MAX_GROUP], l[MAX_GROUP], f[MAX_GROUP];
  const uint32_t h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int warp = d >> 5, lane = d & 31;
  const int32_t slot = p.slot ? p.slot[b] : (int32_t)b;
  if (slot == -1) return;
  const uint32_t G = p.group, QH = G * p.c.heads;
  __half* out = p.out + ((size_t)b * QH + h * G) * HD;
  int32_t n = 0;
  uint32_t rr = 0;
  if (const uint32_t bad = check_sequence(p, b, slot, &n, &rr)) {
    if (d == 0) atomicOr(p.flags, bad);
    for (uint32_t i = 0; i < G; ++i) out[i * HD + d] = __float2half_rn(0.f);
    return;
  }
  const __half* qr = p.q + (size_t)b * p.q_stride + (size_t)h * G * HD;
  for (uint32_t i = 0; i < G; ++i)
    q[i][d] = __half2float(__float2half_rn(rotated(qr + i * HD, d, p, rr))) * 0.08838834764831845f;
  __half* tk = tail_rows(p.c, slot, 0, h);
  __half* tv = tail_rows(p.c, slot, 1, h);
  const uint32_t last = n % PAGE, full = n / PAGE;
  tk[last * HD + d] = __float2half_rn(rotated(p.k_new + (size_t)b * p.kv_stride + h * HD, d, p, rr));
  tv[last * HD + d] = p.v_new[(size_t)b * p.kv_stride + h * HD + d];
  if (d < G) {
    m[d] = -CUDART_INF_F;
    l[d] = 0.f;
  }
  float o[MAX_GROUP];
  for (uint32_t i = 0; i < MAX_GROUP; ++i) o[i] = 0.f;
  __syncthreads();
  const int32_t* row = p.c.table + (size_t)slot * p.c.max_pages;
  for (uint32_t j = 0; j <= full; ++j) {
    const bool open = j == full;
    const uint32_t live = open ? last + 1 : PAGE;
    const uint8_t *kc = nullptr, *vc = nullptr;
    float sk = 1.f, sv = 1.f;
    if (!open) {
      const int32_t page = row[j];
      if (page < 0 || (uint32_t)page >= p.c.pages) {
        if (d == 0) atomicOr(p.flags, kFlagPage);
        sk = sv = CUDART_NAN_F;
        kc = vc = p.c.codes;
      } else {
        kc = block_codes(p.c, page, 0, h);
        vc = block_codes(p.c, page, 1, h);
        sk = p.c.scales[((size_t)page * p.c.heads + h) * 2];
        sv = p.c.scales[((size_t)page * p.c.heads + h) * 2 + 1];
      }
    }
    auto value = [&](const uint8_t* codes, const __half* tail, uint32_t r, uint32_t e) {
      if (open) return __half2float(tail[r * HD + e]);
      if (CODE == PVLC_KV8_INT8) return (float)(int8_t)codes[r * HD + e];
      return __half2float(__half(__nv_cvt_fp8_to_halfraw(codes[r * HD + e], __NV_E4M3)));
    };
    for (uint32_t r = warp; r < live; r += HD / 32)
      for (uint32_t i = 0; i < G; ++i) {
        float s = 0.f;
        for (uint32_t e = lane; e < HD; e += 32) s += q[i][e] * value(kc, tk, r, e);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (lane == 0) w[i][r] = s * sk;
      }
    __syncthreads();
    for (uint32_t i = warp; i < G; i += HD / 32) {
      const float s = lane < live ? w[i][lane] : -CUDART_INF_F;
      float top = fmaxf(m[i], s);
      for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float e = lane < live ? expf(s - top) : 0.f;
      float sum = e;
      for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      w[i][lane] = e * sv;
      __syncwarp();
      if (lane == 0) {
        f[i] = expf(m[i] - top);
        l[i] = l[i] * f[i] + sum;
        m[i] = top;
      }
    }
    __syncthreads();
    for (uint32_t i = 0; i < G; ++i) {
      float s = o[i] * f[i];
      for (uint32_t r = 0; r < live; ++r) s += w[i][r] * value(vc, tv, r, d);
      o[i] = s;
    }
    __syncthreads();
  }
  for (uint32_t i = 0; i < G; ++i) out[i * HD + d] = __float2half_rn(o[i] / l[i]);
  if (last == PAGE - 1 && warp < 2) {   // the block is full: warp 0 its keys, warp 1 its values
    const int32_t page = row[full];
    if (page < 0 || (uint32_t)page >= p.c.pages) {
      if (lane == 0) atomicOr(p.flags, kFlagPage);
      return;
    }
    const uint4* x4 = reinterpret_cast<const uint4*>(warp ? tv : tk);
    uint4 x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[2 * i] = x4[(4 * i + (lane >> 3)) * (HD / 8) + 2 * (lane & 7)];
      x[2 * i + 1] = x4[(4 * i + (lane >> 3)) * (HD / 8) + 2 * (lane & 7) + 1];
    }
    quantise_block<CODE>(x, block_codes(p.c, page, warp, h),
                         p.c.scales + ((size_t)page * p.c.heads + h) * 2 + warp, lane);
  }
}

}  // namespace kv8

size_t kv8_decode_scratch_bytes(uint32_t, uint32_t, uint32_t) { return 0; }

int kv8_decode_launch(const pvlc_kv8_cache& c, uint32_t layer, const Kv8DecodeArgs& a,
                      cudaStream_t stream) {
  kv8::DecodeParams p;
  p.c = kv8::view_of(c, layer);
  p.q = reinterpret_cast<const __half*>(a.q);
  p.k_new = reinterpret_cast<const __half*>(a.k_new);
  p.v_new = reinterpret_cast<const __half*>(a.v_new);
  p.rope_cos = a.rope_cos;
  p.rope_sin = a.rope_sin;
  p.rope_row = a.rope_row;
  p.slot = a.slot;
  p.out = reinterpret_cast<__half*>(a.out);
  p.q_stride = a.q_stride;
  p.kv_stride = a.kv_stride;
  p.rope_rows = a.rope_rows;
  p.batch = a.batch;
  p.group = a.query_heads / c.kv_heads;
  p.flags = static_cast<uint32_t*>(a.workspace);
  const dim3 grid(c.kv_heads, a.batch);
  if (c.code_type == PVLC_KV8_E4M3)
    kv8::kv8_decode_kernel<PVLC_KV8_E4M3><<<grid, kv8::HD, 0, stream>>>(p);
  else
    kv8::kv8_decode_kernel<PVLC_KV8_INT8><<<grid, kv8::HD, 0, stream>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

}  // namespace pvlc
