// beam_topk.cu -- the best continuations of every request's beams.
//
// For request r with beams w (score s_w) and logits x_w[0 .. V), the K largest
//   c(w, v) = s_w + x_w[v] - log sum_u exp(x_w[u])
// with their beams and tokens, best first.  A NaN logit counts as -infinity
// and so does a candidate that comes out as NaN.  Candidates are ordered by
// their f64 score; equal scores by the lower beam, then the larger logit, then
// the lower token.  Within a beam the order is that of the logits, so each
// row's K best logits are enough, and they need no logarithm.
//
// One pass over the logits: a block holds a chunk of a row in registers, sums
// its exponentials against its own maximum and keeps its K best logits as
// 64-bit keys (ordered logit, then ~token).  A block per request then joins
// the chunks: the rows' log-sums in f64, so that candidates of two beams that
// differ by more than 1e-7 are told apart, and the K best of all.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "pvlc_internal.h"

namespace pvlc {
namespace beam {

constexpr int THREADS = 256;
constexpr int PER = 32;                      // logits a thread
constexpr uint32_t CHUNK = THREADS * PER;

typedef unsigned long long u64;

// Order-preserving bits of a float: -0 equals +0, NaN is -infinity.
__device__ __forceinline__ uint32_t ordered(float x) {
  x = isnan(x) ? -CUDART_INF_F : x + 0.f;
  const uint32_t b = __float_as_uint(x);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ u64 block_max(u64 v) {
  __shared__ u64 part[THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 y = __shfl_xor_sync(0xffffffffu, v, o);
    v = y > v ? y : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = part[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) r = part[i] > r ? part[i] : r;
  return r;
}

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) r += part[i];
  return r;
}

struct Params {
  const void* logits;
  uint64_t ld;
  const float* scores;
  uint32_t batch, beams, vocab, topk, chunks;
  u64* keys;          // [rows][chunks][topk]
  float2* sums;       // [rows][chunks] (maximum, sum of exponentials against it)
  float* out_score;
  int32_t* out_beam;
  int32_t* out_token;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) beam_chunk_kernel(const Params p) {
  const uint32_t row = blockIdx.y, c = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  float v[PER];
  u64 best = 0;       // below every logit's key
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t at = c * CHUNK + i * THREADS + threadIdx.x;
    v[i] = at < p.vocab ? (float)x[at] : -CUDART_INF_F;
    const u64 key = at < p.vocab ? (u64)ordered(v[i]) << 32 | (0xffffffffu - at) : 0;
    best = key > best ? key : best;
  }
  u64 top = block_max(best);
  const float m = from_ordered((uint32_t)(top >> 32));
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) s += v[i] > -CUDART_INF_F ? expf(v[i] - m) : 0.f;
  s = block_sum(s);
  const size_t slot = (size_t)row * p.chunks + c;
  if (threadIdx.x == 0) p.sums[slot] = make_float2(m, s);
  for (uint32_t k = 0; k < p.topk; ++k) {
    if (threadIdx.x == 0) p.keys[slot * p.topk + k] = top;
    if (top == 0) continue;                  // fewer logits than K
    best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t at = c * CHUNK + i * THREADS + threadIdx.x;
      const u64 key = at < p.vocab ? (u64)ordered(v[i]) << 32 | (0xffffffffu - at) : 0;
      if (key < top && key > best) best = key;
    }
    top = block_max(best);
  }
}

struct Cand {
  double score;       // NaN marks "none"
  uint32_t beam;
  u64 key;
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) {
  if (a.key == 0 || b.key == 0) return a.key != 0;
  if (a.score != b.score) return a.score > b.score;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}
__device__ __forceinline__ Cand shfl(const Cand& c, int o) {
  Cand r;
  r.score = __shfl_xor_sync(0xffffffffu, c.score, o);
  r.beam = __shfl_xor_sync(0xffffffffu, c.beam, o);
  r.key = __shfl_xor_sync(0xffffffffu, c.key, o);
  return r;
}

__global__ void __launch_bounds__(THREADS) beam_join_kernel(const Params p) {
  __shared__ double base[PVLC_BEAM_MAX_BEAMS];
  __shared__ Cand part[THREADS / 32];
  const uint32_t r = blockIdx.x, W = p.beams;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (uint32_t w = warp; w < W; w += THREADS / 32) {
    const float2* s = p.sums + (size_t)(r * W + w) * p.chunks;
    float m = -CUDART_INF_F;
    for (uint32_t c = lane; c < p.chunks; c += 32) m = fmaxf(m, s[c].x);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    double t = 0.0;
    for (uint32_t c = lane; c < p.chunks; c += 32)
      if (s[c].x > -CUDART_INF_F) t += (double)s[c].y * exp((double)s[c].x - (double)m);
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) base[w] = (double)p.scores[r * W + w] - ((double)m + log(t));
  }
  __syncthreads();
  const uint32_t per = p.chunks * p.topk, n = W * per;
  const u64* keys = p.keys + (size_t)r * n;
  Cand last;
  last.key = 0;
  for (uint32_t k = 0; k < p.topk; ++k) {
    Cand best;
    best.key = 0;
    best.score = 0.0;
    best.beam = 0;
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
      Cand c;
      c.key = keys[i];
      if (c.key == 0) continue;
      c.beam = i / per;
      c.score = base[c.beam] + (double)from_ordered((uint32_t)(c.key >> 32));
      if (isnan(c.score)) c.score = -CUDART_INF;
      if ((k == 0 || before(last, c)) && before(c, best)) best = c;
    }
    for (int o = 16; o; o >>= 1) {
      const Cand y = shfl(best, o);
      if (before(y, best)) best = y;
    }
    __syncthreads();
    if (lane == 0) part[warp] = best;
    __syncthreads();
    best = part[0];
    for (int i = 1; i < THREADS / 32; ++i)
      if (before(part[i], best)) best = part[i];
    last = best;
    if (threadIdx.x == 0) {
      const size_t at = (size_t)r * p.topk + k;
      p.out_score[at] = (float)best.score;
      p.out_beam[at] = (int32_t)best.beam;
      p.out_token[at] = (int32_t)(0xffffffffu - (uint32_t)best.key);
    }
  }
}

uint32_t chunks_of(uint32_t vocab) { return (vocab + CHUNK - 1) / CHUNK; }

}  // namespace beam

size_t beam_topk_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t topk) {
  const size_t slots = (size_t)batch * beams * beam::chunks_of(vocab);
  return (slots * (topk + 1) * 8 + 255) / 256 * 256;
}

int beam_topk_launch(const BeamArgs& a, cudaStream_t stream) {
  beam::Params p;
  p.logits = a.logits;
  p.ld = a.ld;
  p.scores = a.scores;
  p.batch = a.batch;
  p.beams = a.beams;
  p.vocab = a.vocab;
  p.topk = a.topk;
  p.chunks = beam::chunks_of(a.vocab);
  p.keys = static_cast<beam::u64*>(a.workspace);
  p.sums = reinterpret_cast<float2*>(p.keys + (size_t)a.batch * a.beams * p.chunks * a.topk);
  p.out_score = a.out_score;
  p.out_beam = a.out_beam;
  p.out_token = a.out_token;
  const dim3 grid(p.chunks, a.batch * a.beams);
  if (a.half_logits)
    beam::beam_chunk_kernel<__half><<<grid, beam::THREADS, 0, stream>>>(p);
  else
    beam::beam_chunk_kernel<float><<<grid, beam::THREADS, 0, stream>>>(p);
  beam::beam_join_kernel<<<a.batch, beam::THREADS, 0, stream>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

}  // namespace pvlc
