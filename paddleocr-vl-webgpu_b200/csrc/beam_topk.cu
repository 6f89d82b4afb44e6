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
// One pass over the logits, bound by HBM: a block holds a chunk of a row in
// registers, sums its exponentials against its own maximum and keeps its K best
// logits as 64-bit keys (ordered logit, then ~token), best first.  A block per
// request then joins the chunks: the rows' log-sums, added in f64 over the
// chunks, and the K best by their f64 scores.  A chunk's own sum is f32 (differences,
// exponentials within 2^-22, their sum), so a log-sum is within about 1e-6 and
// candidates of two beams that are further apart than two such errors are told apart;
// those of one beam share its log-sum and are in the order of their logits.
//
// Selection: of any disjoint groups' maxima the K-th largest is a bound that at
// least K elements reach, so only what reaches it is looked at -- in a chunk, of
// the maxima of 64 groups of 4 lanes; in a join, of the chunks' best, or of the
// first few of each where there are not K chunks -- a few
// dozen elements, which are ranked by counting.  Where too many reach the bound (equal
// logits) the K are taken one at a time.
// Keys are unique, so nothing depends on the order in which threads arrive.
//
// Measured, calls back to back, a vocabulary of 103,424, the best 8:
//   64 x 4 beams, f32, 106 MB   25.4 us   4.2 TB/s, 64 % of a copy: 16.4 for the loads,
//     maxima and exponentials alone (a copy's rate), 0.8 for the bound, 4.1 for listing and
//     ranking, 4.1 for the join, one block a request, which is bound by the latency of its
//     chain of sums, logarithm and ranking
//   1 x 4 beams, fp16   6.6 us   two launches' latency
// A join by the block that leaves a request's last chunk, in one launch, took 38.9 us against 27.9:
// each block then holds its place on the SM for a fence and an atomic's way there and back.
// Blocks that go from chunk to chunk with the next one's loads under the ranking took 34.3
// (five an SM, whose registers then spill) and 30.4 (four).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>
#include <string.h>

#include "pvlc_common.cuh"
#include "pvlc_internal.h"

namespace pvlc {
namespace beam {

constexpr int THREADS = 256;
constexpr uint32_t LIST = 512;               // elements ranked by counting
constexpr uint32_t MAX_HEADS = 2 * THREADS;  // elements of a request that a join bounds by
constexpr int BLOCKS = 5;                    // of an SM: 27.8 us for the 64 x 4 beams, 29.2 with 4

typedef unsigned long long u64;
constexpr float kLog2e = 1.4426950408889634f;

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

__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// The K-th largest of x[0 .. n), K <= n, equal ones counting one each; all threads
// get it.  x is padded with -infinity to a multiple of 16.  Four lanes take an element.
__device__ __forceinline__ float kth_largest(const float* x, uint32_t n, uint32_t K, float* result) {
  for (uint32_t i0 = 0; i0 < n; i0 += THREADS / 4) {
    const uint32_t i = i0 + threadIdx.x / 4;
    const float mine = i < n ? x[i] : 0.f;
    uint32_t before = 0;                     // how many come ahead of it
#pragma unroll 4
    for (uint32_t j = threadIdx.x % 4 * 4; j < n; j += 16) {
      const float4 y = *reinterpret_cast<const float4*>(x + j);
      before += (y.x > mine || (y.x == mine && j < i)) + (y.y > mine || (y.y == mine && j + 1 < i)) +
                (y.z > mine || (y.z == mine && j + 2 < i)) + (y.w > mine || (y.w == mine && j + 3 < i));
    }
    before += __shfl_xor_sync(0xffffffffu, before, 1);
    before += __shfl_xor_sync(0xffffffffu, before, 2);
    if (i < n && before == K - 1) *result = mine;
  }
  __syncthreads();
  return *result;
}

// PER logits a thread; VEC: rows are 16-byte aligned.
template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS, BLOCKS) beam_chunk_kernel(const Params p) {
  constexpr uint32_t CHUNK = THREADS * PER;
  constexpr uint32_t W = 16 / sizeof(T);             // logits of one 16-byte load
  constexpr uint32_t GROUPS = THREADS / 4;           // of 4 lanes
  __shared__ __align__(16) float group_top[GROUPS];
  __shared__ float2 warp_sum[THREADS / 32];
  __shared__ float bound_out;
  __shared__ u64 list[LIST];
  __shared__ __align__(16) float handed[THREADS / 32][PER];
  __shared__ uint32_t listed;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t row = blockIdx.y, c = blockIdx.x, K = p.topk;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  // logit i of thread t is token(t, i): w neighbours a load, THREADS loads apart
  const uint32_t w = VEC && (c + 1) * CHUNK <= p.vocab ? W : 1;
  auto token = [&](uint32_t t, uint32_t i) { return c * CHUNK + (i / w * THREADS + t) * w + i % w; };
  float v[PER];
  if (w == W) {
    uint4 y[PER / W];
#pragma unroll
    for (uint32_t i = 0; i < PER / W; ++i)
      y[i] = __ldg(reinterpret_cast<const uint4*>(x + c * CHUNK + (i * THREADS + tid) * W));
#pragma unroll
    for (uint32_t i = 0; i < PER; i += W) {
      T z[W];
      memcpy(z, &y[i / W], sizeof(T) * W);
#pragma unroll
      for (uint32_t e = 0; e < W; ++e) v[i + e] = to_float(z[e]);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
      const uint32_t at = c * CHUNK + i * THREADS + tid;
      v[i] = at < p.vocab ? to_float(x[at]) : -CUDART_INF_F;
    }
  }
  if (tid == 0) listed = 0;
  float best = -CUDART_INF_F;                // the maxima pass over NaN
#pragma unroll
  for (int i = 0; i < PER; i += 2) best = fmax3(best, v[i], v[i + 1]);
  // ---- the warp's maximum and its sum of exponentials
  float m = best;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (o == 2 && lane % 4 == 0) group_top[tid / 4] = m;
  }
  float s = 0.f;
  if (m > -CUDART_INF_F) {                   // a masked token adds 2^-infinity
    const uint64_t shift = f2_pack(-m, -m), unit = f2_pack(kLog2e, kLog2e);
    uint64_t sum = f2_pack(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
      const float2 y = f2_unpack(f2_mul(f2_add(f2_pack(v[i], v[i + 1]), shift), unit));
      sum = f2_add(sum, f2_pack(fast_exp2(y.x), fast_exp2(y.y)));
    }
    const float2 both = f2_unpack(sum);
    s = both.x + both.y;
    if (isnan(s) && m < CUDART_INF_F) {      // a NaN counts as -infinity
      s = 0.f;
#pragma unroll 1
      for (uint32_t i = 0; i < PER; ++i) {
        const float y = token(tid, i) < p.vocab ? to_float(x[token(tid, i)]) : -CUDART_INF_F;
        if (y > -CUDART_INF_F) s += fast_exp2((y - m) * kLog2e);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) warp_sum[warp] = make_float2(m, s);
  __syncthreads();
  // ---- what reaches the K-th largest group maximum
  const size_t slot = (size_t)row * p.chunks + c;
  u64* keys = p.keys + slot * K;
  const float bound = kth_largest(group_top, GROUPS, K, &bound_out);
  auto key_of = [](float y, uint32_t at) -> u64 { return (u64)ordered(y) << 32 | (0xffffffffu - at); };
  // The warp looks at each thread that has something together, one of its logits a lane,
  // handed over through shared memory: as unrolled code on registers this rare work took
  // longer to fetch than to run.  Masked logits are left to the end.
  uint32_t found = __ballot_sync(0xffffffffu, best >= bound && best > -CUDART_INF_F);
  while (found) {
    const uint32_t who = __ffs(found) - 1;
    found &= found - 1;
    if (lane == who) {
#pragma unroll
      for (int i = 0; i < PER; i += 4)
        *reinterpret_cast<float4*>(handed[warp] + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
    __syncwarp();
    const float y = lane < PER ? handed[warp][lane] : -CUDART_INF_F;
    if (y >= bound && y > -CUDART_INF_F) {
      const uint32_t to = atomicAdd(&listed, 1);
      if (to < LIST) list[to] = key_of(y, token(warp * 32 + who, lane));
    }
    __syncwarp();
  }
  __syncthreads();
  // the last warp joins the sums while the first ones rank: both chains are long
  if (warp == THREADS / 32 - 1) {
    const float2 x = lane < THREADS / 32 ? warp_sum[lane] : make_float2(-CUDART_INF_F, 0.f);
    float top = x.x;
#pragma unroll
    for (int o = THREADS / 64; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float all = x.x > -CUDART_INF_F ? x.y * fast_exp2((x.x - top) * kLog2e) : 0.f;
#pragma unroll
    for (int o = THREADS / 64; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) p.sums[slot] = make_float2(top, all);
  }
  const uint32_t n = listed;
  if (n <= LIST) {
    for (uint32_t i = tid; i < n; i += THREADS) {
      const u64 mine = list[i];
      uint32_t rank = 0;
#pragma unroll 8
      for (uint32_t j = 0; j < n; ++j) rank += list[j] > mine;
      if (rank < K) keys[rank] = mine;
    }
    if (n < K && warp == 0) {                // then the first masked ones, then none
      uint32_t have = n;
      const uint32_t end = min(p.vocab, (c + 1) * CHUNK);
      for (uint32_t at = c * CHUNK + lane; have < K && at - lane < end; at += 32) {
        const bool masked = at < end && !(to_float(x[at]) > -CUDART_INF_F);
        const uint32_t all = __ballot_sync(0xffffffffu, masked);
        const uint32_t rank = have + __popc(all & ((1u << lane) - 1));
        if (masked && rank < K) keys[rank] = key_of(-CUDART_INF_F, at);
        have += __popc(all);
      }
      for (uint32_t k = have + lane; k < K; k += 32) keys[k] = 0;
    }
    return;
  }
  u64 top = ~0ull;
  for (uint32_t k = 0; k < K; ++k) {
    u64 next = 0;                            // below every logit's key; 0 also where logits run out
#pragma unroll 8
    for (uint32_t i = 0; i < PER; ++i) {
      const uint32_t at = token(tid, i);
      const u64 key = at < p.vocab ? key_of(to_float(x[at]), at) : 0;
      if (key < top && key > next) next = key;
    }
    top = block_max(next);
    if (tid == 0) keys[k] = top;
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
  __shared__ double list_score[LIST];
  __shared__ u64 list_key[LIST];
  __shared__ uint32_t list_beam[LIST];
  __shared__ __align__(16) float head_score[MAX_HEADS];
  __shared__ float bound_out;
  __shared__ uint32_t listed;
  const uint32_t r = blockIdx.x, W = p.beams, K = p.topk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the first `each` of every chunk bound the rest: at least K of them
  const uint32_t per = p.chunks * K, chunks = W * p.chunks, n = W * per;
  const uint32_t each = chunks < K ? (K + chunks - 1) / chunks : 1, heads = chunks * each;
  const u64* keys = p.keys + (size_t)r * n;
  const bool bounded = heads <= MAX_HEADS;
  auto chunk_of = [&](uint32_t i) { return each == 1 ? i : i / each; };
  if (threadIdx.x == 0) listed = 0;
  pdl_wait();
  pdl_launch_dependents();
  // this thread's first keys and what follows them, in flight under the log-sums
  constexpr uint32_t EARLY = 2;
  u64 mine[2][EARLY];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k) {
      const uint32_t i = threadIdx.x + e * THREADS;
      const uint32_t chunk = chunk_of(i), at = i - chunk * each + k;
      mine[e][k] = bounded && i < heads && at < K ? keys[(size_t)chunk * K + at] : 0;
    }
  for (uint32_t w = warp; w < W; w += THREADS / 32) {
    const float2* s = p.sums + (size_t)(r * W + w) * p.chunks;
    const float score = p.scores[r * W + w];
    float m = -CUDART_INF_F;
    double t = 0.0;                        // against m, rescaled where m grows
    for (uint32_t c0 = 0; c0 < p.chunks; c0 += 32) {
      const float2 x = c0 + lane < p.chunks ? s[c0 + lane] : make_float2(-CUDART_INF_F, 0.f);
      float top = x.x;
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (top > m) {
        if (m > -CUDART_INF_F) t *= (double)expf(m - top);
        m = top;
      }
      if (x.x > -CUDART_INF_F) t += (double)x.y * (double)expf(x.x - m);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) base[w] = (double)score - ((double)m + log(t));
  }
  __syncthreads();
  auto made = [&](u64 key, uint32_t beam) {
    Cand c;
    c.key = key;
    c.beam = beam;
    c.score = base[beam] + (double)from_ordered((uint32_t)(key >> 32));
    if (isnan(c.score)) c.score = -CUDART_INF;
    return c;
  };
  auto candidate = [&](uint32_t i) { return made(keys[i], i / per); };
  auto write = [&](uint32_t k, const Cand& c) {
    const size_t at = (size_t)r * K + k;
    p.out_score[at] = (float)c.score;
    p.out_beam[at] = (int32_t)c.beam;
    p.out_token[at] = (int32_t)(0xffffffffu - (uint32_t)c.key);
  };
  if (bounded) {
    // scores rounded down to f32: at least K of the first ones reach the K-th largest of them
    float score[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = threadIdx.x + e * THREADS;
      score[e] = i < heads ? __double2float_rd(made(mine[e][0], chunk_of(i) / p.chunks).score) : -CUDART_INF_F;
      head_score[i] = score[e];
    }
    __syncthreads();
    const float bound = kth_largest(head_score, heads, K, &bound_out);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t i = threadIdx.x + e * THREADS;
      if (i >= heads || !(score[e] >= bound)) continue;
      auto add = [&](const Cand& c) {        // a chunk's list is in order: false behind the last
        if (c.key == 0 || c.score < (double)bound) return false;
        const uint32_t at = atomicAdd(&listed, 1);
        if (at < LIST) {
          list_score[at] = c.score;
          list_key[at] = c.key;
          list_beam[at] = c.beam;
        }
        return true;
      };
      const uint32_t chunk = chunk_of(i), at = i - chunk * each, beam = chunk / p.chunks;
      bool more = add(made(mine[e][0], beam)) && at == each - 1;      // the last of them goes on
#pragma unroll
      for (uint32_t k = 1; k < EARLY; ++k) more = more && add(made(mine[e][k], beam));
      for (uint32_t k = at + EARLY; k < K && more; ++k) more = add(candidate(chunk * K + k));
    }
    __syncthreads();
    const uint32_t found = listed;
    if (found <= LIST) {
      for (uint32_t i = threadIdx.x; i < found; i += THREADS) {
        const Cand c{list_score[i], list_beam[i], list_key[i]};
        uint32_t rank = 0;                   // how many are before() it
#pragma unroll 4
        for (uint32_t j = 0; j < found; ++j) {
          const bool same = list_score[j] == c.score, beam = list_beam[j] == c.beam;
          rank += (list_score[j] > c.score) |
                  (same & ((list_beam[j] < c.beam) | (beam & (list_key[j] > c.key))));
        }
        if (rank < K) write(rank, c);
      }
      return;
    }
  }
  Cand last;
  last.key = 0;
  for (uint32_t k = 0; k < K; ++k) {
    Cand best;
    best.key = 0;
    best.score = 0.0;
    best.beam = 0;
    for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
      const Cand c = candidate(i);
      if (c.key != 0 && (k == 0 || before(last, c)) && before(c, best)) best = c;
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
    if (threadIdx.x == 0) write(k, best);
  }
}

// Logits a thread.  A chunk costs about 2 us beside its loads, so 32, as many as the registers
// of five blocks an SM hold: 64 x 4 beams took 27.6 us, with 16 and seven blocks 32.1, with 8
// 67.9, when all were tried; 4 x 4 beams 8.7, 9.1, 15.3.  Where such chunks would leave half the SMs without one, 16:
// one row takes 6.4 us against 7.7, 1 x 4 beams 7.2 against 7.6, but 2 x 4 beams 8.2 against 7.7.
uint32_t per_thread(uint32_t rows, uint32_t vocab) {
  const uint64_t wide = (vocab + THREADS * 32 - 1) / (THREADS * 32);
  return 2 * rows * wide < (uint32_t)sms_or_default_count() ? 16 : 32;
}
uint32_t chunks_of(uint32_t rows, uint32_t vocab) {
  const uint32_t chunk = THREADS * per_thread(rows, vocab);
  return (vocab + chunk - 1) / chunk;
}

template <typename T, bool VEC>
cudaError_t launch_chunks(const Params& p, uint32_t per, const cudaLaunchConfig_t& cfg) {
  return per == 16 ? cudaLaunchKernelEx(&cfg, beam_chunk_kernel<T, 16, VEC>, p)
                   : cudaLaunchKernelEx(&cfg, beam_chunk_kernel<T, 32, VEC>, p);
}

}  // namespace beam

size_t beam_topk_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t topk) {
  // enough for every call of these sizes or smaller ones: fewer rows may have chunks of half
  // the size, at most two for each wide one, as long as those are below half the SMs
  const size_t rows = (size_t)batch * beams;
  const size_t wide = (vocab + beam::THREADS * 32 - 1) / (beam::THREADS * 32);
  const size_t few = (size_t)sms_or_default_count(), low = 2 * rows * wide < few ? 2 * rows * wide : few;
  const size_t slots = rows * wide > low ? rows * wide : low;
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
  const uint32_t rows = a.batch * a.beams, per = beam::per_thread(rows, a.vocab);
  p.chunks = beam::chunks_of(rows, a.vocab);
  p.keys = static_cast<beam::u64*>(a.workspace);
  p.sums = reinterpret_cast<float2*>(p.keys + (size_t)rows * p.chunks * a.topk);
  p.out_score = a.out_score;
  p.out_beam = a.out_beam;
  p.out_token = a.out_token;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.chunks, rows);
  cfg.blockDim = dim3(beam::THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
                   a.ld % (a.half_logits ? 8 : 4) == 0;
  const cudaError_t e =
      a.half_logits ? (vec ? beam::launch_chunks<__half, true>(p, per, cfg)
                           : beam::launch_chunks<__half, false>(p, per, cfg))
                    : (vec ? beam::launch_chunks<float, true>(p, per, cfg)
                           : beam::launch_chunks<float, false>(p, per, cfg));
  if (e != cudaSuccess) return PVLC_CUDA_ERROR;
  cfg.gridDim = dim3(a.batch);
  return cudaLaunchKernelEx(&cfg, beam::beam_join_kernel, p) == cudaSuccess ? PVLC_OK
                                                                            : PVLC_CUDA_ERROR;
}

}  // namespace pvlc
