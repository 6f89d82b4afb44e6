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
// One pass over the logits, bound by HBM: all rows' chunks of 8192 are laid end
// to end and cut into equal ranges, one per block.  A block's threads each
// stream their own 32 logits of a chunk through two cp.async stages, keep a running maximum and sum of exponentials, and push what may be among the
// K best of the row into a list.  Per part of a row the block leaves its sum and
// its K best logits as 64-bit keys (ordered logit, then ~token), best first.  A
// block per request joins the parts: the rows' log-sums in f64, so that candidates
// of two beams that differ by more than 1e-7 are told apart, and the K best.
//
// Selection: of any disjoint groups' maxima the K-th largest is a bound that at
// least K elements reach, so only what reaches it is looked at -- in a row's first
// chunk (and in one that raises the level), of the maxima of 8 .. 64 groups of
// lanes; in a join, of the parts' best -- a few dozen elements, which are ranked
// by counting.  A ranked list's K-th key is the bound of the chunks that follow.
// Where too many reach the bound (equal or masked logits) the K are taken one at
// a time.
// Keys are unique, so nothing depends on the order in which threads arrive.
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
constexpr int PER = 32;                      // logits of a chunk a thread (and a warp's lanes)
constexpr uint32_t CHUNK = THREADS * PER;
constexpr int BLOCKS = 3;                    // of an SM
constexpr uint32_t LIST = 512;               // elements ranked by counting
constexpr uint32_t MAX_HEADS = 2 * THREADS;  // parts of a request that a join bounds by

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
  uint32_t batch, beams, vocab, topk;
  uint32_t chunks;    // of a row
  uint32_t blocks;    // of the chunk kernel
  uint32_t parts;     // most blocks that share a row
  u64* keys;          // [rows][parts][topk]
  float2* sums;       // [rows][parts] (maximum, sum of exponentials against it)
  uint32_t* counts;   // [rows] how many parts the row has
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
// get it.  x is padded with -infinity to a multiple of 4.
__device__ __forceinline__ float kth_largest(const float* x, uint32_t n, uint32_t K, float* result) {
  for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
    const float mine = x[i];
    uint32_t above = 0, equal_before = 0;
    for (uint32_t j = 0; j < n; j += 4) {
      const float4 y = *reinterpret_cast<const float4*>(x + j);
      above += (y.x > mine) + (y.y > mine) + (y.z > mine) + (y.w > mine);
      equal_before += (y.x == mine && j < i) + (y.y == mine && j + 1 < i) +
                      (y.z == mine && j + 2 < i) + (y.w == mine && j + 3 < i);
    }
    if (above + equal_before == K - 1) *result = mine;
  }
  __syncthreads();
  return *result;
}

// Block i's chunks are [cut(i), cut(i + 1)) of the rows' chunks end to end.
__host__ __device__ __forceinline__ uint64_t cut(const Params& p, uint64_t i) {
  const uint64_t x = i * ((uint64_t)p.batch * p.beams * p.chunks);
  return x >> 32 ? x / p.blocks : (uint32_t)x / p.blocks;
}
// The block that holds chunk u.
__device__ __forceinline__ uint32_t block_of(const Params& p, uint64_t u) {
  const uint64_t n = (uint64_t)p.batch * p.beams * p.chunks, x = (u + 1) * p.blocks + n - 1;
  return (uint32_t)(x >> 32 ? x / n : (uint32_t)x / (uint32_t)n) - 1;
}

// VEC: rows are 16-byte aligned.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS, BLOCKS) beam_chunk_kernel(const Params p) {
  constexpr int W = 16 / sizeof(T);                  // logits of one 16-byte piece
  constexpr int PIECES = PER / W;
  extern __shared__ __align__(16) uint8_t ring[];    // [2][PIECES][THREADS] x 16 bytes
  __shared__ __align__(16) float group_top[64];
  __shared__ float bound_out;
  __shared__ u64 list[LIST];
  __shared__ u64 best_keys[PVLC_BEAM_MAX_TOPK];
  __shared__ uint32_t listed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t K = p.topk;
  pdl_wait();
  pdl_launch_dependents();
  const uint64_t u0 = cut(p, blockIdx.x), u1 = cut(p, blockIdx.x + 1);
  // v[i] of chunk c is token(c, i): pieces of W neighbours, THREADS pieces apart
  auto token = [&](uint32_t c, int i) { return c * CHUNK + (i / W * THREADS + tid) * W + i % W; };
  uint32_t next_row = (uint32_t)(u0 / p.chunks), next_chunk = (uint32_t)(u0 % p.chunks);
  uint64_t next = u0;
  // Start this thread's copies of the next chunk.  Only the thread itself reads them.
  auto fetch = [&](uint32_t stage) {
    if (next < u1) {
      const T* x = static_cast<const T*>(p.logits) + next_row * p.ld;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        uint8_t* to = ring + ((stage * PIECES + i) * THREADS + tid) * 16;
        const uint32_t at = token(next_chunk, i * W);
        if (VEC && at + W <= p.vocab) {
          cp_async_16(smem_u32(to), x + at);
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e)    // behind the row: masked
            reinterpret_cast<T*>(to)[e] = at + e < p.vocab ? x[at + e] : T(-CUDART_INF_F);
        }
      }
      if (++next_chunk == p.chunks) {
        next_chunk = 0;
        ++next_row;
      }
      ++next;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(0);

  uint32_t row = (uint32_t)(u0 / p.chunks), c = (uint32_t)(u0 % p.chunks), stage = 0;
  uint32_t from = c;                     // the row's first chunk in this block
  float m = -CUDART_INF_F, s = 0.f;      // this thread's, of the row so far
  u64 bound = 0;                         // only larger keys matter
  uint32_t kept = 0;                     // keys in the list, at most LIST / 4
  bool first = true;
  if (tid == 0) listed = 0;
  __syncthreads();
  // The list's K best, in order, become the list; the K-th is the bound.
  auto rank_list = [&]() {
    const uint32_t n = listed;           // at most LIST
    for (uint32_t i = tid; i < n; i += THREADS) {
      const u64 mine = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; ++j) rank += list[j] > mine;
      if (rank < K) best_keys[rank] = mine;
    }
    __syncthreads();
    kept = n < K ? n : K;
    for (uint32_t i = tid; i < kept; i += THREADS) list[i] = best_keys[i];
    if (tid == 0) listed = kept;
    if (kept == K) bound = best_keys[K - 1];
    __syncthreads();
  };
  for (uint64_t u = u0; u < u1; ++u) {
    fetch(stage ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    float v[PER];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const uint4 y = reinterpret_cast<const uint4*>(ring)[(stage * PIECES + i) * THREADS + tid];
      T z[W];
      memcpy(z, &y, 16);
#pragma unroll
      for (int e = 0; e < W; ++e) v[i * W + e] = to_float(z[e]);
    }
    float best = -CUDART_INF_F;          // the maxima pass over NaN
#pragma unroll
    for (int i = 0; i < PER; i += 2) best = fmax3(best, v[i], v[i + 1]);
    if (best > m) {
      s *= fast_exp2((m - best) * kLog2e);
      m = best;
    }
    if (m > -CUDART_INF_F) {             // a masked token adds 2^-infinity
      const uint64_t shift = f2_pack(-m, -m), unit = f2_pack(kLog2e, kLog2e);
      uint64_t sum = f2_pack(s, 0.f);
#pragma unroll
      for (int i = 0; i < PER; i += 2) {
        const float2 x = f2_unpack(f2_mul(f2_add(f2_pack(v[i], v[i + 1]), shift), unit));
        sum = f2_add(sum, f2_pack(fast_exp2(x.x), fast_exp2(x.y)));
      }
      const float2 both = f2_unpack(sum);
      s = both.x + both.y;
    }
    // The rare work on single logits reads them again: the code stays small, and with
    // it the time to fetch its instructions (unrolled, it cost 5 us a chunk).
    const uint32_t now = stage;
    auto each = [&](auto f) {              // f(ordered logit, token)
#pragma unroll 1
      for (int i = 0; i < PIECES; ++i) {
        const uint4 y = reinterpret_cast<const uint4*>(ring)[(now * PIECES + i) * THREADS + tid];
        const uint32_t at = token(c, i * W);
        T z[W];
        memcpy(z, &y, 16);
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (at + e < p.vocab) f(to_float(z[e]), at + e);
      }
    };
    auto key_of = [](float x, uint32_t at) -> u64 { return (u64)ordered(x) << 32 | (0xffffffffu - at); };
    // a float that every key above the bound reaches (0 bounds nothing)
    const float level = bound ? from_ordered((uint32_t)(bound >> 32)) : -CUDART_INF_F;
    const int reach = __syncthreads_count(best >= level && (best > -CUDART_INF_F || bound == 0));
    if (reach) {
      bool singly = false;
      u64 bar = bound;
      if (reach > THREADS / 4) {
        // raise the bound by this chunk's groups: 32 lanes for K <= 8, .. 4 lanes for K <= 64
        const uint32_t split = K <= 8 ? 1 : K <= 16 ? 2 : K <= 32 ? 4 : 8, size = 32 / split;
        float top = best;
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
          const float y = __shfl_xor_sync(0xffffffffu, top, o);
          if (o < size) top = fmaxf(top, y);
        }
        if (lane % size == 0) group_top[warp * split + lane / size] = top;
        __syncthreads();
        const float kth = kth_largest(group_top, THREADS / 32 * split, K, &bound_out);
        if (kth > -CUDART_INF_F) {
          const u64 key = ((u64)ordered(kth) << 32) - 1;
          bar = key > bar ? key : bar;
        } else {
          singly = true;                 // fewer than K groups hold anything
        }
      }
      if (!singly) {
        const float lowest = bar ? from_ordered((uint32_t)(bar >> 32)) : -CUDART_INF_F;
        // the warp looks at each such thread's logits together, one a lane
        uint32_t found = __ballot_sync(0xffffffffu, best >= lowest);
        while (found) {
          const int who = warp * 32 + __ffs(found) - 1;
          found &= found - 1;
          const int piece = lane / W;
          const uint32_t at = c * CHUNK + (piece * THREADS + who) * W + lane % W;
          const float x = to_float(reinterpret_cast<const T*>(
              ring + ((now * PIECES + piece) * THREADS + who) * 16)[lane % W]);
          if (x >= lowest && at < p.vocab) {
            const u64 key = key_of(x, at);
            if (key > bar) {
              const uint32_t to = atomicAdd(&listed, 1);
              if (to < LIST) list[to] = key;
            }
          }
        }
        __syncthreads();
        singly = listed > LIST;
      }
      if (singly) {
        // too many: this chunk's K best one by one behind the row's
        u64 top = ~0ull;
        uint32_t n = kept;
        for (uint32_t k = 0; k < K; ++k) {
          u64 after = 0;                 // 0: the chunk's logits have run out
          each([&](float x, uint32_t at) {
            const u64 key = key_of(x, at);
            if (key < top && key > after) after = key;
          });
          top = block_max(after);
          if (top <= bound) break;
          if (tid == 0) list[n] = top;
          ++n;
        }
        if (tid == 0) listed = n;
        __syncthreads();
      }
      kept = listed;
      if (first || kept > LIST / 4) rank_list();
      first = false;
    }
    stage ^= 1;
    if (++c == p.chunks || u + 1 == u1) {
      // ------------------------------------------- the part's record
      rank_list();
      float top = m;
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) group_top[warp] = top;
      __syncthreads();
      top = group_top[0];
#pragma unroll
      for (int w = 1; w < THREADS / 32; ++w) top = fmaxf(top, group_top[w]);
      float sum = block_sum(m > -CUDART_INF_F ? s * fast_exp2((m - top) * kLog2e) : 0.f);
      if (isnan(sum) && top < CUDART_INF_F) {
        // NaN among the logits: they count as -infinity, so sum the part again without them
        s = 0.f;
        const T* x = static_cast<const T*>(p.logits) + row * p.ld;
#pragma unroll 1
        for (uint32_t at = from * CHUNK + tid; at < min(c * CHUNK, p.vocab); at += THREADS)
          if (to_float(x[at]) > -CUDART_INF_F) s += fast_exp2((to_float(x[at]) - top) * kLog2e);
        sum = block_sum(s);
      }
      const uint32_t part = blockIdx.x - block_of(p, (uint64_t)row * p.chunks);
      const size_t slot = (size_t)row * p.parts + part;
      if (tid == 0) {
        p.sums[slot] = make_float2(top, sum);
        if (c == p.chunks) p.counts[row] = part + 1;
      }
      const uint32_t n = listed;
      for (uint32_t k = tid; k < K; k += THREADS) p.keys[slot * K + k] = k < n ? list[k] : 0;
      __syncthreads();
      if (tid == 0) listed = 0;
      __syncthreads();
      kept = 0;
      m = -CUDART_INF_F;
      s = 0.f;
      bound = 0;
      first = true;
      c = from = 0;
      ++row;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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
  __shared__ Cand list[LIST];
  __shared__ __align__(16) float head_score[MAX_HEADS];
  __shared__ float bound_out;
  __shared__ uint32_t listed;
  const uint32_t r = blockIdx.x, W = p.beams, K = p.topk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t P = p.parts, heads = W * P;          // at most MAX_HEADS
  const u64* keys = p.keys + (size_t)r * heads * K;
  __shared__ uint32_t parts[PVLC_BEAM_MAX_BEAMS];    // that each row has
  if (threadIdx.x == 0) listed = 0;
  pdl_wait();
  pdl_launch_dependents();
  // this thread's parts' first keys (of parts that are there or not), in flight under the log-sums
  constexpr uint32_t EARLY = 4;
  u64 mine[2][EARLY];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k) {
      const uint32_t i = threadIdx.x + e * THREADS;
      mine[e][k] = i < heads && k < K ? keys[(size_t)i * K + k] : 0;
    }
  for (uint32_t w = warp; w < W; w += THREADS / 32) {
    const float2* s = p.sums + (size_t)(r * W + w) * P;
    const float2 lead = lane < P ? s[lane] : make_float2(0.f, 0.f);
    const uint32_t count = p.counts[r * W + w];
    const float score = p.scores[r * W + w];
    float m = -CUDART_INF_F;
    double t = 0.0;                        // against m, rescaled where m grows
    for (uint32_t c0 = 0; c0 < count; c0 += 32) {
      const float2 x = c0 + lane < count ? (c0 ? s[c0 + lane] : lead) : make_float2(-CUDART_INF_F, 0.f);
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
    if (lane == 0) {
      base[w] = (double)score - ((double)m + log(t));
      parts[w] = count;
    }
  }
  __syncthreads();
  auto there = [&](uint32_t i) { return i < heads && i % P < parts[i / P]; };   // part i of the request
  auto made = [&](u64 key, uint32_t beam) {
    Cand c;
    c.key = key;
    c.beam = beam;
    c.score = base[beam] + (double)from_ordered((uint32_t)(key >> 32));
    if (isnan(c.score)) c.score = -CUDART_INF;
    return c;
  };
  // candidate k of part i
  auto candidate = [&](uint32_t i, uint32_t k) { return made(keys[(size_t)i * K + k], i / P); };
  auto write = [&](uint32_t k, const Cand& c) {
    const size_t at = (size_t)r * K + k;
    p.out_score[at] = (float)c.score;
    p.out_beam[at] = (int32_t)c.beam;
    p.out_token[at] = (int32_t)(0xffffffffu - (uint32_t)c.key);
  };
  // scores rounded down to f32: at least K parts' best reach the K-th largest of them (where
  // there are fewer parts it is -infinity, and everything does)
  float score[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t i = threadIdx.x + e * THREADS;
    score[e] = there(i) ? __double2float_rd(made(mine[e][0], i / P).score) : -CUDART_INF_F;
    head_score[i] = score[e];
  }
  __syncthreads();
  const float bound =
      heads >= K ? kth_largest(head_score, heads, K, &bound_out) : -CUDART_INF_F;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t i = threadIdx.x + e * THREADS;
    if (!there(i) || !(score[e] >= bound)) continue;
    auto add = [&](const Cand& c) {          // a part's list is in order: false behind the last
      if (c.key == 0 || c.score < (double)bound) return false;
      const uint32_t at = atomicAdd(&listed, 1);
      if (at < LIST) list[at] = c;
      return true;
    };
    bool more = true;
#pragma unroll
    for (uint32_t k = 0; k < EARLY; ++k) more = more && add(made(mine[e][k], i / P));
    for (uint32_t k = EARLY; k < K && more; ++k) more = add(candidate(i, k));
  }
  __syncthreads();
  const uint32_t found = listed;
  if (found <= LIST) {
    for (uint32_t i = threadIdx.x; i < found; i += THREADS) {
      const Cand c = list[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < found; ++j) rank += before(list[j], c);
      if (rank < K) write(rank, c);
    }
    return;
  }
  Cand last;
  last.key = 0;
  for (uint32_t k = 0; k < K; ++k) {
    Cand best;
    best.key = 0;
    best.score = 0.0;
    best.beam = 0;
    for (uint32_t i = threadIdx.x; i < heads * K; i += THREADS) {
      if (!there(i / K)) continue;
      const Cand c = candidate(i / K, i % K);
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

// How the rows' chunks are shared out: BLOCKS blocks an SM, or fewer where a
// request would get more parts than its join can bound by.
void share(Params& p) {
  const uint64_t rows = (uint64_t)p.batch * p.beams;
  p.chunks = (p.vocab + CHUNK - 1) / CHUNK;
  const uint64_t units = rows * p.chunks;
  uint64_t blocks = (uint64_t)BLOCKS * sms_or_default_count();
  if (blocks > units) blocks = units;
  while (true) {
    const uint64_t q = units / blocks;             // every block has that many chunks or more
    const uint64_t parts = (p.chunks - 1) / q + 2;
    p.parts = (uint32_t)(parts < p.chunks ? parts : p.chunks);
    if (p.parts * p.beams <= MAX_HEADS) break;
    blocks = blocks * 7 / 8;                       // at `rows` blocks a row has 2 parts at most
  }
  p.blocks = (uint32_t)blocks;
}

template <typename T, bool VEC>
int launch_chunks(const Params& p, cudaLaunchConfig_t cfg) {
  cfg.gridDim = dim3(p.blocks);
  cfg.dynamicSmemBytes = 2 * CHUNK * sizeof(T);
  const void* fn = reinterpret_cast<const void*>(beam_chunk_kernel<T, VEC>);
  if (const int st = set_smem_attribute_once(fn, 2 * CHUNK * sizeof(T))) return st;
  return cudaLaunchKernelEx(&cfg, beam_chunk_kernel<T, VEC>, p) == cudaSuccess ? PVLC_OK
                                                                                : PVLC_CUDA_ERROR;
}

}  // namespace beam

size_t beam_topk_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t topk) {
  // Enough for every call of these sizes or smaller ones: rows x parts is at most rows x chunks,
  // and at most 2 BLOCKS an SM and 2 a row (every block has a chunk; where it has q >= 2, a row has
  // chunks / q + 2 parts and chunks / q is below 3 / 2 of the blocks per row).
  const size_t rows = (size_t)batch * beams;
  const size_t chunks = (vocab + beam::CHUNK - 1) / beam::CHUNK;
  const size_t most = 2 * (size_t)beam::BLOCKS * sms_or_default_count() + 2 * rows;
  const size_t slots = rows * chunks < most ? rows * chunks : most;
  return (slots * (topk + 1) * 8 + rows * 4 + 255) / 256 * 256;
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
  beam::share(p);
  const size_t rows = (size_t)a.batch * a.beams;
  p.keys = static_cast<beam::u64*>(a.workspace);
  p.sums = reinterpret_cast<float2*>(p.keys + rows * p.parts * a.topk);
  p.counts = reinterpret_cast<uint32_t*>(p.sums + rows * p.parts);
  if (rows * p.parts * (a.topk + 1) * 8 + rows * 4 > beam_topk_workspace_bytes(a.batch, a.beams, a.vocab, a.topk))
    return PVLC_WORKSPACE_TOO_SMALL;
  p.out_score = a.out_score;
  p.out_beam = a.out_beam;
  p.out_token = a.out_token;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(beam::THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 &&
                   a.ld % (a.half_logits ? 8 : 4) == 0;
  const int st = a.half_logits ? (vec ? beam::launch_chunks<__half, true>(p, cfg)
                                      : beam::launch_chunks<__half, false>(p, cfg))
                               : (vec ? beam::launch_chunks<float, true>(p, cfg)
                                      : beam::launch_chunks<float, false>(p, cfg));
  if (st) return st;
  cfg.gridDim = dim3(a.batch);
  return cudaLaunchKernelEx(&cfg, beam::beam_join_kernel, p) == cudaSuccess ? PVLC_OK
                                                                            : PVLC_CUDA_ERROR;
}

}  // namespace pvlc
