// kv8_decode.cu -- one token of every sequence against the 8-bit paged cache,
// with the decode M-RoPE and the append fused.
//
// Per sequence with n rows before the append: q and the new key are rotated
// at rope_row; the rotated key and the value become row n % 32 of the tail;
// attention runs over the n / 32 full pages (8 bits) and the 1 .. 32 tail rows
// (fp16); a tail that is now full is quantised into page table[slot][n / 32].
//   s_r = scale_K(r) (q . k_r) / sqrt(128),   out = sum_r softmax(s)_r scale_V(r) v_r
//
// The scales never touch a matrix operand.  scale_K multiplies the f32 scores
// of a page.  scale_V goes into the exponent: with t_r = s_r log2(e) +
// log2(scale_V(r)) and M the running maximum of t,
//   w_r = 2^(t_r - M + 14)   (fp16, at most 2^14, kept down to 2^-24: 2^-38 of the largest)
//   O = sum_r w_r code_r,    L = sum_r w_r / scale_V(r),    out = O / L,
// so the codes go to the tensor cores as the fp16 numbers they are.
//
// Bound by HBM: 2 x 128 bytes a row and KV head, 16 operations a byte at a
// group of 8.  That is 6 % of the tensor cores' rate, so mma.sync on registers,
// which needs no second copy of the codes, is enough (their pipe is active 15 % of
// the time).  Measured, a layer of 16 query and 2 KV heads, calls back to back:
//   64 sequences of 606 .. 8,011 rows   34.2 us   4.3 TB/s, 65 % of a copy
//   16 sequences, 8 KV heads, 4 k .. 8 k rows   37.9 us   4.8 TB/s, 72 %
//   64 x 4 beams of 1,248 .. 1,499 rows   46.0 us   190 MB through L2, 55 MB of them distinct
//   1 sequence of 1,023 rows   9.5 us   bound by its chain of dependent loads
// Of the 34.2 us 22.3 are the stream at a copy's rate.  4 pass before the first
// page lands (launch, the sequences' slots, lengths and page ids, each read after
// the other), 3 in joining the split units, the rest in the uneven end: without
// its arithmetic the kernel takes 32.3, without its pages 28.7.  The beams are
// bound by the warps' arithmetic, a page's 48 matrix and some 630 other
// instructions, each waiting for the one ahead of it more than for a pipe: 31.0
// and 43.6 (int8, whose conversions are a byte permutation and a subtraction).
// More warps an SM do not help (5, 6 and 8 a block: 49, 48 and 56), nor does
// loading a page that four beams share once, a warp a beam (65: the same work in
// more code).
// What the design does about it:
//   * The (sequence, KV head) units, each its pages and a tail, are laid end to
//     end with an allowance for a unit's end, and cut into equal ranges, one per
//     block and two blocks per SM, whatever the lengths are.
//   * A producer warp streams pages (4 KB of K and of V codes, one TMA tile
//     each, 128-byte swizzle) through a ring of 8 KB stages, a lane per stage, so the
//     table is read a ring ahead (one lane for all: 41.7 us for the 64 sequences
//     against 37.2 then).  A page's scales follow by cp.async on the same barrier.
//   * Four consumer warps take the pages in turn, each with its own running
//     (O, M, L), so they meet only at a unit's end.
//   * The rotated q goes in as its fp16 rounding and the rest of it, two operands,
//     so the scores are exact to f32; the weights' fp16 rounding (2^-11 each, many
//     of them averaged) is the one loss before the output's own.  Root mean square
//     error 2.7e-4 relative against 64 bits, 2.1e-4 of it the output's rounding; with
//     q rounded to fp16 alone 3.4e-4.
//   * S^T = K Q^T and O^T += V^T W^T with mma.m16n8k16: the 8 query heads of a
//     group are the N side (two N tiles above 8).  The contraction order is
//     free, so a lane's 16-byte loads are whole operand fragments: 16 dims of a
//     key row, and 16 dims of four value rows whose bytes are paired with prmt.
//     Keys are permuted by pi(g) = g / 2 + 4 (g % 2) within 8 and value dims by
//     the same map of 16-dim chunks, which makes every load conflict free.
//   * A unit that spans blocks leaves a partial record per block; the last one to
//     finish joins them in block order.
//
// The rotation multiplies and adds with a rounding each (no fused
// multiply-add), so a cached key row is the plain f32 formula's, bit for bit.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <mutex>

#include "kv8.cuh"
#include "tcgen05.cuh"

namespace pvlc {
namespace kv8 {

// Consumer warps: two blocks of 4 an SM fill its registers.  64 ragged sequences take
// 34.8 us with 4, 37.5 with 5, 36.8 with 6, 46.2 with 8.
constexpr int WARPS = 4;
constexpr int THREADS = (WARPS + 2) * 32;         // + the producer and the sequence warp
constexpr int CTHREADS = WARPS * 32;
constexpr uint32_t STAGE = 8192;                  // a page's K and V codes of one head
// A unit's end, in pages: joining four warps and writing takes a block about as long as 8 pages
// do.  64 ragged sequences: 37.7 us at 1, 36.6 at 2, 35.8 at 3, 34.2 at 8, 34.0 at 12, 34.4 at 16.
constexpr uint32_t END_COST = 8;
// Least work of a block, in pages; fewer would cut short sequences into more records to join.
// 1 sequence of 1,023 rows: 11.4 us at 4, 11.8 at 8, 15.2 at 16; batches do not come near it.
constexpr uint32_t MIN_COST = 8;
constexpr int ACC_PITCH = HD + 4;
constexpr float W_SHIFT = 14.f;

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
  uint32_t q_stride, kv_stride, rope_rows, batch, group, stages;
  uint32_t* flags;
  uint32_t* tickets;
  float* records;
};

// What is wrong with sequence b (0: nothing); its rows and rope row.
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

// Two values as an fp16 pair, and what that rounds off (or cuts off, beyond
// fp16's range) as another.
__device__ __forceinline__ float in_range(float x) {      // a NaN stays one
  return x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& pair, uint32_t& rest) {
  pair = pack_half2(in_range(a), in_range(b));
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&pair));
  rest = pack_half2(a - h.x, b - h.y);
}

// The rotation of 16 dims d .. d + 15 (d a multiple of 16, below 64) of a row and their
// partners 64 above: lo cos - hi sin, hi cos + lo sin.
struct Turns {                        // the table's values
  float4 cl[4], ch[4], sl[4], sh[4];
  __device__ __forceinline__ Turns(const DecodeParams& p, uint32_t d, uint32_t r) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const size_t at = ((size_t)mrope_axis(d + 4 * e) * p.rope_rows + r) * HD + d + 4 * e;
      cl[e] = __ldg(reinterpret_cast<const float4*>(p.rope_cos + at));
      ch[e] = __ldg(reinterpret_cast<const float4*>(p.rope_cos + at + 64));
      sl[e] = __ldg(reinterpret_cast<const float4*>(p.rope_sin + at));
      sh[e] = __ldg(reinterpret_cast<const float4*>(p.rope_sin + at + 64));
    }
  }
};
struct Piece {                        // a row's values
  uint2 lo[4], hi[4];
  __device__ __forceinline__ Piece(const __half* row, uint32_t d) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = __ldg(reinterpret_cast<const uint2*>(row + d + 4 * e));
      hi[e] = __ldg(reinterpret_cast<const uint2*>(row + d + 64 + 4 * e));
    }
  }
  // put(i, x, y): pair i of the low dims, 8 + i of the high ones
  template <typename F>
  __device__ __forceinline__ void rotate(const Turns& t, F put) const {
    auto turn = [](float x, float c, float y, float s) {
      return __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    };
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 l0 = __half22float2(*reinterpret_cast<const __half2*>(&lo[e].x));
      const float2 l1 = __half22float2(*reinterpret_cast<const __half2*>(&lo[e].y));
      const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi[e].x));
      const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi[e].y));
      const float4 &c = t.cl[e], &d = t.ch[e], &s = t.sl[e], &u = t.sh[e];
      put(2 * e, turn(l0.x, c.x, -h0.x, s.x), turn(l0.y, c.y, -h0.y, s.y));
      put(2 * e + 1, turn(l1.x, c.z, -h1.x, s.z), turn(l1.y, c.w, -h1.y, s.w));
      put(2 * e + 8, turn(h0.x, d.x, l0.x, u.x), turn(h0.y, d.y, l0.y, u.y));
      put(2 * e + 9, turn(h1.x, d.z, l1.x, u.z), turn(h1.y, d.w, l1.y, u.w));
    }
  }
};

// The low / high two code bytes of a word as an fp16 pair (exact).
template <int CODE>
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  if (CODE == PVLC_KV8_E4M3) {
    uint32_t d;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(d) : "r"(w));
    return d;
  }
  // 0x6400 | u is 1024 + u for a byte u; u = code + 128
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(1152.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int CODE>
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  if (CODE == PVLC_KV8_E4M3) {
    uint32_t d;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(d) : "r"(w));
    return d;
  }
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(1152.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// A loaded word of codes as codes_lo / codes_hi take it.  (int8 keys that keep their 1152 until the
// score is made save a subtraction an operand word, but the sums then hold 1152 sum(q) beside the
// score, and lose up to ten of its bits where the q of a head have a common part.)
template <int CODE>
__device__ __forceinline__ uint32_t biased(uint32_t w) {
  return CODE == PVLC_KV8_E4M3 ? w : w ^ 0x80808080u;
}

// A consumer warp's state over one unit: O^T tiles (tile i: dims 16 chunk +
// 2 i and + 2 i + 1 on fragment rows g and g + 8; heads 2 t, 2 t + 1), the
// running maximum and this lane's share of L, per head.
template <int NT>
struct Acc {
  float o[NT][8][4];
  float m[NT][2], l[NT][2];
};

// Scores of 32 keys (fragment row g of half tile mt is key 16 mt + pi(g), g + 8
// eight above) into weights, with the running maximum; `live` keys count.
template <int NT>
__device__ __forceinline__ void weigh(float (&s)[2][NT][4], Acc<NT>& a, float kk,
                                      float off, float rsv, int key0, int live, uint32_t (&w)[2][NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float t0 = -CUDART_INF_F, t1 = -CUDART_INF_F;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float* x = s[mt][nt] + 2 * r;
        const bool on = key0 + 16 * mt + 8 * r < live;
        x[0] = on ? x[0] * kk + off : -CUDART_INF_F;
        x[1] = on ? x[1] * kk + off : -CUDART_INF_F;
        t0 = fmaxf(t0, x[0]);
        t1 = fmaxf(t1, x[1]);
      }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
    }
    if (__any_sync(0xffffffffu, t0 > a.m[nt][0] || t1 > a.m[nt][1])) {
      const float m0 = fmaxf(a.m[nt][0], t0), m1 = fmaxf(a.m[nt][1], t1);
      const float f0 = fast_exp2(a.m[nt][0] - m0), f1 = fast_exp2(a.m[nt][1] - m1);
      a.m[nt][0] = m0;
      a.m[nt][1] = m1;
      a.l[nt][0] *= f0;
      a.l[nt][1] *= f1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a.o[nt][i][0] *= f0;
        a.o[nt][i][1] *= f1;
        a.o[nt][i][2] *= f0;
        a.o[nt][i][3] *= f1;
      }
    }
    const float c0 = W_SHIFT - a.m[nt][0], c1 = W_SHIFT - a.m[nt][1];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float p0 = fast_exp2(s[mt][nt][2 * r] + c0), p1 = fast_exp2(s[mt][nt][2 * r + 1] + c1);
        a.l[nt][0] += p0 * rsv;
        a.l[nt][1] += p1 * rsv;
        w[mt][nt][r] = movmatrix_t(pack_half2(p0, p1));
      }
  }
}

// The lane's fragments of q's rounding rest, words 4 i .. 4 i + 3 of N tile nt.
__device__ __forceinline__ uint4 rest_words(const uint8_t* rest, int nt, int i) {
  return reinterpret_cast<const uint4*>(rest)[(nt * 4 + i) * 32 + (threadIdx.x & 31)];
}

// One page of codes at `st` (K, then V 4 KB above, both swizzled).
template <int CODE, int NT>
__device__ __forceinline__ void page_tile(const uint8_t* st, float sk, float sv, float qk,
                                          const uint32_t (&qf)[NT][16], const uint8_t* rest,
                                          Acc<NT>& a, int g, int t) {
  const int pi = (g >> 1) | ((g & 1) << 2);
  float s[2][NT][4], low[2][NT][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[mt][nt][e] = low[mt][nt][e] = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t wa[2][4], wb[2][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint8_t* at = st + (16 * mt + pi) * HD + (((t + 4 * j) ^ pi) << 4);
      const uint4 xa = *reinterpret_cast<const uint4*>(at);
      const uint4 xb = *reinterpret_cast<const uint4*>(at + 8 * HD);
      wa[mt][0] = xa.x, wa[mt][1] = xa.y, wa[mt][2] = xa.z, wa[mt][3] = xa.w;
      wb[mt][0] = xb.x, wb[mt][1] = xb.y, wb[mt][2] = xb.z, wb[mt][3] = xb.w;
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      uint4 r[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) r[nt] = rest_words(rest, nt, 2 * j + f);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const int i = 2 * f + e;
          const uint32_t ya = biased<CODE>(wa[mt][i]), yb = biased<CODE>(wb[mt][i]);
          const uint32_t a0 = codes_lo<CODE>(ya), a1 = codes_lo<CODE>(yb);
          const uint32_t a2 = codes_hi<CODE>(ya), a3 = codes_hi<CODE>(yb);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816(s[mt][nt], a0, a1, a2, a3, qf[nt][8 * j + 2 * i], qf[nt][8 * j + 2 * i + 1]);
            mma_16816(low[mt][nt], a0, a1, a2, a3, e ? r[nt].z : r[nt].x, e ? r[nt].w : r[nt].y);
          }
        }
    }
  }
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[mt][nt][e] += low[mt][nt][e];
  uint32_t w[2][NT][2];
  // t = s kk + log2(scale_V)
  weigh<NT>(s, a, sk * qk, __log2f(sv), __frcp_rn(sv), 0, 64, w);
  // value rows t, t + 4, t + 8, t + 12 of a half tile: keys pi(2 t), pi(2 t + 1), ..
  const uint8_t* v = st + 4096;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    uint32_t x[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * mt + t + 4 * r;
      const uint4 y = *reinterpret_cast<const uint4*>(v + row * HD + ((pi ^ (row & 7)) << 4));
      x[r][0] = biased<CODE>(y.x);
      x[r][1] = biased<CODE>(y.y);
      x[r][2] = biased<CODE>(y.z);
      x[r][3] = biased<CODE>(y.w);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
      const uint32_t y0 = __byte_perm(x[0][i >> 1], x[1][i >> 1], sel);
      const uint32_t y1 = __byte_perm(x[2][i >> 1], x[3][i >> 1], sel);
      const uint32_t a0 = codes_lo<CODE>(y0), a1 = codes_hi<CODE>(y0);
      const uint32_t a2 = codes_lo<CODE>(y1), a3 = codes_hi<CODE>(y1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        mma_16816(a.o[nt][i], a0, a1, a2, a3, w[mt][nt][0], w[mt][nt][1]);
    }
  }
}

// The open block: fp16 rows 0 .. last - 1 at kt, vt and row `last` at kn, vn.
template <int NT>
__device__ __forceinline__ void tail_tile(const uint8_t* kt, const uint8_t* vt, const uint8_t* kn,
                                          const uint8_t* vn, int last, float qk,
                                          const uint32_t (&qf)[NT][16], const uint8_t* rest,
                                          Acc<NT>& a, int g, int t) {
  const int pi = (g >> 1) | ((g & 1) << 2);
  float s[2][NT][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
    const int ra = 16 * mt + pi, rb = ra + 8;
    const uint8_t* pa = ra < last ? kt + ra * 256 : kn;
    const uint8_t* pb = rb < last ? kt + rb * 256 : kn;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const uint4 xa = *reinterpret_cast<const uint4*>(pa + (t + 4 * j) * 32 + 16 * f);
        const uint4 xb = *reinterpret_cast<const uint4*>(pb + (t + 4 * j) * 32 + 16 * f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint32_t* qq = qf[nt] + 8 * j + 4 * f;
          const uint4 r = rest_words(rest, nt, 2 * j + f);
          mma_16816(s[mt][nt], xa.x, xb.x, xa.y, xb.y, qq[0], qq[1]);
          mma_16816(s[mt][nt], xa.x, xb.x, xa.y, xb.y, r.x, r.y);
          mma_16816(s[mt][nt], xa.z, xb.z, xa.w, xb.w, qq[2], qq[3]);
          mma_16816(s[mt][nt], xa.z, xb.z, xa.w, xb.w, r.z, r.w);
        }
      }
  }
  uint32_t w[2][NT][2];
  weigh<NT>(s, a, qk, 0.f, 1.f, pi, last + 1, w);
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      uint32_t x[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * mt + t + 4 * r;
        const uint8_t* at = row < last ? vt + row * 256 : vn;
        uint4 y = *reinterpret_cast<const uint4*>(at + pi * 32 + 16 * f);
        if (row > last) y = make_uint4(0, 0, 0, 0);
        x[r][0] = y.x;
        x[r][1] = y.y;
        x[r][2] = y.z;
        x[r][3] = y.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t a0 = __byte_perm(x[0][e], x[1][e], 0x5410);
        const uint32_t a1 = __byte_perm(x[0][e], x[1][e], 0x7632);
        const uint32_t a2 = __byte_perm(x[2][e], x[3][e], 0x5410);
        const uint32_t a3 = __byte_perm(x[2][e], x[3][e], 0x7632);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_16816(a.o[nt][4 * f + e], a0, a1, a2, a3, w[mt][nt][0], w[mt][nt][1]);
      }
    }
  }
}

// A line of C cut into N ranges, the first `more` of them one longer than `each`.
struct Cuts {
  uint64_t each;
  uint32_t more;
  __device__ __forceinline__ Cuts(uint64_t C, uint32_t N) {
    each = C >> 32 ? C / N : (uint32_t)C / N;
    more = (uint32_t)(C - each * N);
  }
  __device__ __forceinline__ uint64_t begin(uint32_t i) const { return i * each + min(i, more); }
  __device__ __forceinline__ uint32_t owner(uint64_t y) const {      // the range that y is in
    const uint64_t longer = more * (each + 1);
    return (uint32_t)(y < longer ? y / (each + 1) : more + (y - longer) / each);
  }
};

struct Seq {
  uint32_t cost;     // cost position of the sequence's first unit, per KV head
  int32_t slot, rows;
  uint32_t rope;
};

template <int NT>
constexpr uint32_t record_floats() { return 8 * NT * (HD + 2); }
// acc += f x[0 .. 8)
__device__ __forceinline__ void add_scaled(float (&acc)[8], const float* x, float f) {
  const float4 a = *reinterpret_cast<const float4*>(x), b = *reinterpret_cast<const float4*>(x + 4);
  acc[0] += a.x * f;
  acc[1] += a.y * f;
  acc[2] += a.z * f;
  acc[3] += a.w * f;
  acc[4] += b.x * f;
  acc[5] += b.y * f;
  acc[6] += b.z * f;
  acc[7] += b.w * f;
}
__device__ __forceinline__ void write_out(__half* out, const float (&o)[8], float l) {
  const float r = 1.f / l;
  *reinterpret_cast<uint4*>(out) =
      make_uint4(pack_half2(o[0] * r, o[1] * r), pack_half2(o[2] * r, o[3] * r),
                 pack_half2(o[4] * r, o[5] * r), pack_half2(o[6] * r, o[7] * r));
}

// A unit that spans blocks, as this block leaves it for the join.
struct Split {
  uint32_t unit;      // b * KV heads + h
  uint32_t blocks;    // how many it spans (0: no such unit)
  uint32_t record;    // the first one's record; the others left their first
};

// The output of head i of a unit from its blocks' records, in block order: 8
// lanes take a head, lane `sub` dims 16 sub .. + 15 and every 8th record's
// maximum and sum.  A group of 4 records is read with independent loads, the
// first one before the maxima are known.
template <int NT>
__device__ __forceinline__ void join_head(const float* records, const Split& u, uint32_t i,
                                          __half* out, uint32_t sub) {
  constexpr int R = 4;
  const uint32_t n = u.blocks;
  auto record = [&](uint32_t c) {
    return records + (size_t)(c == 0 ? u.record : (u.record & ~1u) + 2 * c) * record_floats<NT>();
  };
  float4 x[R][4];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (int e = 0; e < R; ++e)
      if (base + e < n) {
        const float4* r = reinterpret_cast<const float4*>(record(base + e) + i * HD + 16 * sub);
#pragma unroll
        for (int d = 0; d < 4; ++d) x[e][d] = __ldcg(r + d);
      }
  };
  load(0);
  // lane `sub` keeps the maximum and the sum of record `sub`; a unit of more than 8 asks again
  float m_own = -CUDART_INF_F, l_own = 0.f;
  if (sub < n) {
    const float* r = record(sub) + 8 * NT * HD + i;
    m_own = __ldcg(r);
    l_own = __ldcg(r + 8 * NT);
  }
  float m = m_own;
  for (uint32_t c = sub + 8; c < n; c += 8) m = fmaxf(m, __ldcg(record(c) + 8 * NT * HD + i));
#pragma unroll
  for (int o = 4; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.f;
  float4 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = make_float4(0.f, 0.f, 0.f, 0.f);
  // the lanes of a warp may have units of different spans: they stay together
  const uint32_t most = __reduce_max_sync(0xffffffffu, n);
  for (uint32_t base = 0; base < most; base += R) {
    if (base && base % 8 == 0 && base + sub < n) {
      const float* r = record(base + sub) + 8 * NT * HD + i;
      m_own = __ldcg(r);
      l_own = __ldcg(r + 8 * NT);
    }
    const float f = base / 8 * 8 + sub < n ? fast_exp2(m_own - m) : 0.f, fl = f * l_own;
#pragma unroll
    for (int e = 0; e < R; ++e) {
      const float fe = __shfl_sync(0xffffffffu, f, base % 8 + e, 8);
      const float le = __shfl_sync(0xffffffffu, fl, base % 8 + e, 8);
      if (base + e < n) {
        l += le;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          o[d].x += x[e][d].x * fe;
          o[d].y += x[e][d].y * fe;
          o[d].z += x[e][d].z * fe;
          o[d].w += x[e][d].w * fe;
        }
      }
    }
    if (base + R < most) load(base + R);
  }
  if (n == 0) return;
  const float r = 1.f / l;
#pragma unroll
  for (int d = 0; d < 2; ++d)
    reinterpret_cast<uint4*>(out + i * HD + 16 * sub)[d] =
        make_uint4(pack_half2(o[2 * d].x * r, o[2 * d].y * r),
                   pack_half2(o[2 * d].z * r, o[2 * d].w * r),
                   pack_half2(o[2 * d + 1].x * r, o[2 * d + 1].y * r),
                   pack_half2(o[2 * d + 1].z * r, o[2 * d + 1].w * r));
}

// The units of a block's range [y0, y1): sequence b, KV head h, whose items
// [i0, i1) are the block's: item 0 is the tail, item i > 0 page i - 1.  The tail
// comes first so that its latency passes under the pages' stream.
struct Units {
  const Seq* seq;
  uint32_t B, H, b, h, np, i0, i1;
  uint64_t y0, y1, u0;
  Seq sq;
  __device__ __forceinline__ Units(const Seq* seq_, uint32_t B_, uint32_t H_, uint64_t y0_,
                                   uint64_t y1_, uint32_t b_)
      : seq(seq_), B(B_), H(H_), b(b_), y0(y0_), y1(y1_) {
    const uint32_t len = seq[b].rows / PAGE + 1 + END_COST;
    const uint64_t past = y0 - (uint64_t)seq[b].cost * H;     // below H len
    h = past >> 32 ? (uint32_t)(past / len) : (uint32_t)past / len;
    set();
  }
  __device__ __forceinline__ void set() {
    sq = seq[b];
    np = sq.rows / PAGE;
    const uint32_t len = np + 1 + END_COST;
    u0 = (uint64_t)sq.cost * H + (uint64_t)h * len;
    i0 = u0 < y0 ? (uint32_t)(y0 - u0) : 0;
    i1 = u0 < y1 ? min((uint32_t)umin64(y1 - u0, len), np + 1) : 0;
  }
  __device__ __forceinline__ bool valid() const { return b < B && u0 < y1; }
  __device__ __forceinline__ bool has_items() const { return i0 < i1; }
  __device__ __forceinline__ bool has_tail() const { return i0 == 0; }
  __device__ __forceinline__ bool whole() const { return i0 == 0 && i1 == np + 1; }
  // ring positions: a tail takes two, K and V
  __device__ __forceinline__ uint32_t positions() const {
    return has_items() ? i1 - i0 + (has_tail() ? 1 : 0) : 0;
  }
  __device__ __forceinline__ void step() {
    if (++h == H) {
      h = 0;
      do ++b; while (b < B && seq[b].slot < 0);
    }
    if (b < B) set();
  }
};

// A unit's rotated q as the consumers' fragments [NT][4][32 lanes] x 16 bytes, what it rounds
// off in the same form, then its new key and value rows.
template <int NT>
constexpr uint32_t seq_slot() { return 2 * NT * 2048 + 512; }

template <int NT>
constexpr uint32_t fixed_smem() {
  return WARPS * 8 * NT * (ACC_PITCH + 2) * 4 + 2 * seq_slot<NT>() + 64 + 64;
}

template <int CODE, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 2 : 1)
    kv8_decode_kernel(const DecodeParams p, const __grid_constant__ CUtensorMap map) {
  extern __shared__ __align__(1024) uint8_t smem[];
  // ring | unit ends [WARPS][8 NT] rows, maxima, sums | two unit slots | sequences | scales and
  // barriers of the stages
  const uint32_t S = p.stages, B = p.batch, H = p.c.heads, G = p.group;
  uint8_t* ring = smem;
  float* end_acc = reinterpret_cast<float*>(smem + S * STAGE);
  float* end_m = end_acc + WARPS * 8 * NT * ACC_PITCH;
  float* end_l = end_m + WARPS * 8 * NT;
  uint8_t* slots = reinterpret_cast<uint8_t*>(end_l + WARPS * 8 * NT);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(slots + 2 * seq_slot<NT>());   // [2]
  uint64_t* row_full = q_full + 2;                                     // [2]
  uint64_t* slot_empty = row_full + 2;                                 // [2]
  uint32_t* misc = reinterpret_cast<uint32_t*>(q_full + 8);            // [16]
  Split* splits = reinterpret_cast<Split*>(misc + 8);                  // [2]
  Seq* seq = reinterpret_cast<Seq*>(misc + 16);                        // [B + 1]
  float2* scale = reinterpret_cast<float2*>(seq + B + 1);              // [S]
  uint64_t* full = reinterpret_cast<uint64_t*>(scale + S);             // [S]
  uint64_t* empty = full + S;                                          // [S]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (uint32_t i = 0; i < S; ++i) {
      mbar_init(full + i, 2);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 32);
      mbar_init(row_full + i, 32);
      mbar_init(slot_empty + i, WARPS);
      splits[i].blocks = 0;
    }
    fence_mbar_init();
  }
  pdl_wait();
  pdl_launch_dependents();

  // ---- the line of costs: pages + 1 + END_COST for each valid sequence and head
  {
    const uint32_t per = (B + THREADS - 1) / THREADS;
    const uint32_t b0 = min(B, tid * per), b1 = min(B, b0 + per);
    uint32_t sum = 0;
    for (uint32_t b = b0; b < b1; ++b) {
      Seq s;
      s.slot = p.slot ? p.slot[b] : (int32_t)b;
      s.rows = 0;
      s.rope = 0;
      s.cost = sum;
      uint32_t bad = 0;
      if (s.slot != -1) bad = check_sequence(p, b, s.slot, &s.rows, &s.rope);
      if (bad) {
        s.slot = -1;
        if (b % gridDim.x == blockIdx.x) {
          atomicOr(p.flags, bad);
          uint4* o = reinterpret_cast<uint4*>(p.out + (size_t)b * G * H * HD);
          for (uint32_t i = 0; i < G * H * HD / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
        }
      }
      if (s.slot >= 0) sum += s.rows / PAGE + 1 + END_COST;
      seq[b] = s;
    }
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) misc[warp] = incl;
    __syncthreads();
    uint32_t before = incl - sum;
    for (int i = 0; i < warp; ++i) before += misc[i];
    for (uint32_t b = b0; b < b1; ++b) seq[b].cost += before;
    if (tid == THREADS - 1) seq[B].cost = before + sum;
    __syncthreads();
  }
  const uint64_t C = (uint64_t)seq[B].cost * H;
  if (C == 0) return;
  const uint64_t N = C / MIN_COST >= gridDim.x ? gridDim.x : umax64(1, C / MIN_COST);
  if (blockIdx.x >= N) return;
  const Cuts cuts(C, (uint32_t)N);
  const uint64_t y0 = cuts.begin(blockIdx.x), y1 = cuts.begin(blockIdx.x + 1);
  // the last sequence whose line starts at or before y (idle ones have no length); a warp
  // looks at 32 places at once
  auto seq_at = [&](uint64_t y) -> uint32_t {
    uint32_t lo = 0, n = B;              // it is one of [lo, lo + n)
    while (n > 1) {
      const uint32_t step = (n + 31) / 32, off = lane * step;
      const bool before = off < n && (uint64_t)seq[lo + off].cost * H <= y;
      const uint32_t skip = (__popc(__ballot_sync(0xffffffffu, before)) - 1) * step;
      lo += skip;
      n = min(step, n - skip);
    }
    return lo;
  };

  if (warp == WARPS) {
    // ============================ producer ============================
    // Lane l feeds stage l: ring positions l, l + S, .. of the block's items.
    // It walks the units by itself and loads its next page's id while it waits
    // for the stage, so one pass of the loop serves every stage that is free, in
    // ring order (the consumers' waits rely on it).
    Units it(seq, B, H, y0, y1, seq_at(y0));
    uint32_t base = 0;                // ring position of the unit's first item
    int32_t page = -1;                // >= 0: a page; -1: an id out of range; -2, -3: K, V tail
    auto find = [&](uint32_t k) {     // the item of ring position k; false behind the last
      while (it.valid()) {
        const uint32_t n = it.positions();
        if (k < base + n) {
          const uint32_t j = k - base;
          if (it.has_tail() && j < 2) {
            page = -2 - (int32_t)j;
          } else {
            const uint32_t i = it.has_tail() ? j - 2 : it.i0 - 1 + j;
            page = p.c.table[(size_t)it.sq.slot * p.c.max_pages + i];
            if (page < 0 || (uint32_t)page >= p.c.pages) page = -1;
          }
          return true;
        }
        base += n;
        it.step();
      }
      return false;
    };
    uint32_t k = lane, phase = 0;
    bool more = lane < (int)S && find(k);
    uint64_t* my_full = full + lane;
    uint8_t* st = ring + lane * STAGE;
    uint32_t head = 0, head_stage = 0;   // the first position not issued, the same in all lanes
    uint32_t idle = 0;
    uint64_t since = 0;
    while (__any_sync(0xffffffffu, more)) {
      const uint64_t ready =
          __ballot_sync(0xffffffffu, more && mbar_try_wait(empty + lane, phase ^ 1));
      // stages ready in a row from the head's on
      const uint64_t row = (ready | ready << S) >> head_stage;
      const uint32_t n = min(S, (uint32_t)__ffsll((long long)~row) - 1);
      if (more && k - head < n) {
        if (page >= 0) {
          mbar_arrive_expect_tx(my_full, STAGE);
          const int32_t row = (int32_t)(((uint32_t)page * 2 * H + it.h) * PAGE);
          tc::tma_load_2d(st, &map, 0, row, my_full);
          tc::tma_load_2d(st + 4096, &map, 0, row + (int32_t)(H * PAGE), my_full);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(scale + lane)),
                       "l"(p.c.scales + ((size_t)page * H + it.h) * 2)
                       : "memory");
          cp_async_arrive_noinc(my_full);
        } else if (page == -1) {
          atomicOr(p.flags, kFlagPage);
          scale[lane] = make_float2(CUDART_NAN_F, CUDART_NAN_F);
          mbar_arrive(my_full);
          mbar_arrive(my_full);
        } else {
          // the tail's rows before the append
          const uint32_t bytes = it.sq.rows % PAGE * 256;
          mbar_arrive(my_full);
          if (bytes) {
            mbar_arrive_expect_tx(my_full, bytes);
            bulk_g2s(st, tail_rows(p.c, it.sq.slot, -2 - page, it.h), bytes, my_full);
          } else {
            mbar_arrive(my_full);
          }
        }
        phase ^= 1;
        k += S;
        more = find(k);
      }
      head += n;
      head_stage += n;
      if (head_stage >= S) head_stage -= S;
      if (n) {
        idle = 0;
      } else if (++idle >= 64) {      // nothing was free for a while: bound the wait
        const uint64_t now = globaltimer();
        if (idle == 64) since = now;
        if (__any_sync(0xffffffffu, now - since > kWaitLimitNs)) {
          if (lane == 0) atomicOr(p.flags, kFlagTimeout);
          break;
        }
      }
    }
    // leave no copy in flight, whatever the consumers did
    if (lane < (int)S && k >= S) mbar_wait(my_full, phase ^ 1);
    cp_async_wait_all();
    return;
  }

  if (warp == WARPS + 1) {
    // ========================= sequence warp ========================
    // Per unit of this block, up to two ahead of the consumers: the rotated q
    // into the unit's slot, then, where the block holds the unit's tail, the
    // rotated key and the value into the slot and into the tail (the append).
    Units it(seq, B, H, y0, y1, seq_at(y0));
    uint32_t n = 0;
    for (; it.valid(); it.step()) {
      if (!it.has_items()) continue;
      const uint32_t s = n & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(slot_empty + s, (n >> 1 & 1) ^ 1))) {
        if (lane == 0) atomicOr(p.flags, kFlagTimeout);
        return;
      }
      uint8_t* slot = slots + s * seq_slot<NT>();
      // The new rows' loads go with q's, and the key takes the same table values: 1 x 1,023 rows
      // 9.8 -> 9.5 us, 169 sequences of 22 .. 57 rows with 8 KV heads 43.8 -> 41.9.
      const size_t new_row = (size_t)it.b * p.kv_stride + it.h * HD;
      const uint32_t d = 16 * (lane & 3);
      const Turns turns(p, d, it.sq.rope);
      const Piece key(p.k_new + new_row, d);
      const uint4 value = __ldg(reinterpret_cast<const uint4*>(p.v_new + new_row) + (lane & 15));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t w[16], rest[16];
        const uint32_t head = nt * 8 + (lane >> 2);
        if (head < G) {
          const Piece q(p.q + (size_t)it.b * p.q_stride + ((size_t)it.h * G + head) * HD, d);
          q.rotate(turns, [&](int i, float x, float y) { split2(x, y, w[i], rest[i]); });
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = rest[e] = 0;
        }
        uint4* to = reinterpret_cast<uint4*>(slot) + nt * 128 + lane;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          to[e * 32] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
          to[NT * 128 + e * 32] = make_uint4(rest[4 * e], rest[4 * e + 1], rest[4 * e + 2], rest[4 * e + 3]);
        }
      }
      mbar_arrive(q_full + s);
      if (it.has_tail()) {
        const int last = it.sq.rows % PAGE;
        uint4* kn = reinterpret_cast<uint4*>(slot + 2 * NT * 2048);
        uint4* vn = kn + 16;
        if (lane < 4) {
          uint32_t kw[16];
          key.rotate(turns, [&](int i, float x, float y) { kw[i] = pack_half2(x, y); });
          uint4* row = reinterpret_cast<uint4*>(tail_rows(p.c, it.sq.slot, 0, it.h) + last * HD);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 x = make_uint4(kw[4 * e], kw[4 * e + 1], kw[4 * e + 2], kw[4 * e + 3]);
            const int at = (e & 2) * 4 + 2 * lane + (e & 1);
            row[at] = x;
            kn[at] = x;
          }
        } else if (lane >= 16) {
          reinterpret_cast<uint4*>(tail_rows(p.c, it.sq.slot, 1, it.h) + last * HD)[lane - 16] = value;
          vn[lane - 16] = value;
        }
        __syncwarp();
      }
      if (lane == 0 && !it.whole()) {
        // the unit spans blocks c0 .. c1: it is the last one of c0, the first of the others
        const uint32_t c0 = cuts.owner(it.u0), c1 = cuts.owner(it.u0 + it.np);
        Split& u = splits[it.u0 >= y0 ? 1 : 0];
        u.unit = it.b * H + it.h;
        u.blocks = c1 - c0 + 1;
        u.record = c0 * 2 + 1;
      }
      mbar_arrive(row_full + s);
      if (it.has_tail() && it.sq.rows % PAGE == PAGE - 1) {
        // the open block is full: its rows (the last one just written by this warp) to its page
        const int32_t page = p.c.table[(size_t)it.sq.slot * p.c.max_pages + it.np];
        if (page < 0 || (uint32_t)page >= p.c.pages) {
          if (lane == 0) atomicOr(p.flags, kFlagPage);
        } else {
#pragma unroll 1
          for (uint32_t kv = 0; kv < 2; ++kv) {
            const uint4* from = reinterpret_cast<const uint4*>(tail_rows(p.c, it.sq.slot, kv, it.h));
            uint4 x[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              x[e] = from[(e >> 1) * 64 + (lane >> 3) * 16 + (lane & 7) * 2 + (e & 1)];
            quantise_block<CODE>(x, block_codes(p.c, page, kv, it.h),
                                 p.c.scales + ((size_t)page * H + it.h) * 2 + kv, lane);
          }
        }
      }
      ++n;
    }
    return;
  }

  // ============================= consumers ============================
  const int g = lane >> 2, t = lane & 3;
  const float qk = 1.4426950408889634f * 0.08838834764831845f;   // log2(e) / sqrt(128)
  uint32_t at = 0;                    // ring position of the unit's first item
  uint32_t turn = 0;                  // items before this unit, modulo WARPS
  bool alive = true;
  uint32_t stage = 0, phase = 0;      // of ring position `seen`
  uint32_t seen = 0;
  auto seek = [&](uint32_t k) {       // less than two rounds ahead
    stage += k - seen;
    seen = k;
    while (stage >= S) {
      stage -= S;
      phase ^= 1;
    }
  };
  auto arrived = [&](uint64_t* bar, uint32_t parity) {
    if (alive) {
      alive = __all_sync(0xffffffffu, mbar_wait(bar, parity));
      if (!alive && lane == 0) atomicOr(p.flags, kFlagTimeout);
    }
    return alive;
  };
  // The current stage's data.  Copies may land out of order, so a warp may get
  // here before the stage's previous page (another warp's) has even landed, when
  // the full barrier is a phase behind and its parity says the wrong thing.  So
  // it waits for that page to be freed first: the empty barrier is never more
  // than a phase behind, because a position less than S - 1 earlier has been seen.
  auto landed = [&]() {
    return arrived(empty + stage, phase ^ 1) && arrived(full + stage, phase);
  };
  // A warp that gave up frees no more stages, so the producer gives up too; it
  // goes on to meet the other warps at the unit ends.
  auto release = [&](uint32_t s) {
    __syncwarp();
    if (alive && lane == 0) mbar_arrive(empty + s);
  };

  uint32_t unit = 0;                  // units of this block so far
  for (Units it(seq, B, H, y0, y1, seq_at(y0)); it.valid(); it.step()) {
    const Seq sq = it.sq;
    const uint32_t b = it.b, h = it.h, i0 = it.i0, i1 = it.i1;
    const uint64_t u0 = it.u0;
    if (it.has_items()) {
      // ---------------------------------------------- this block's pages
      Acc<NT> a;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) a.o[nt][i][e] = 0.f;
        a.m[nt][0] = a.m[nt][1] = -CUDART_INF_F;
        a.l[nt][0] = a.l[nt][1] = 0.f;
      }
      const uint32_t first = (warp + WARPS - turn) % WARPS;     // this warp's first item
      const uint8_t* slot = slots + (unit & 1) * seq_slot<NT>();
      const uint32_t slot_phase = unit >> 1 & 1;
      if (i0 + first < i1 && arrived(q_full + (unit & 1), slot_phase)) {
        uint32_t qf[NT][16];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint4 x = reinterpret_cast<const uint4*>(slot)[(nt * 4 + e) * 32 + lane];
            qf[nt][4 * e] = x.x;
            qf[nt][4 * e + 1] = x.y;
            qf[nt][4 * e + 2] = x.z;
            qf[nt][4 * e + 3] = x.w;
          }
        uint32_t i = i0 + first;
        if (i == 0) {
          // --------------------------------------------------------- tail
          seek(at);
          const int last = sq.rows % PAGE;
          const uint8_t* rows = slot + 2 * NT * 2048;
          const uint32_t s0 = stage;
          landed();
          const uint8_t* kt = ring + stage * STAGE;
          seek(at + 1);
          landed();
          const uint8_t* vt = ring + stage * STAGE;
          if (arrived(row_full + (unit & 1), slot_phase)) {
            tail_tile<NT>(kt, vt, rows, rows + 256, last, qk, qf, slot + NT * 2048, a, g, t);
          }
          release(stage);
          release(s0);
          i += WARPS;
        }
        const uint32_t skew = it.has_tail() ? 1 : 0;
        for (; i < i1; i += WARPS) {
          seek(at + i - i0 + skew);
          if (landed()) {
            const float2 sc = scale[stage];
            page_tile<CODE, NT>(ring + stage * STAGE, sc.x, sc.y, qk, qf, slot + NT * 2048, a, g, t);
          }
          release(stage);
        }
      }
      // the row barrier advances with the slot, also past warps that do not use it
      arrived(row_full + (unit & 1), slot_phase);
      __syncwarp();
      if (alive && lane == 0) mbar_arrive(slot_empty + (unit & 1));
      ++unit;
      at += it.positions();
      turn = (turn + i1 - i0) % WARPS;
      // ------------------------------------------------- join the warps
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float l = a.l[nt][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          const int head = warp * 8 * NT + nt * 8 + 2 * t + c;
          if (g == 0) {
            end_m[head] = a.m[nt][c];
            end_l[head] = l;
          }
          float* row = end_acc + head * ACC_PITCH + 16 * ((g >> 1) | ((g & 1) << 2));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<float4*>(row + 4 * k) =
                make_float4(a.o[nt][2 * k][c], a.o[nt][2 * k][c + 2], a.o[nt][2 * k + 1][c],
                            a.o[nt][2 * k + 1][c + 2]);
        }
      }
      named_bar_sync(1, CTHREADS);
      // half a warp takes a head, each lane 8 of its dims
      const bool whole = it.whole();
      float* rec = p.records + (size_t)(blockIdx.x * 2 + (u0 >= y0 ? 1 : 0)) * record_floats<NT>();
      __half* out = p.out + ((size_t)b * H + h) * G * HD;
      const uint32_t sub = lane & 15;
      for (uint32_t i = 2 * warp + (lane >> 4); i < G; i += 2 * WARPS) {
        float m = -CUDART_INF_F, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, end_m[w * 8 * NT + i]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const int head = w * 8 * NT + i;
          const float wl = end_l[head];
          // a warp without pages has maximum -inf and adds nothing
          const float f = wl == 0.f ? 0.f : fast_exp2(end_m[head] - m);
          l += wl * f;
          add_scaled(o, end_acc + head * ACC_PITCH + 8 * sub, f);
        }
        if (whole) {
          write_out(out + i * HD + 8 * sub, o, l);
        } else {
          float4* to = reinterpret_cast<float4*>(rec + i * HD + 8 * sub);
          to[0] = make_float4(o[0], o[1], o[2], o[3]);
          to[1] = make_float4(o[4], o[5], o[6], o[7]);
          if (sub == 0) {
            rec[8 * NT * HD + i] = m;
            rec[8 * NT * (HD + 1) + i] = l;
          }
        }
      }
      named_bar_sync(1, CTHREADS);     // the unit's buffers have been read
    }
  }

  // -------------------------------------------------- join the blocks
  // At most two units span blocks: one that began in an earlier block (its
  // record is this block's first) and one that goes on in a later block.  The
  // last block to leave a unit's record joins it.
  named_bar_sync(1, CTHREADS);
  if (tid < 2 && splits[tid].blocks) {
    __threadfence();
    uint32_t* ticket = p.tickets + splits[tid].unit;
    const bool mine = atomicAdd(ticket, 1) == splits[tid].blocks - 1;
    if (mine) {
      *ticket = 0;
      __threadfence();
    } else {
      splits[tid].blocks = 0;
    }
  }
  named_bar_sync(1, CTHREADS);
  if (splits[0].blocks + splits[1].blocks == 0) return;
  // 8 lanes take a (unit, head)
  for (uint32_t k = tid >> 3; k < 2 * 8 * NT; k += CTHREADS / 8) {
    Split u = splits[k & 1];
    const uint32_t i = k >> 1;
    if (i >= G) u.blocks = 0;
    join_head<NT>(p.records, u, i, p.out + (size_t)u.unit * G * HD, lane & 7);
  }
}

// ------------------------------------------------------------------- host
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(ptr);
  });
  return fn;
}

// Two blocks on an SM with one N tile; with two (groups above 8), whose accumulators do not fit
// the 168 registers that two blocks leave a thread, one block.
template <int NT>
constexpr uint32_t block_smem() { return NT == 1 ? 112 * 1024 : 224 * 1024; }

template <int CODE, int NT>
int decode_variant(DecodeParams& p, const CUtensorMap& map, uint64_t most_cost, int sms,
                   cudaStream_t stream) {
  const uint32_t fixed = fixed_smem<NT>() + (p.batch + 1) * sizeof(Seq);
  constexpr uint32_t per = STAGE + 8 + 16;
  p.stages = (block_smem<NT>() - fixed) / per;
  if (p.stages > 32) p.stages = 32;      // a producer lane each
  // a warp's items are at most WARPS + 1 ring positions apart
  static_assert((block_smem<NT>() - fixed_smem<NT>() - (PVLC_KV8_MAX_BATCH + 1) * sizeof(Seq)) / per >=
                    WARPS + 2,
                "too few ring stages");
  const uint32_t bytes = fixed + p.stages * per;
  const void* fn = reinterpret_cast<const void*>(kv8_decode_kernel<CODE, NT>);
  if (const int st = set_smem_attribute_once(fn, block_smem<NT>())) return st;
  const uint64_t blocks = most_cost / MIN_COST, room = (NT == 1 ? 2 : 1) * (uint64_t)sms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((uint32_t)(blocks < 1 ? 1 : blocks < room ? blocks : room));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv8_decode_kernel<CODE, NT>, p, map) == cudaSuccess
             ? PVLC_OK
             : PVLC_CUDA_ERROR;
}

}  // namespace kv8

size_t kv8_decode_scratch_bytes(uint32_t, uint32_t query_heads, uint32_t kv_heads) {
  const bool wide = query_heads / kv_heads > 8;
  return (size_t)sms_or_default_count() * 2 * 2 * 4 *
         (wide ? kv8::record_floats<2>() : kv8::record_floats<1>());
}

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
  p.stages = 0;
  p.flags = static_cast<uint32_t*>(a.workspace);
  p.tickets = kv8_tickets(a.workspace);
  p.records = reinterpret_cast<float*>(kv8_scratch(a.workspace));
  const int sms = device_sm_count();
  if (sms <= 0) return PVLC_CUDA_ERROR;
  kv8::EncodeTiled enc = kv8::encoder();
  if (!enc) return PVLC_CUDA_ERROR;
  // a layer's codes as 128-byte rows; a box is one (page, K or V, head) block
  CUtensorMap map;
  const cuuint64_t dims[2] = {128, (cuuint64_t)c.pages * 2 * c.kv_heads * kv8::PAGE};
  const cuuint64_t strides[1] = {128};
  const cuuint32_t box[2] = {128, kv8::PAGE};
  const cuuint32_t estr[2] = {1, 1};
  if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p.c.codes, dims, strides, box, estr,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return PVLC_CUDA_ERROR;
  const uint64_t most = (uint64_t)a.batch * c.kv_heads * (c.max_pages + 1 + kv8::END_COST);
  const bool e4m3 = c.code_type == PVLC_KV8_E4M3;
  if (p.group > 8)
    return e4m3 ? kv8::decode_variant<PVLC_KV8_E4M3, 2>(p, map, most, sms, stream)
                : kv8::decode_variant<PVLC_KV8_INT8, 2>(p, map, most, sms, stream);
  return e4m3 ? kv8::decode_variant<PVLC_KV8_E4M3, 1>(p, map, most, sms, stream)
              : kv8::decode_variant<PVLC_KV8_INT8, 1>(p, map, most, sms, stream);
}

}  // namespace pvlc
