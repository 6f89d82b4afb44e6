// kv8_store.cu -- rows of prompts into the 8-bit paged KV cache.
//
// Sequence b's new rows follow the tokens[slot[b]] rows it holds: with the
// old = tokens % 32 rows of its open block in front, every full block of 32
// is quantised into its page (kv8.cuh) and what is left becomes the new tail.
//
// One warp takes one (sequence, block, K or V, head): 8 KB of fp16 rows in
// 16 independent 16-byte loads a lane, the block maximum by shuffles, 4 KB of
// codes out, everything read and written once.  Bound by HBM: 256 prompts of 1,238
// rows, 2 heads, 490 MB, take 76 us (6.4 TB/s, 98 % of a copy).  A prompt of 1,564
// rows behind 23 takes 4.7 us, the latency of a launch and three dependent loads.
// The warp's block stays in registers between its two passes, the maximum and the
// rounding: 109 registers, 16 warps an SM, 128 KB of loads in flight.
#include <cuda_runtime.h>

#include "kv8.cuh"

namespace pvlc {
namespace kv8 {

constexpr int STORE_WARPS = 4;

struct StoreParams {
  View c;
  const __half* k;
  const __half* v;
  const int32_t* begin;
  const int32_t* count;
  const int32_t* slot;
  uint32_t rows, row_stride, max_count;
  uint32_t* flags;
};

template <int CODE>
__global__ void __launch_bounds__(STORE_WARPS * 32) kv8_store_kernel(const StoreParams p) {
  const int lane = threadIdx.x & 31;
  const uint32_t b = blockIdx.y;
  const uint32_t H = p.c.heads;
  const uint32_t unit = blockIdx.x * STORE_WARPS + (threadIdx.x >> 5);
  const uint32_t j = unit / (2 * H), kv = unit / H % 2, h = unit % H;   // block, K/V, head
  const int32_t slot = p.slot[b];
  if (slot == -1) return;                       // idle
  const int32_t count = p.count[b], begin = p.begin[b];
  uint32_t bad = 0;
  int32_t held = 0;
  if (slot < 0 || (uint32_t)slot >= p.c.slots) {
    bad |= kFlagSlot;
  } else {
    held = p.c.tokens[slot];
    if (held < 0 || count < 0 || !rows_fit((uint64_t)held + (uint32_t)count, p.c.max_pages))
      bad |= kFlagCacheRow;
  }
  if (count < 0 || (uint32_t)count > p.max_count || begin < 0 ||
      (uint64_t)begin + (uint32_t)count > p.rows)
    bad |= kFlagRows;
  if (bad) {
    if (unit == 0 && lane == 0) atomicOr(p.flags, bad);
    return;
  }
  const uint32_t old = held % PAGE;
  const uint32_t total = old + count;           // rows from the open block's start
  const uint32_t full = total / PAGE;
  const __half* src = (kv ? p.v : p.k) + (size_t)begin * p.row_stride + h * HD;
  __half* tail = tail_rows(p.c, slot, kv, h);

  // rows [max(old, 32 full), total) become the tail
  auto write_tail = [&]() {
    const uint32_t r0 = full ? full * PAGE : old;
    for (uint32_t r = r0 + (lane >> 4); r < total; r += 2)
      *reinterpret_cast<uint4*>(tail + (size_t)(r - full * PAGE) * HD + (lane & 15) * 8) =
          __ldg(reinterpret_cast<const uint4*>(src + (size_t)(r - old) * p.row_stride) + (lane & 15));
  };
  // The warp of block 0 reads the old tail; where there is one, it also
  // writes the new tail, after its reads.  Otherwise the warp behind the last
  // full block does.
  const bool by_first = old > 0 && full > 0;
  if (j == full && !by_first) {
    write_tail();
    return;
  }
  if (j >= full) return;

  uint4 x[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t r = j * PAGE + 4 * i + (lane >> 3);
    const __half* row = r < old ? tail + (size_t)r * HD : src + (size_t)(r - old) * p.row_stride;
    const uint4* at = reinterpret_cast<const uint4*>(row) + 2 * (lane & 7);
    x[2 * i] = at[0];
    x[2 * i + 1] = at[1];
  }
  const int32_t page = p.c.table[(size_t)slot * p.c.max_pages + held / PAGE + j];
  if (page < 0 || (uint32_t)page >= p.c.pages) {
    if (lane == 0) atomicOr(p.flags, kFlagPage);
  } else {
    quantise_block<CODE>(x, block_codes(p.c, page, kv, h),
                         p.c.scales + ((size_t)page * H + h) * 2 + kv, lane);
  }
  if (by_first && j == 0) {
    __syncwarp();
    write_tail();
  }
}

}  // namespace kv8

int kv8_store_launch(const pvlc_kv8_cache& c, uint32_t layer, const Kv8StoreArgs& a,
                     cudaStream_t stream) {
  kv8::StoreParams p;
  p.c = kv8::view_of(c, layer);
  p.k = reinterpret_cast<const __half*>(a.k);
  p.v = reinterpret_cast<const __half*>(a.v);
  p.begin = a.begin;
  p.count = a.count;
  p.slot = a.slot;
  p.rows = a.rows;
  p.row_stride = a.row_stride;
  p.max_count = a.max_count;
  p.flags = static_cast<uint32_t*>(a.workspace);
  // blocks 0 .. (31 + max_count) / 32, the last of them a tail
  const uint64_t units = ((uint64_t)(a.max_count + kv8::PAGE - 1) / kv8::PAGE + 1) * 2 * c.kv_heads;
  const dim3 grid((uint32_t)((units + kv8::STORE_WARPS - 1) / kv8::STORE_WARPS), a.batch);
  const dim3 block(kv8::STORE_WARPS * 32);
  if (c.code_type == PVLC_KV8_E4M3)
    kv8::kv8_store_kernel<PVLC_KV8_E4M3><<<grid, block, 0, stream>>>(p);
  else
    kv8::kv8_store_kernel<PVLC_KV8_INT8><<<grid, block, 0, stream>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

}  // namespace pvlc
