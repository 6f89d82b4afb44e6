// kv8_pages.cu -- the page book-keeping of the 8-bit KV cache: grow (advance
// sequences and give them pages), fork (reorder, duplicate and drop
// sequences) and compact (copy the live pages into another cache).
//
// All of it runs on the device, so a captured decode loop needs no host.
// Pages are shared by count (refs); a full page is never written again, so a
// fork copies only a sequence's table row and the fp16 rows of its open block.
// What the kernels decide does not depend on the order in which threads run:
// pages and slots are given out lowest id first, in sequence order, by prefix
// sums, and the reference counts are integer sums.
//
// Deciding is one block's work (a few thousand integers); the copies that
// follow are spread over the GPU.
#include <cuda_runtime.h>

#include "kv8.cuh"

namespace pvlc {
namespace kv8 {

constexpr int PLAN_THREADS = 1024;
constexpr int COPY_THREADS = 256;

// Exclusive prefix sum of `v` over the block's PLAN_THREADS threads; every
// thread gets the total.
__device__ uint32_t block_scan(uint32_t v, uint32_t* total) {
  __shared__ uint32_t warp_sum[PLAN_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();                       // the previous call's sums have been read
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  uint32_t s = warp_sum[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, s, warp ? warp - 1 : 0);
  return (warp ? before : 0u) + incl - v;
}

struct PageParams {
  int32_t* table;
  int32_t* tokens;
  int32_t* refs;
  uint32_t pages, slots, max_pages;
  uint32_t* flags;
  const int32_t* slot;
  uint32_t batch;
};

// Every slot is idle (-1) or in range, and none is named twice.  `seen` is a
// bitmap over the slots in shared memory.
__device__ bool slots_valid(const PageParams& p, uint32_t* seen) {
  for (uint32_t i = threadIdx.x; i < (p.slots + 31) / 32; i += PLAN_THREADS) seen[i] = 0;
  __syncthreads();
  int bad = 0;
  for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
    const int32_t s = p.slot[b];
    if (s == -1) continue;
    if (s < 0 || (uint32_t)s >= p.slots) {
      bad = 1;
      continue;
    }
    const uint32_t bit = 1u << (s & 31);
    if (atomicOr(seen + (s >> 5), bit) & bit) bad = 1;
  }
  return !__syncthreads_or(bad);
}

// ------------------------------------------------------------------- grow
struct GrowParams {
  PageParams b;
  const int32_t* advance;   // rows per sequence, or null: advance_by for all
  const int32_t* ahead;
  int32_t advance_by, ahead_by;
  int32_t* list;            // [pages] scratch: free page of each rank
};

__global__ void __launch_bounds__(PLAN_THREADS, 1) kv8_grow_kernel(const GrowParams g) {
  extern __shared__ uint32_t seen[];
  const PageParams& p = g.b;
  int bad = slots_valid(p, seen) ? 0 : (int)kFlagSlot;
  // sequences [b0, b1) are this thread's: ranks follow the sequence order
  const uint32_t per = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t b0 = min(p.batch, threadIdx.x * per), b1 = min(p.batch, b0 + per);
  if (!bad) {
    for (uint32_t b = b0; b < b1; ++b) {
      const int32_t s = p.slot[b];
      if (s < 0) continue;
      const int64_t adv = g.advance ? g.advance[b] : g.advance_by;
      const int64_t ahead = g.ahead ? g.ahead[b] : g.ahead_by;
      const int64_t n = p.tokens[s];
      if (adv < 0 || ahead < 0 || n < 0 || !rows_fit(n + adv + ahead, p.max_pages))
        bad |= kFlagCacheRow;
    }
  }
  bad = __syncthreads_or(bad) ? (bad ? bad : -1) : 0;
  if (bad) {                             // nothing is changed
    if (bad > 0) atomicOr(p.flags, (uint32_t)bad);
    return;
  }
  uint32_t need = 0;
  for (uint32_t b = b0; b < b1; ++b) {
    const int32_t s = p.slot[b];
    if (s < 0) continue;
    const int32_t n = p.tokens[s] + (g.advance ? g.advance[b] : g.advance_by);
    p.tokens[s] = n;
    const int32_t end = (n + (g.ahead ? g.ahead[b] : g.ahead_by)) / PAGE;
    const int32_t* row = p.table + (size_t)s * p.max_pages;
    for (int32_t j = n / PAGE; j < end; ++j) need += row[j] < 0;
  }
  uint32_t total;
  uint32_t rank = block_scan(need, &total);
  if (total == 0) return;
  // the first `total` free pages, lowest first
  uint32_t found = 0;
  for (uint32_t base = 0; base < p.pages && found < total; base += 4 * PLAN_THREADS) {
    uint32_t mine = 0;
    const uint32_t at = base + 4 * threadIdx.x;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (at + i < p.pages && p.refs[at + i] == 0) mine |= 1u << i;
    uint32_t n;
    uint32_t r = found + block_scan(__popc(mine), &n);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (mine >> i & 1u) {
        if (r < total) g.list[r] = at + i;
        ++r;
      }
    found += n;
  }
  found = min(found, total);
  __syncthreads();                       // the list is complete
  for (uint32_t b = b0; b < b1; ++b) {
    const int32_t s = p.slot[b];
    if (s < 0) continue;
    const int32_t n = p.tokens[s];
    const int32_t end = (n + (g.ahead ? g.ahead[b] : g.ahead_by)) / PAGE;
    int32_t* row = p.table + (size_t)s * p.max_pages;
    for (int32_t j = n / PAGE; j < end; ++j) {
      if (row[j] >= 0) continue;
      if (rank < found) {
        const int32_t page = g.list[rank];
        row[j] = page;
        p.refs[page] = 1;
      }
      ++rank;
    }
  }
  if (found < total && threadIdx.x == 0) atomicOr(p.flags, kFlagExhausted);
}

// ------------------------------------------------------------------- fork
struct ForkParams {
  PageParams b;
  const int32_t* parent;
  int32_t* slot_out;
  int32_t advance_by;
  // scratch: free slots [slots]; touched slots and where each copies from (-1:
  // it is only emptied) [2 batch]; how many
  int32_t* free_list;
  int32_t* dst;
  int32_t* src;
  uint32_t* touched;
  __half* tails;
  uint32_t layers, heads;
};

// Shared memory: slots' bitmaps "named by slot[]" and "kept", then the eldest
// child of every sequence.
__global__ void __launch_bounds__(PLAN_THREADS, 1) kv8_fork_plan_kernel(const ForkParams f) {
  extern __shared__ uint32_t sm[];
  const PageParams& p = f.b;
  const uint32_t words = (p.slots + 31) / 32;
  uint32_t* named = sm;
  uint32_t* kept = named + words;
  uint32_t* eldest = kept + words;
  int bad = slots_valid(p, named) ? 0 : (int)kFlagSlot;
  for (uint32_t i = threadIdx.x; i < words; i += PLAN_THREADS) kept[i] = 0;
  for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
    eldest[b] = 0xffffffffu;
    const int32_t m = f.parent[b];
    if (m < -1 || m >= (int32_t)p.batch) bad |= kFlagSlot;
  }
  if (!bad)
    for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
      const int32_t s = p.slot[b];
      if (s < 0) continue;
      const int64_t n = p.tokens[s];
      if (n < 0 || !rows_fit(n + f.advance_by, p.max_pages)) bad |= kFlagCacheRow;
    }
  const bool refuse = __syncthreads_or(bad);
  if (threadIdx.x == 0) *f.touched = 0;
  if (refuse) {                          // nothing is changed
    if (bad) atomicOr(p.flags, (uint32_t)bad);
    for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) f.slot_out[b] = p.slot[b];
    return;
  }
  for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
    const int32_t s = p.slot[b];
    if (s >= 0) p.tokens[s] += f.advance_by;
    const int32_t m = f.parent[b];
    if (m >= 0 && p.slot[m] >= 0) {
      atomicMin(eldest + m, b);
      atomicOr(kept + (p.slot[m] >> 5), 1u << (p.slot[m] & 31));
    }
  }
  __syncthreads();
  // free slots in ascending order: those given up here, and the empty ones
  // that no sequence of this call names
  const uint32_t sper = (p.slots + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t s0 = min(p.slots, threadIdx.x * sper), s1 = min(p.slots, s0 + sper);
  auto is_free = [&](uint32_t s) {
    const uint32_t bit = 1u << (s & 31);
    if (kept[s >> 5] & bit) return false;
    return (named[s >> 5] & bit) != 0 || p.tokens[s] == 0;
  };
  uint32_t nfree = 0;
  for (uint32_t s = s0; s < s1; ++s) nfree += is_free(s);
  uint32_t free_total;
  uint32_t r = block_scan(nfree, &free_total);
  for (uint32_t s = s0; s < s1; ++s)
    if (is_free(s)) f.free_list[r++] = s;
  // the children that need a slot, in sequence order
  const uint32_t per = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t b0 = min(p.batch, threadIdx.x * per), b1 = min(p.batch, b0 + per);
  auto moves = [&](uint32_t b) {
    const int32_t m = f.parent[b];
    return m >= 0 && p.slot[m] >= 0 && eldest[m] != b;
  };
  uint32_t n = 0;
  for (uint32_t b = b0; b < b1; ++b) n += moves(b);
  uint32_t children;
  uint32_t rank = block_scan(n, &children);    // its barriers also publish free_list
  const uint32_t given = min(children, free_total);
  for (uint32_t b = b0; b < b1; ++b) {
    const int32_t m = f.parent[b];
    int32_t to = -1;
    if (moves(b)) {
      if (rank < given) {
        to = f.free_list[rank];
        f.dst[rank] = to;
        f.src[rank] = p.slot[m];
      }
      ++rank;
    } else if (m >= 0 && p.slot[m] >= 0) {
      to = p.slot[m];
    }
    f.slot_out[b] = to;
  }
  // slots given up and not taken: emptied
  uint32_t emptied = 0;
  auto empties = [&](uint32_t q) {      // rank q of the free list
    const uint32_t s = f.free_list[q];
    return (named[s >> 5] >> (s & 31) & 1u) != 0;
  };
  const uint32_t left = free_total - given;
  const uint32_t fper = (left + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t f0 = given + min(left, threadIdx.x * fper), f1 = min(free_total, f0 + fper);
  for (uint32_t q = f0; q < f1; ++q) emptied += empties(q);
  uint32_t emptied_total;
  uint32_t e = given + block_scan(emptied, &emptied_total);
  for (uint32_t q = f0; q < f1; ++q)
    if (empties(q)) {
      f.dst[e] = f.free_list[q];
      f.src[e++] = -1;
    }
  if (threadIdx.x == 0) {
    *f.touched = given + emptied_total;
    if (given < children) atomicOr(p.flags, kFlagExhausted);
  }
}

// Block (i, 0): the table row, count and page references of touched slot i;
// block (i, 1 + l): its tail rows in layer l.  A source slot is a kept one and
// a destination is not, so no block reads what another writes.
__global__ void __launch_bounds__(128) kv8_fork_copy_kernel(const ForkParams f) {
  const PageParams& p = f.b;
  if (blockIdx.x >= *f.touched) return;
  const int32_t dst = f.dst[blockIdx.x], src = f.src[blockIdx.x];
  const int32_t n = src >= 0 ? p.tokens[src] : 0;
  if (blockIdx.y == 0) {
    int32_t* to = p.table + (size_t)dst * p.max_pages;
    const int32_t* from = p.table + (size_t)(src >= 0 ? src : 0) * p.max_pages;
    for (uint32_t j = threadIdx.x; j < p.max_pages; j += blockDim.x) {
      const int32_t old = to[j];
      const int32_t page = (int32_t)j < n / PAGE ? from[j] : -1;
      if (old >= 0 && (uint32_t)old < p.pages) atomicSub(p.refs + old, 1);
      if (page >= 0 && (uint32_t)page < p.pages) atomicAdd(p.refs + page, 1);
      to[j] = page;
    }
    if (threadIdx.x == 0) p.tokens[dst] = n;
    return;
  }
  if (src < 0) return;
  const uint32_t rows = n % PAGE;
  const size_t layer = (size_t)(blockIdx.y - 1) * p.slots;
  const uint4* from = reinterpret_cast<const uint4*>(f.tails + (layer + src) * 2 * f.heads * BLOCK_CODES);
  uint4* to = reinterpret_cast<uint4*>(f.tails + (layer + dst) * 2 * f.heads * BLOCK_CODES);
  const uint32_t per = rows * (HD / 8);        // 16-byte pieces of one (K/V, head)
  for (uint32_t i = threadIdx.x; i < per * 2 * f.heads; i += blockDim.x) {
    const size_t at = (size_t)(i / per) * (BLOCK_CODES / 8) + i % per;
    to[at] = from[at];
  }
}

// ---------------------------------------------------------------- compact
struct CompactParams {
  PageParams a;             // the source (flags are the call's)
  const uint8_t* codes;
  const float* scales;
  const __half* tails;
  uint8_t* to_codes;
  float* to_scales;
  __half* to_tails;
  int32_t* to_table;
  int32_t* to_tokens;
  int32_t* to_refs;
  uint32_t to_pages, to_slots, to_max_pages;
  uint32_t layers, heads;
  int32_t* order;           // [pages] scratch: the page that becomes page i
  int32_t* map;             // [pages] scratch: a live page's new id, or -1
  uint32_t* live;           // scratch: live pages, or ~0 when they do not fit
  int32_t* live_out;        // or null
};

__global__ void __launch_bounds__(PLAN_THREADS, 1) kv8_compact_plan_kernel(const CompactParams c) {
  uint32_t count = 0;
  for (uint32_t base = 0; base < c.a.pages; base += 4 * PLAN_THREADS) {
    const uint32_t at = base + 4 * threadIdx.x;
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (at + i < c.a.pages && c.a.refs[at + i] > 0) mine |= 1u << i;
    uint32_t n;
    uint32_t r = count + block_scan(__popc(mine), &n);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if (at + i >= c.a.pages) break;
      const bool is = mine >> i & 1u;
      c.map[at + i] = is ? (int32_t)r : -1;
      if (is) c.order[r++] = at + i;
    }
    count += n;
  }
  // a sequence's entries all have to fit the other table's rows
  int wide = 0;
  for (uint32_t s = threadIdx.x; s < c.a.slots; s += PLAN_THREADS) {
    const int32_t n = c.a.tokens[s];
    if (n < 0 || !rows_fit((uint32_t)n, c.to_max_pages)) wide = 1;
  }
  wide = __syncthreads_or(wide);
  if (threadIdx.x == 0) {
    const bool fits = count <= c.to_pages && !wide;
    if (!fits) atomicOr(c.a.flags, wide ? kFlagCacheRow : kFlagExhausted);
    *c.live = fits ? count : 0xffffffffu;
    if (c.live_out) *c.live_out = fits ? (int32_t)count : -1;
  }
}

__global__ void __launch_bounds__(COPY_THREADS) kv8_compact_copy_kernel(const CompactParams c) {
  const uint32_t live = *c.live;
  if (live == 0xffffffffu) return;       // nothing is changed
  const uint32_t t = blockIdx.x * COPY_THREADS + threadIdx.x, T = gridDim.x * COPY_THREADS;
  // the tables, counts and references
  for (uint64_t i = t; i < (uint64_t)c.to_slots * c.to_max_pages; i += T) {
    const uint32_t s = (uint32_t)(i / c.to_max_pages), j = (uint32_t)(i % c.to_max_pages);
    int32_t page = -1;
    if (s < c.a.slots && j < c.a.max_pages) page = c.a.table[(size_t)s * c.a.max_pages + j];
    c.to_table[i] = page >= 0 && (uint32_t)page < c.a.pages ? c.map[page] : -1;
  }
  for (uint32_t s = t; s < c.to_slots; s += T) c.to_tokens[s] = s < c.a.slots ? c.a.tokens[s] : 0;
  for (uint32_t i = t; i < c.to_pages; i += T) c.to_refs[i] = i < live ? c.a.refs[c.order[i]] : 0;
  // scales, then codes: one block takes a (layer, page) at a time
  const uint32_t H = c.heads;
  for (uint64_t u = blockIdx.x; u < (uint64_t)c.layers * live; u += gridDim.x) {
    const uint32_t l = (uint32_t)(u / live), i = (uint32_t)(u % live);
    const size_t from = (size_t)l * c.a.pages + c.order[i], to = (size_t)l * c.to_pages + i;
    for (uint32_t h = threadIdx.x; h < 2 * H; h += COPY_THREADS)
      c.to_scales[to * 2 * H + h] = c.scales[from * 2 * H + h];
    const uint4* x = reinterpret_cast<const uint4*>(c.codes + from * 2 * H * BLOCK_CODES);
    uint4* y = reinterpret_cast<uint4*>(c.to_codes + to * 2 * H * BLOCK_CODES);
    for (uint32_t e = threadIdx.x; e < 2 * H * BLOCK_CODES / 16; e += COPY_THREADS) y[e] = x[e];
  }
  // the open blocks' rows
  for (uint64_t u = blockIdx.x; u < (uint64_t)c.layers * c.a.slots; u += gridDim.x) {
    const uint32_t l = (uint32_t)(u / c.a.slots), s = (uint32_t)(u % c.a.slots);
    const uint32_t per = c.a.tokens[s] % PAGE * (HD / 8);
    const uint4* x = reinterpret_cast<const uint4*>(c.tails + ((size_t)l * c.a.slots + s) * 2 * H * BLOCK_CODES);
    uint4* y = reinterpret_cast<uint4*>(c.to_tails + ((size_t)l * c.to_slots + s) * 2 * H * BLOCK_CODES);
    for (uint32_t e = threadIdx.x; e < per * 2 * H; e += COPY_THREADS) {
      const size_t at = (size_t)(e / per) * (BLOCK_CODES / 8) + e % per;
      y[at] = x[at];
    }
  }
}

PageParams page_params(const pvlc_kv8_cache& c, const int32_t* slot, uint32_t batch, void* ws) {
  PageParams p;
  p.table = c.table;
  p.tokens = c.tokens;
  p.refs = c.refs;
  p.pages = c.pages;
  p.slots = c.slots;
  p.max_pages = c.max_pages;
  p.flags = static_cast<uint32_t*>(ws);
  p.slot = slot;
  p.batch = batch;
  return p;
}

}  // namespace kv8

int kv8_grow_launch(const pvlc_kv8_cache& c, const int32_t* slot, uint32_t batch,
                    const int32_t* advance, int32_t advance_by, const int32_t* ahead,
                    int32_t ahead_by, void* ws, cudaStream_t stream) {
  kv8::GrowParams g;
  g.b = kv8::page_params(c, slot, batch, ws);
  g.advance = advance;
  g.ahead = ahead;
  g.advance_by = advance_by;
  g.ahead_by = ahead_by;
  g.list = kv8_scratch(ws);
  kv8::kv8_grow_kernel<<<1, kv8::PLAN_THREADS, (c.slots + 31) / 32 * 4, stream>>>(g);
  return cudaPeekAtLastError() == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

int kv8_fork_launch(const pvlc_kv8_cache& c, const int32_t* slot, const int32_t* parent,
                    uint32_t batch, int32_t advance_by, int32_t* slot_out, void* ws,
                    cudaStream_t stream) {
  kv8::ForkParams f;
  f.b = kv8::page_params(c, slot, batch, ws);
  f.parent = parent;
  f.slot_out = slot_out;
  f.advance_by = advance_by;
  int32_t* s = kv8_scratch(ws);
  f.touched = reinterpret_cast<uint32_t*>(s);
  f.dst = s + 4;
  f.src = f.dst + 2 * batch;
  f.free_list = f.src + 2 * batch;
  f.tails = reinterpret_cast<__half*>(c.tails);
  f.layers = c.layers;
  f.heads = c.kv_heads;
  const uint32_t smem = 2 * ((c.slots + 31) / 32) * 4 + batch * 4;
  kv8::kv8_fork_plan_kernel<<<1, kv8::PLAN_THREADS, smem, stream>>>(f);
  kv8::kv8_fork_copy_kernel<<<dim3(2 * batch, 1 + c.layers), 128, 0, stream>>>(f);
  return cudaPeekAtLastError() == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

int kv8_compact_launch(const pvlc_kv8_cache& a, const pvlc_kv8_cache& b, int32_t* live_out,
                       void* ws, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (sms <= 0) return PVLC_CUDA_ERROR;
  kv8::CompactParams c;
  c.a = kv8::page_params(a, nullptr, 0, ws);
  c.codes = static_cast<const uint8_t*>(a.codes);
  c.scales = a.scales;
  c.tails = reinterpret_cast<const __half*>(a.tails);
  c.to_codes = static_cast<uint8_t*>(b.codes);
  c.to_scales = b.scales;
  c.to_tails = reinterpret_cast<__half*>(b.tails);
  c.to_table = b.table;
  c.to_tokens = b.tokens;
  c.to_refs = b.refs;
  c.to_pages = b.pages;
  c.to_slots = b.slots;
  c.to_max_pages = b.max_pages;
  c.layers = a.layers;
  c.heads = a.kv_heads;
  int32_t* s = kv8_scratch(ws);
  c.live = reinterpret_cast<uint32_t*>(s);
  c.order = s + 4;
  c.map = c.order + a.pages;
  c.live_out = live_out;
  kv8::kv8_compact_plan_kernel<<<1, kv8::PLAN_THREADS, 0, stream>>>(c);
  kv8::kv8_compact_copy_kernel<<<8 * sms, kv8::COPY_THREADS, 0, stream>>>(c);
  return cudaPeekAtLastError() == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

}  // namespace pvlc
