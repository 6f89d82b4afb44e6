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
// follow are spread over the GPU.  Measured, 18 layers of 2 heads, calls back to back:
//   fork and grow of 2 x 4 beams 8.8 us, of 64 x 4 beams 17.3 us (44 MB of open rows, 6.7 us
//     of a copy's rate; the rest is three launches, each a chain of dependent loads and scans,
//     that wait for one another)
//   compact of 32 sequences, 951 MB read and written, 166 us (5.7 TB/s, 87 % of a copy); of
//     65 pages 8.7 us, two launches
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

// Copies the slots to shared memory; whether each is idle (-1) or in range, and
// none is named twice.  `seen` is a bitmap over the slots in shared memory, `first`
// this thread's slot of the first PLAN_THREADS, which its caller has asked for early.
__device__ bool slots_valid(const PageParams& p, uint32_t* seen, int32_t* slot, int32_t first) {
  for (uint32_t i = threadIdx.x; i < (p.slots + 31) / 32; i += PLAN_THREADS) seen[i] = 0;
  for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS)
    slot[b] = b == threadIdx.x ? first : p.slot[b];
  __syncthreads();
  int bad = 0;
  for (uint32_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
    const int32_t s = slot[b];
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
  // The slots, their rows when advanced, the blocks that end within the rows ahead, then a bitmap
  // over all slots.  The call's arrays are read once, before anything is written: they may be
  // the cache's own (advance by tokens doubles every sequence).
  extern __shared__ uint32_t sm[];
  const PageParams& p = g.b;
  int32_t* slot = reinterpret_cast<int32_t*>(sm);
  int32_t* rows = slot + p.batch;
  int32_t* ends = rows + p.batch;
  pdl_wait();
  pdl_launch_dependents();
  // the slots and the first pages' counts at once, although few calls need the latter
  const int32_t first = threadIdx.x < p.batch ? p.slot[threadIdx.x] : -1;
  auto free_pages = [&](uint32_t at) {     // of the four from `at` on, as bits
    uint32_t bits = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (at + i < p.pages && p.refs[at + i] == 0) bits |= 1u << i;
    return bits;
  };
  const uint32_t free_first = free_pages(4 * threadIdx.x);
  int bad = slots_valid(p, sm + 3 * p.batch, slot, first) ? 0 : (int)kFlagSlot;
  // sequences [b0, b1) are this thread's: ranks follow the sequence order
  const uint32_t per = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t b0 = min(p.batch, threadIdx.x * per), b1 = min(p.batch, b0 + per);
  if (!bad) {
    for (uint32_t b = b0; b < b1; ++b) {
      const int32_t s = slot[b];
      if (s < 0) continue;
      const int64_t adv = g.advance ? g.advance[b] : g.advance_by;
      const int64_t ahead = g.ahead ? g.ahead[b] : g.ahead_by;
      const int64_t n = p.tokens[s];
      if (adv < 0 || ahead < 0 || n < 0 || !rows_fit(n + adv + ahead, p.max_pages))
        bad |= kFlagCacheRow;
      rows[b] = (int32_t)(n + adv);
      ends[b] = (int32_t)((n + adv + ahead) / PAGE);
    }
  }
  bad = __syncthreads_or(bad) ? (bad ? bad : -1) : 0;
  if (bad) {                             // nothing is changed
    if (bad > 0) atomicOr(p.flags, (uint32_t)bad);
    return;
  }
  uint32_t need = 0;
  for (uint32_t b = b0; b < b1; ++b) {
    const int32_t s = slot[b];
    if (s < 0) continue;
    p.tokens[s] = rows[b];
    const int32_t* row = p.table + (size_t)s * p.max_pages;
    for (int32_t j = rows[b] / PAGE; j < ends[b]; ++j) need += row[j] < 0;
  }
  uint32_t total;
  uint32_t rank = block_scan(need, &total);
  if (total == 0) return;
  // the first `total` free pages, lowest first
  uint32_t found = 0;
  for (uint32_t base = 0; base < p.pages && found < total; base += 4 * PLAN_THREADS) {
    const uint32_t at = base + 4 * threadIdx.x, mine = base ? free_pages(at) : free_first;
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
    const int32_t s = slot[b];
    if (s < 0) continue;
    int32_t* row = p.table + (size_t)s * p.max_pages;
    for (int32_t j = rows[b] / PAGE; j < ends[b]; ++j) {
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
  // scratch: touched slots, where each copies from (-1: it is only emptied) and its rows
  // [2 batch]; how many are copies, how many there are
  int32_t* dst;
  int32_t* src;
  int32_t* rows;
  uint32_t* counts;
  __half* tails;
  uint32_t layers, heads;
};

// Shared memory: the slots, the parents, the eldest child of every sequence, its rows, the
// free slots that are taken, and bitmaps over all slots: "named by slot[]", "kept" and "holds
// no rows".  Global memory is asked three times: for what the call names and the slots' row
// counts, for the named ones' counts, and to write.
uint32_t fork_plan_smem(uint32_t batch, uint32_t slots) { return 5 * batch * 4 + 3 * ((slots + 31) / 32) * 4; }

__global__ void __launch_bounds__(PLAN_THREADS, 1) kv8_fork_plan_kernel(const ForkParams f) {
  extern __shared__ uint32_t sm[];
  __shared__ uint32_t emptied;
  const PageParams& p = f.b;
  const uint32_t words = (p.slots + 31) / 32, tid = threadIdx.x;
  int32_t* slot = reinterpret_cast<int32_t*>(sm);
  int32_t* parent = slot + p.batch;
  uint32_t* eldest = sm + 2 * p.batch;
  int32_t* rows = reinterpret_cast<int32_t*>(sm + 3 * p.batch);
  int32_t* taken = reinterpret_cast<int32_t*>(sm + 4 * p.batch);
  uint32_t* named = sm + 5 * p.batch;
  uint32_t* kept = named + words;
  uint32_t* none = kept + words;
  pdl_wait();
  pdl_launch_dependents();
  const int32_t first_slot = tid < p.batch ? p.slot[tid] : -1;
  const int32_t first_parent = tid < p.batch ? f.parent[tid] : -1;
  int bad = 0;
  for (uint32_t s = tid; s < words * 32; s += PLAN_THREADS) {      // whole warps
    const uint32_t w = __ballot_sync(0xffffffffu, s < p.slots && p.tokens[s] == 0);
    if (s % 32 == 0) none[s / 32] = w;
  }
  for (uint32_t i = tid; i < words; i += PLAN_THREADS) kept[i] = 0;
  for (uint32_t b = tid; b < p.batch; b += PLAN_THREADS) {
    eldest[b] = 0xffffffffu;
    parent[b] = b == tid ? first_parent : f.parent[b];
    if (parent[b] < -1 || parent[b] >= (int32_t)p.batch) bad |= kFlagSlot;
  }
  if (tid == 0) emptied = 0;
  if (!slots_valid(p, named, slot, first_slot)) bad |= kFlagSlot;
  if (!bad)
    for (uint32_t b = tid; b < p.batch; b += PLAN_THREADS) {
      if (slot[b] < 0) continue;
      const int64_t n = p.tokens[slot[b]];
      if (n < 0 || !rows_fit(n + f.advance_by, p.max_pages)) bad |= kFlagCacheRow;
      rows[b] = (int32_t)(n + f.advance_by);
    }
  if (__syncthreads_or(bad)) {           // nothing is changed
    if (tid == 0) f.counts[0] = f.counts[1] = 0;
    if (bad) atomicOr(p.flags, (uint32_t)bad);
    for (uint32_t b = tid; b < p.batch; b += PLAN_THREADS) f.slot_out[b] = slot[b];
    return;
  }
  auto source = [&](uint32_t b) { return parent[b] >= 0 ? slot[parent[b]] : -1; };
  for (uint32_t b = tid; b < p.batch; b += PLAN_THREADS) {
    if (f.advance_by && slot[b] >= 0) p.tokens[slot[b]] = rows[b];
    const int32_t s = source(b);
    if (s >= 0) {
      atomicMin(eldest + parent[b], b);
      atomicOr(kept + (s >> 5), 1u << (s & 31));
    }
  }
  __syncthreads();
  // Free slots in ascending order: those given up here, and the empty ones that no
  // sequence of this call names.  The children that need one, in sequence order.  One
  // prefix sum for both: at most 65,536 slots below, at most 2,048 children above.
  static_assert(PVLC_KV8_MAX_SLOTS <= 1u << 16 && PVLC_KV8_MAX_BATCH < 1u << 15, "packed counts");
  const uint32_t sper = (p.slots + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t s0 = min(p.slots, tid * sper), s1 = min(p.slots, s0 + sper);
  auto is_free = [&](uint32_t s) {
    const uint32_t bit = 1u << (s & 31);
    if (kept[s >> 5] & bit) return false;
    return ((named[s >> 5] | none[s >> 5]) & bit) != 0;
  };
  const uint32_t per = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS;
  const uint32_t b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  auto moves = [&](uint32_t b) { return source(b) >= 0 && eldest[parent[b]] != b; };
  uint32_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s) mine += is_free(s);
  for (uint32_t b = b0; b < b1; ++b) mine += (uint32_t)moves(b) << 17;
  uint32_t total;
  const uint32_t before = block_scan(mine, &total);
  const uint32_t free_total = total & 0x1ffff, children = total >> 17;
  const uint32_t given = min(children, free_total);
  uint32_t r = before & 0x1ffff;
  for (uint32_t s = s0; s < s1; ++s)
    if (is_free(s)) {
      if (r < given) taken[r] = s;
      if (r >= given && (named[s >> 5] >> (s & 31) & 1u)) {     // given up and not taken
        const uint32_t e = given + atomicAdd(&emptied, 1);
        f.dst[e] = s;
        f.src[e] = -1;
        f.rows[e] = 0;
      }
      ++r;
    }
  __syncthreads();                       // the list is complete
  uint32_t rank = before >> 17;
  for (uint32_t b = b0; b < b1; ++b) {
    int32_t to = source(b);
    if (moves(b)) {
      const int32_t from = to;
      to = -1;
      if (rank < given) {
        to = taken[rank];
        f.dst[rank] = to;
        f.src[rank] = from;
        f.rows[rank] = rows[parent[b]];
      }
      ++rank;
    }
    f.slot_out[b] = to;
  }
  if (tid == 0) {
    f.counts[0] = given;
    f.counts[1] = given + emptied;
    if (given < children) atomicOr(p.flags, kFlagExhausted);
  }
}

// A warp copies the open rows of one (copy, layer, K or V, head), up to 8 KB, eight loads a
// lane at a time (64 x 4 beams: 17.7 us, with four 18.3, with sixteen 18.4); a block does the
// table row, count and page references of one touched slot.  A source slot is a
// kept one and a destination is not, so nothing is read that another one writes.
__global__ void __launch_bounds__(COPY_THREADS) kv8_fork_copy_kernel(const ForkParams f) {
  const PageParams& p = f.b;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t copies = f.counts[0], touched = f.counts[1];
  for (uint32_t i = blockIdx.x; i < touched; i += gridDim.x) {
    const int32_t dst = f.dst[i], src = f.src[i], n = f.rows[i];
    int32_t* to = p.table + (size_t)dst * p.max_pages;
    const int32_t* from = p.table + (size_t)(src >= 0 ? src : 0) * p.max_pages;
    for (uint32_t j = threadIdx.x; j < p.max_pages; j += COPY_THREADS) {
      const int32_t old = to[j];
      const int32_t page = (int32_t)j < n / PAGE ? from[j] : -1;
      if (old >= 0 && (uint32_t)old < p.pages) atomicSub(p.refs + old, 1);
      if (page >= 0 && (uint32_t)page < p.pages) atomicAdd(p.refs + page, 1);
      to[j] = page;
    }
    if (threadIdx.x == 0) p.tokens[dst] = n;
  }
  const uint32_t lane = threadIdx.x & 31, parts = 2 * f.heads;
  const uint32_t warp = blockIdx.x * (COPY_THREADS / 32) + (threadIdx.x >> 5);
  const uint32_t warps = gridDim.x * (COPY_THREADS / 32), units = copies * f.layers * parts;
  for (uint32_t u = warp; u < units; u += warps) {
    const uint32_t i = u / (f.layers * parts), l = u / parts % f.layers, kvh = u % parts;
    const int32_t dst = f.dst[i], src = f.src[i];
    const uint32_t n = f.rows[i] % PAGE * (HD / 8);          // 16-byte pieces
    const size_t layer = (size_t)l * p.slots;
    const uint4* from = reinterpret_cast<const uint4*>(f.tails + ((layer + src) * parts + kvh) * BLOCK_CODES);
    uint4* to = reinterpret_cast<uint4*>(f.tails + ((layer + dst) * parts + kvh) * BLOCK_CODES);
    for (uint32_t e = lane; e < n; e += 8 * 32) {
      uint4 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + 32 * k < n) x[k] = from[e + 32 * k];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + 32 * k < n) to[e + 32 * k] = x[k];
    }
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
  pdl_wait();
  pdl_launch_dependents();
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
  if (c.a.max_pages > c.to_max_pages) {  // nor may a page for later rows be left behind
    const uint64_t more = c.a.max_pages - c.to_max_pages;
    for (uint64_t i = threadIdx.x; i < c.a.slots * more; i += PLAN_THREADS)
      if (c.a.table[i / more * c.a.max_pages + c.to_max_pages + i % more] >= 0) wide = 1;
  }
  wide = __syncthreads_or(wide);
  if (threadIdx.x == 0) {
    const bool fits = count <= c.to_pages && !wide;
    if (!fits) atomicOr(c.a.flags, wide ? kFlagCacheRow : kFlagExhausted);
    *c.live = fits ? count : 0xffffffffu;
    if (c.live_out) *c.live_out = fits ? (int32_t)count : -1;
  }
}

// Pages move through shared memory in pieces of 8 KB (a head's share), each by one
// bulk copy in and one out, so that no registers or load slots bound the bytes in
// flight: two warps of 12 lanes, a stage each, 192 KB an SM.  The two warps' reads
// and writes alternate against each other.  The other warps do the small things.
// 32 sequences: 166 us, with loads and stores through registers 174.
constexpr uint32_t PIECE = 2 * BLOCK_CODES;
constexpr uint32_t LANES = 12, ENGINES = 2;
constexpr uint32_t COMPACT_SMEM = LANES * ENGINES * (PIECE + 8);

__global__ void __launch_bounds__(COPY_THREADS, 1) kv8_compact_copy_kernel(const CompactParams c) {
  extern __shared__ __align__(128) uint8_t ring[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + LANES * ENGINES * PIECE);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < ENGINES && lane < LANES) {
    mbar_init(bars + warp * LANES + lane, 1);
    fence_mbar_init();
  }
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t live = *c.live;
  if (live == 0xffffffffu) return;       // nothing is changed
  const uint32_t H = c.heads;
  if (warp < ENGINES) {
    uint8_t* stage = ring + (warp * LANES + lane) * PIECE;
    uint64_t* bar = bars + warp * LANES + lane;
    const uint64_t n = (uint64_t)c.layers * live * H;
    const uint64_t step = (uint64_t)gridDim.x * ENGINES * LANES;
    uint32_t phase = 0;
    __syncwarp();
    for (uint64_t first = (uint64_t)(blockIdx.x * ENGINES + warp) * LANES; first < n; first += step) {
      const uint64_t k = first + lane;
      const bool on = lane < LANES && k < n;
      size_t to = 0;
      if (on) {
        const uint64_t u = k / H;
        const uint32_t l = (uint32_t)(u / live), i = (uint32_t)(u % live), part = (uint32_t)(k % H);
        const size_t from = ((size_t)l * c.a.pages + c.order[i]) * H + part;
        to = ((size_t)l * c.to_pages + i) * H + part;
        // the stage's last copy out has been read
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        mbar_arrive_expect_tx(bar, PIECE);
        bulk_g2s(stage, c.codes + from * PIECE, PIECE, bar);
      }
      const bool landed = !on || mbar_wait(bar, phase);
      if (!__all_sync(0xffffffffu, landed)) {
        if (lane == 0) atomicOr(c.a.flags, kFlagTimeout);
        if (on) mbar_wait(bar, phase);   // leave no copy in flight
        break;
      }
      phase ^= 1;
      if (on) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                         c.to_codes + to * PIECE),
                     "r"(smem_u32(stage)), "r"(PIECE)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    return;
  }
  constexpr uint32_t REST = COPY_THREADS - ENGINES * 32;
  const uint32_t tid = threadIdx.x - ENGINES * 32;
  const uint32_t t = blockIdx.x * REST + tid, T = gridDim.x * REST;
  // the tables, counts and references
  for (uint64_t i = t; i < (uint64_t)c.to_slots * c.to_max_pages; i += T) {
    const uint32_t s = (uint32_t)(i / c.to_max_pages), j = (uint32_t)(i % c.to_max_pages);
    int32_t page = -1;
    if (s < c.a.slots && j < c.a.max_pages) page = c.a.table[(size_t)s * c.a.max_pages + j];
    c.to_table[i] = page >= 0 && (uint32_t)page < c.a.pages ? c.map[page] : -1;
  }
  for (uint32_t s = t; s < c.to_slots; s += T) c.to_tokens[s] = s < c.a.slots ? c.a.tokens[s] : 0;
  for (uint32_t i = t; i < c.to_pages; i += T) c.to_refs[i] = i < live ? c.a.refs[c.order[i]] : 0;
  // scales
  for (uint64_t e = t; e < (uint64_t)c.layers * live * 2 * H; e += T) {
    const uint64_t u = e / (2 * H);
    const uint32_t l = (uint32_t)(u / live), i = (uint32_t)(u % live), h = (uint32_t)(e % (2 * H));
    c.to_scales[((size_t)l * c.to_pages + i) * 2 * H + h] =
        c.scales[((size_t)l * c.a.pages + c.order[i]) * 2 * H + h];
  }
  // the open blocks' rows: a warp takes one (layer, slot, K or V, head)
  const uint32_t parts = 2 * H, warps = T / 32;
  for (uint64_t u = t / 32; u < (uint64_t)c.layers * c.a.slots * parts; u += warps) {
    const uint32_t l = (uint32_t)(u / parts / c.a.slots), s = (uint32_t)(u / parts % c.a.slots);
    const uint32_t kvh = (uint32_t)(u % parts), n = c.a.tokens[s] % PAGE * (HD / 8);
    const uint4* x = reinterpret_cast<const uint4*>(
        c.tails + (((size_t)l * c.a.slots + s) * parts + kvh) * BLOCK_CODES);
    uint4* y = reinterpret_cast<uint4*>(
        c.to_tails + (((size_t)l * c.to_slots + s) * parts + kvh) * BLOCK_CODES);
    for (uint32_t e = lane; e < n; e += 4 * 32) {
      uint4 z[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + 32 * k < n) z[k] = x[e + 32 * k];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + 32 * k < n) y[e + 32 * k] = z[k];
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

namespace {

// A launch that may start under the end of the kernel ahead of it; each of these
// kernels waits for that one before it does anything.
template <typename P>
int launch(void (*kernel)(P), const P& params, dim3 grid, int threads, uint32_t smem,
           cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, params) == cudaSuccess ? PVLC_OK : PVLC_CUDA_ERROR;
}

}  // namespace

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
  return launch(kv8::kv8_grow_kernel, g, dim3(1), kv8::PLAN_THREADS,
                3 * batch * 4 + (c.slots + 31) / 32 * 4, stream);
}

int kv8_fork_launch(const pvlc_kv8_cache& c, const int32_t* slot, const int32_t* parent,
                    uint32_t batch, int32_t advance_by, int32_t* slot_out, void* ws,
                    cudaStream_t stream) {
  kv8::ForkParams f;
  f.b = kv8::page_params(c, slot, batch, ws);
  f.parent = parent;
  f.slot_out = slot_out;
  f.advance_by = advance_by;
  const int sms = device_sm_count();
  if (sms <= 0) return PVLC_CUDA_ERROR;
  int32_t* s = kv8_scratch(ws);
  f.counts = reinterpret_cast<uint32_t*>(s);
  f.dst = s + 4;
  f.src = f.dst + 2 * batch;
  f.rows = f.src + 2 * batch;
  f.tails = reinterpret_cast<__half*>(c.tails);
  f.layers = c.layers;
  f.heads = c.kv_heads;
  const uint32_t smem = kv8::fork_plan_smem(batch, c.slots);
  if (const int st = set_smem_attribute_once(
          reinterpret_cast<const void*>(kv8::kv8_fork_plan_kernel),
          kv8::fork_plan_smem(PVLC_KV8_MAX_BATCH, PVLC_KV8_MAX_SLOTS)))
    return st;
  if (const int st = launch(kv8::kv8_fork_plan_kernel, f, dim3(1), kv8::PLAN_THREADS, smem, stream))
    return st;
  // a warp for each copy where all but one sequence move, up to eight blocks an SM
  const uint64_t blocks = ((uint64_t)batch * c.layers * 2 * c.kv_heads + 7) / 8;
  return launch(kv8::kv8_fork_copy_kernel, f, dim3((uint32_t)(blocks < 8u * sms ? blocks : 8u * sms)),
                kv8::COPY_THREADS, 0, stream);
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
  if (const int st = launch(kv8::kv8_compact_plan_kernel, c, dim3(1), kv8::PLAN_THREADS, 0, stream))
    return st;
  if (const int st = set_smem_attribute_once(
          reinterpret_cast<const void*>(kv8::kv8_compact_copy_kernel), kv8::COMPACT_SMEM))
    return st;
  return launch(kv8::kv8_compact_copy_kernel, c, dim3(sms), kv8::COPY_THREADS, kv8::COMPACT_SMEM,
                stream);
}

}  // namespace pvlc
