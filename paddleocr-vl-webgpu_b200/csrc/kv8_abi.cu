// kv8_abi.cu -- the extern "C" boundary of the 8-bit paged KV cache and of the
// beam selection: host checks, before any device effect, in the order zero
// dimensions, geometry, null pointers, alignment, workspace.
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/pvlc_cuda_attn.h"
#include "pvlc_common.cuh"
#include "pvlc_internal.h"

namespace pvlc {

namespace {

// Workspace: fault word, 256 bytes; then one ticket for each (sequence, KV
// head) of the largest call; then scratch that no call needs of another.
constexpr size_t kHeader = 256;
constexpr size_t kTickets = (size_t)PVLC_KV8_MAX_BATCH * PVLC_KV8_MAX_KV_HEADS * 4;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check_cache(const pvlc_kv8_cache* c) {
  if (!c) return PVLC_NULL_POINTER;
  if (!c->layers || !c->pages || !c->slots || !c->max_pages || !c->kv_heads)
    return PVLC_ZERO_DIMENSION;
  if (c->code_type != PVLC_KV8_E4M3 && c->code_type != PVLC_KV8_INT8)
    return PVLC_INVALID_DECODER_GEOMETRY;
  if (c->kv_heads > PVLC_KV8_MAX_KV_HEADS || c->slots > PVLC_KV8_MAX_SLOTS ||
      c->max_pages > PVLC_KV8_MAX_PAGES_PER_SLOT || c->layers > PVLC_KV8_MAX_LAYERS)
    return PVLC_INVALID_DECODER_GEOMETRY;
  // a layer's 128-byte code rows are addressed with 31 bits
  if ((uint64_t)c->pages * c->kv_heads * 2 * PVLC_KV8_PAGE > 0x7fffffffull)
    return PVLC_ARITHMETIC_OVERFLOW;
  if (!c->codes || !c->scales || !c->tails || !c->table || !c->tokens || !c->refs)
    return PVLC_NULL_POINTER;
  if (!aligned(c->codes, 16) || !aligned(c->tails, 16) || !aligned(c->scales, 8) ||
      !aligned(c->table, 4) || !aligned(c->tokens, 4) || !aligned(c->refs, 4))
    return PVLC_MISALIGNED_POINTER;
  return PVLC_OK;
}

// The byte ranges of a cache's arrays.
struct Ranges {
  uintptr_t at[6];
  uint64_t bytes[6];
};
Ranges ranges(const pvlc_kv8_cache& c) {
  const uint64_t heads = (uint64_t)c.layers * c.kv_heads, block = PVLC_KV8_PAGE * 128;
  return {{reinterpret_cast<uintptr_t>(c.codes), reinterpret_cast<uintptr_t>(c.scales),
           reinterpret_cast<uintptr_t>(c.tails), reinterpret_cast<uintptr_t>(c.table),
           reinterpret_cast<uintptr_t>(c.tokens), reinterpret_cast<uintptr_t>(c.refs)},
          {heads * c.pages * 2 * block, heads * c.pages * 8, heads * c.slots * 4 * block,
           (uint64_t)c.slots * c.max_pages * 4, (uint64_t)c.slots * 4, (uint64_t)c.pages * 4}};
}

// Memory that a call writes: whether other arrays share bytes with it.
struct Written {
  uintptr_t at;
  uint64_t bytes;
  Written(const void* p, uint64_t n) : at(reinterpret_cast<uintptr_t>(p)), bytes(n) {}
  bool meets(const void* p, uint64_t n) const {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p);
    return p && at < x + n && x < at + bytes;
  }
  // rows of `n` bytes, `stride` apart
  bool meets_rows(const void* p, uint64_t rows, uint64_t stride, uint64_t n) const {
    if (!rows || !meets(p, (rows - 1) * stride + n)) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(p);
    // the last row that begins at or before it, and the one behind that
    const uint64_t i = at <= x ? 0 : (at - x) / stride;
    const char* row = static_cast<const char*>(p) + (i < rows ? i : rows - 1) * stride;
    return meets(row, n) || (i + 1 < rows && meets(row + stride, n));
  }
  bool meets(const pvlc_kv8_cache& c) const {
    const Ranges r = ranges(c);
    for (int i = 0; i < 6; ++i)
      if (at < r.at[i] + r.bytes[i] && r.at[i] < at + bytes) return true;
    return false;
  }
};

size_t page_scratch(uint32_t batch, uint32_t slots, uint32_t pages) {
  const size_t fork = 4 + 6 * (size_t)batch + slots, compact = 4 + 2 * (size_t)pages;
  return 4 * (fork > compact ? fork : compact);
}

int check_workspace(const void* ws, size_t bytes, size_t scratch) {
  if (!ws) return PVLC_NULL_POINTER;
  if (!aligned(ws, 16)) return PVLC_MISALIGNED_POINTER;
  return bytes < kHeader + kTickets + scratch ? PVLC_WORKSPACE_TOO_SMALL : PVLC_OK;
}

}  // namespace

int32_t* kv8_scratch(void* workspace) {
  return reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + kHeader + kTickets);
}
uint32_t* kv8_tickets(void* workspace) {
  return reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + kHeader);
}

}  // namespace pvlc

using namespace pvlc;

extern "C" {

size_t pvlc_attn_kv8_workspace_bytes(uint32_t batch, uint32_t query_heads, uint32_t kv_heads,
                                     uint32_t slots, uint32_t pages) {
  if (!batch || !query_heads || !kv_heads || batch > PVLC_KV8_MAX_BATCH ||
      kv_heads > PVLC_KV8_MAX_KV_HEADS || query_heads % kv_heads ||
      query_heads / kv_heads > PVLC_KV8_MAX_GROUP || slots > PVLC_KV8_MAX_SLOTS)
    return 0;
  const size_t a = page_scratch(batch, slots, pages);
  const size_t b = kv8_decode_scratch_bytes(batch, query_heads, kv_heads);
  return kHeader + kTickets + ((a > b ? a : b) + 255) / 256 * 256;
}

int pvlc_attn_kv8_workspace_init(void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_workspace(workspace, workspace_bytes, 0);
  if (st) return st;
  return cudaMemsetAsync(workspace, 0, kHeader + kTickets, static_cast<cudaStream_t>(stream)) ==
                 cudaSuccess
             ? PVLC_OK
             : PVLC_CUDA_ERROR;
}

int pvlc_attn_kv8_errors(void* workspace, uint32_t* flags_out, void* stream) {
  if (!workspace || !flags_out) return PVLC_NULL_POINTER;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t flags = 0;
  if (cudaMemcpyAsync(&flags, workspace, 4, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return PVLC_CUDA_ERROR;
  // Blocks that gave up have left tickets behind, by which a later call would join a split unit
  // before all of its records are written.
  const size_t clear = flags & kFlagTimeout ? kHeader + kTickets : 4;
  if (cudaMemsetAsync(workspace, 0, clear, s) != cudaSuccess) return PVLC_CUDA_ERROR;
  *flags_out = flags;
  return flags ? PVLC_DEVICE_FAULT_FLAG : PVLC_OK;
}

int pvlc_attn_kv8_store(const pvlc_kv8_cache* cache, uint32_t layer, const pvlc_half* k,
                        const pvlc_half* v, uint32_t rows, uint32_t row_stride,
                        const int32_t* begin, const int32_t* count, const int32_t* slot,
                        uint32_t batch, uint32_t max_count, void* workspace,
                        size_t workspace_bytes, void* stream) {
  int st = check_cache(cache);
  if (st) return st;
  if (!batch || !rows || !max_count) return PVLC_ZERO_DIMENSION;
  if (batch > PVLC_KV8_MAX_BATCH || layer >= cache->layers) return PVLC_INVALID_DECODER_GEOMETRY;
  if (max_count > cache->max_pages * PVLC_KV8_PAGE + PVLC_KV8_PAGE - 1 || max_count > rows)
    return PVLC_CAPACITY_EXHAUSTED;
  if (row_stride < cache->kv_heads * 128u || row_stride % 8) return PVLC_LENGTH_MISMATCH;
  if (!k || !v || !begin || !count || !slot) return PVLC_NULL_POINTER;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(begin, 4) || !aligned(count, 4) ||
      !aligned(slot, 4))
    return PVLC_MISALIGNED_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, 0))) return st;
  const Kv8StoreArgs a{k, v, rows, row_stride, begin, count, slot, batch, max_count, workspace};
  return kv8_store_launch(*cache, layer, a, static_cast<cudaStream_t>(stream));
}

int pvlc_attn_kv8_decode(const pvlc_kv8_cache* cache, uint32_t layer, const pvlc_half* q,
                         uint32_t q_row_stride, const pvlc_half* k_new, const pvlc_half* v_new,
                         uint32_t kv_row_stride, uint32_t query_heads, const float* rope_cos,
                         const float* rope_sin, uint32_t rope_rows, const int32_t* rope_row,
                         const int32_t* slot, uint32_t batch, void* workspace,
                         size_t workspace_bytes, pvlc_half* out, void* stream) {
  int st = check_cache(cache);
  if (st) return st;
  if (!batch || !query_heads || !rope_rows) return PVLC_ZERO_DIMENSION;
  if (batch > PVLC_KV8_MAX_BATCH || layer >= cache->layers || query_heads % cache->kv_heads ||
      query_heads / cache->kv_heads > PVLC_KV8_MAX_GROUP)
    return PVLC_INVALID_DECODER_GEOMETRY;
  if (!slot && batch > cache->slots) return PVLC_INVALID_DECODER_GEOMETRY;
  if (q_row_stride < query_heads * 128u || kv_row_stride < cache->kv_heads * 128u ||
      q_row_stride % 8 || kv_row_stride % 8)
    return PVLC_LENGTH_MISMATCH;
  if (!q || !k_new || !v_new || !rope_cos || !rope_sin || !out) return PVLC_NULL_POINTER;
  if (!aligned(q, 16) || !aligned(k_new, 16) || !aligned(v_new, 16) || !aligned(rope_cos, 16) ||
      !aligned(rope_sin, 16) || !aligned(out, 16) || !aligned(rope_row, 4) || !aligned(slot, 4))
    return PVLC_MISALIGNED_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes,
                            kv8_decode_scratch_bytes(batch, query_heads, cache->kv_heads))))
    return st;
  // the output of one sequence is written while another's inputs are read
  const Written o(out, (uint64_t)batch * query_heads * 256);
  const uint64_t kv_row = cache->kv_heads * 256ull, table = 3ull * rope_rows * 128 * 4;
  if (o.meets(*cache) || o.meets_rows(q, batch, q_row_stride * 2ull, query_heads * 256ull) ||
      o.meets_rows(k_new, batch, kv_row_stride * 2ull, kv_row) ||
      o.meets_rows(v_new, batch, kv_row_stride * 2ull, kv_row) || o.meets(rope_cos, table) ||
      o.meets(rope_sin, table) || o.meets(rope_row, batch * 4ull) || o.meets(slot, batch * 4ull) ||
      o.meets(workspace, workspace_bytes))
    return PVLC_LENGTH_MISMATCH;
  const Kv8DecodeArgs a{q,         k_new,    v_new, rope_cos, rope_sin,  rope_row, slot,
                        out,       q_row_stride, kv_row_stride, rope_rows, batch, query_heads,
                        workspace};
  return kv8_decode_launch(*cache, layer, a, static_cast<cudaStream_t>(stream));
}

int pvlc_attn_kv8_grow(const pvlc_kv8_cache* cache, const int32_t* slot, uint32_t batch,
                       const int32_t* advance, uint32_t advance_by, const int32_t* ahead,
                       uint32_t ahead_by, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_cache(cache);
  if (st) return st;
  if (!batch) return PVLC_ZERO_DIMENSION;
  if (batch > PVLC_KV8_MAX_BATCH) return PVLC_INVALID_DECODER_GEOMETRY;
  const uint32_t most = cache->max_pages * PVLC_KV8_PAGE + PVLC_KV8_PAGE - 1;
  if (advance_by > most || ahead_by > most) return PVLC_CAPACITY_EXHAUSTED;
  if (!slot) return PVLC_NULL_POINTER;
  if (!aligned(slot, 4) || !aligned(advance, 4) || !aligned(ahead, 4))
    return PVLC_MISALIGNED_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, page_scratch(batch, cache->slots, cache->pages))))
    return st;
  return kv8_grow_launch(*cache, slot, batch, advance, (int32_t)advance_by, ahead,
                         (int32_t)ahead_by, workspace, static_cast<cudaStream_t>(stream));
}

int pvlc_attn_kv8_fork(const pvlc_kv8_cache* cache, const int32_t* slot, const int32_t* parent,
                       uint32_t batch, uint32_t advance_by, int32_t* slot_out, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int st = check_cache(cache);
  if (st) return st;
  if (!batch) return PVLC_ZERO_DIMENSION;
  if (batch > PVLC_KV8_MAX_BATCH) return PVLC_INVALID_DECODER_GEOMETRY;
  if (advance_by > cache->max_pages * PVLC_KV8_PAGE + PVLC_KV8_PAGE - 1)
    return PVLC_CAPACITY_EXHAUSTED;
  if (!slot || !parent || !slot_out) return PVLC_NULL_POINTER;
  if (!aligned(slot, 4) || !aligned(parent, 4) || !aligned(slot_out, 4))
    return PVLC_MISALIGNED_POINTER;
  const intptr_t apart = reinterpret_cast<intptr_t>(slot_out) - reinterpret_cast<intptr_t>(slot);
  const intptr_t apart2 = reinterpret_cast<intptr_t>(slot_out) - reinterpret_cast<intptr_t>(parent);
  const intptr_t span = (intptr_t)batch * 4;
  if ((apart > -span && apart < span) || (apart2 > -span && apart2 < span))
    return PVLC_LENGTH_MISMATCH;           // slot_out is written while slot and parent are read
  if ((st = check_workspace(workspace, workspace_bytes, page_scratch(batch, cache->slots, cache->pages))))
    return st;
  const Written o(slot_out, span);
  if (o.meets(*cache) || o.meets(workspace, workspace_bytes)) return PVLC_LENGTH_MISMATCH;
  return kv8_fork_launch(*cache, slot, parent, batch, (int32_t)advance_by, slot_out, workspace,
                         static_cast<cudaStream_t>(stream));
}

int pvlc_attn_kv8_compact(const pvlc_kv8_cache* from, const pvlc_kv8_cache* into,
                          int32_t* live_out, void* workspace, size_t workspace_bytes,
                          void* stream) {
  int st = check_cache(from);
  if (st || (st = check_cache(into))) return st;
  if (from->layers != into->layers || from->kv_heads != into->kv_heads ||
      from->code_type != into->code_type || from->slots > into->slots)
    return PVLC_INVALID_DECODER_GEOMETRY;
  if (from->codes == into->codes || from->scales == into->scales || from->tails == into->tails ||
      from->table == into->table || from->tokens == into->tokens || from->refs == into->refs)
    return PVLC_LENGTH_MISMATCH;           // the two caches share no memory
  if (!aligned(live_out, 4)) return PVLC_MISALIGNED_POINTER;
  if ((st = check_workspace(workspace, workspace_bytes, page_scratch(1, from->slots, from->pages))))
    return st;
  const Ranges a = ranges(*from), b = ranges(*into);
  for (int i = 0; i < 6; ++i)
    for (int j = 0; j < 6; ++j)
      if (a.at[i] < b.at[j] + b.bytes[j] && b.at[j] < a.at[i] + a.bytes[i])
        return PVLC_LENGTH_MISMATCH;       // nor parts of them
  const Written o(live_out, 4);
  if (live_out && (o.meets(*from) || o.meets(*into) || o.meets(workspace, workspace_bytes)))
    return PVLC_LENGTH_MISMATCH;
  return kv8_compact_launch(*from, *into, live_out, workspace, static_cast<cudaStream_t>(stream));
}

static int check_beam(uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t topk) {
  if (!batch || !beams || !vocab || !topk) return PVLC_ZERO_DIMENSION;
  if (beams > PVLC_BEAM_MAX_BEAMS || topk > PVLC_BEAM_MAX_TOPK || batch > PVLC_KV8_MAX_BATCH ||
      (uint64_t)batch * beams > 65535u || vocab > PVLC_BEAM_MAX_VOCAB)
    return PVLC_INVALID_DECODER_GEOMETRY;
  return PVLC_OK;
}

size_t pvlc_lm_head_beam_topk_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab,
                                              uint32_t topk) {
  return check_beam(batch, beams, vocab, topk) ? 0
                                               : beam_topk_workspace_bytes(batch, beams, vocab, topk);
}

int pvlc_lm_head_beam_topk(const void* logits, uint32_t half_logits, uint64_t row_stride,
                           const float* scores, uint32_t batch, uint32_t beams, uint32_t vocab,
                           uint32_t topk, void* workspace, size_t workspace_bytes,
                           float* out_score, int32_t* out_beam, int32_t* out_token,
                           void* stream) {
  const int st = check_beam(batch, beams, vocab, topk);
  if (st) return st;
  if (half_logits > 1 || row_stride < vocab || (uint64_t)beams * vocab < topk)
    return PVLC_LENGTH_MISMATCH;
  if (!logits || !scores || !workspace || !out_score || !out_beam || !out_token)
    return PVLC_NULL_POINTER;
  if (!aligned(logits, half_logits ? 2 : 4) || !aligned(scores, 4) || !aligned(workspace, 16) ||
      !aligned(out_score, 4) || !aligned(out_beam, 4) || !aligned(out_token, 4))
    return PVLC_MISALIGNED_POINTER;
  if (workspace_bytes < beam_topk_workspace_bytes(batch, beams, vocab, topk))
    return PVLC_WORKSPACE_TOO_SMALL;
  // a request's results are written while others' scores, logits and lists are read
  const void* outs[3] = {out_score, out_beam, out_token};
  const uint64_t n = (uint64_t)batch * topk * 4, unit = half_logits ? 2 : 4;
  for (int i = 0; i < 3; ++i) {
    const Written o(outs[i], n);
    if (o.meets_rows(logits, (uint64_t)batch * beams, row_stride * unit, vocab * unit) ||
        o.meets(scores, (uint64_t)batch * beams * 4) || o.meets(workspace, workspace_bytes) ||
        o.meets(outs[(i + 1) % 3], n))
      return PVLC_LENGTH_MISMATCH;
  }
  const BeamArgs a{logits, half_logits, row_stride, scores, batch, beams, vocab, topk,
                   workspace, out_score, out_beam, out_token};
  return beam_topk_launch(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
