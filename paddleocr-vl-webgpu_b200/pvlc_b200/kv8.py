"""8-bit paged KV cache: store, single-token decode, grow, fork and compact.

A `Cache` holds the pages of every decoder layer in 8-bit codes (e4m3 or int8) with one
power-of-two scale per (page, K or V, KV head), the fp16 rows of each sequence's open block,
and the device-side page tables.  The C ABI (include/pvlc_cuda_attn.h) defines the layout and
the arithmetic; every function here checks placement, type and shape, then enqueues one call
on the current CUDA stream.  Sequences are named by slot tensors (int32, distinct, -1: idle).

A prompt goes in with grow(ahead=rows), store() per layer, grow(advance=rows, ahead=1); a
decode step is decode() per layer, then grow(advance=1, ahead=1) -- or, in a beam search,
ops.beam_topk, fork(advance=1), grow(ahead=1).  None of it waits for the host, so a step can
be captured in a CUDA graph.  Faults that only the device can see (a slot out of range, pages
exhausted) skip the work and set a bit of Workspace.errors().
"""
from __future__ import annotations

import ctypes

import torch

from . import abi

PAGE, HD = 32, 128                       # rows of a page, head dimension
CODE_TYPES = {torch.float8_e4m3fn: 0, torch.int8: 1}

# Workspace.errors() bits
FLAG_ROWS_HELD, FLAG_ROPE_ROW, FLAG_TIMEOUT = 1, 2, 8
FLAG_PAGE, FLAG_SLOT, FLAG_EXHAUSTED, FLAG_INPUT_ROWS = 16, 32, 64, 128


# The current device and a stream's handle as plain numbers: the checks below run once for
# every layer of every decode step, so they ask torch for as little as they can.
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _need(t, dtype, shape, index, name):
    """A contiguous tensor of this type and shape on CUDA device `index`."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index
            and t.shape == shape and t.is_contiguous()):
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the cache on cuda:{index}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    raise ValueError(f"{name} must be contiguous")


def _rows(t, heads, index, name):
    """A [rows, heads, 128] fp16 tensor whose rows may sit apart; (rows, stride in elements)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype is not torch.float16:
        raise TypeError(f"{name} must be torch.float16, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the cache on cuda:{index}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != HD:
        raise ValueError(f"{name} has shape {tuple(shape)}, expected (rows, {heads}, {HD})")
    s0, s1, s2 = t.stride()
    if s2 != 1 or (heads > 1 and s1 != HD):
        raise ValueError(f"{name}: each row must be contiguous")
    if shape[0] == 1:
        return 1, heads * HD
    if s0 >= 1 << 32:
        raise ValueError(f"{name}: rows are too far apart")
    return shape[0], s0


def _batch(slot):
    """The number of sequences a slot tensor names."""
    if not isinstance(slot, torch.Tensor):
        raise TypeError("slot must be a CUDA tensor")
    return slot.numel()


class Cache:
    """The device arrays of an 8-bit paged KV cache (the C ABI's pvlc_kv8_cache).

    codes [layers, pages, 2, kv_heads, 32, 128] (torch.float8_e4m3fn or torch.int8), scales
    [layers, pages, kv_heads, 2] f32, tails [layers, slots, 2, kv_heads, 32, 128] fp16, table
    [slots, max_pages], tokens [slots] and refs [pages] int32; all contiguous, on one device.
    Their contents are the caller's to change, the tensors stay: the kernels have their
    addresses.  Cache.empty() makes one with no sequences."""

    ARRAYS = ("codes", "scales", "tails", "table", "tokens", "refs")

    def __init__(self, codes, scales, tails, table, tokens, refs):
        if not isinstance(codes, torch.Tensor) or not codes.is_cuda:
            raise TypeError("codes must be a CUDA tensor")
        if codes.dtype not in CODE_TYPES:
            raise TypeError(f"codes must be float8_e4m3fn or int8, got {codes.dtype}")
        if codes.dim() != 6 or codes.shape[2] != 2 or codes.shape[4:] != (PAGE, HD):
            raise ValueError("codes must be [layers, pages, 2, kv_heads, 32, 128], got "
                             f"{tuple(codes.shape)}")
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            raise ValueError("table must be [slots, max_pages]")
        L, P, _, H = codes.shape[:4]
        S, M = table.shape
        self.device, self.index = codes.device, codes.get_device()
        _need(codes, codes.dtype, codes.shape, self.index, "codes")
        _need(scales, torch.float32, (L, P, H, 2), self.index, "scales")
        _need(tails, torch.float16, (L, S, 2, H, PAGE, HD), self.index, "tails")
        _need(table, torch.int32, (S, M), self.index, "table")
        _need(tokens, torch.int32, (S,), self.index, "tokens")
        _need(refs, torch.int32, (P,), self.index, "refs")
        self.codes, self.scales, self.tails = codes, scales, tails
        self.table, self.tokens, self.refs = table, tokens, refs
        self.layers, self.pages, self.slots, self.max_pages, self.kv_heads = L, P, S, M, H
        self._c = abi.Kv8CacheStruct(*[t.data_ptr() for t in (codes, scales, tails, table,
                                                              tokens, refs)],
                                     L, P, S, M, H, CODE_TYPES[codes.dtype])
        self._p = ctypes.addressof(self._c)

    def __setattr__(self, name, value):
        if name in self.ARRAYS and getattr(self, name, value) is not value:
            raise AttributeError(f"a cache keeps its {name} tensor: copy into it instead")
        super().__setattr__(name, value)

    @classmethod
    def empty(cls, layers: int, pages: int, slots: int, max_pages: int, kv_heads: int = 2,
              dtype=torch.float8_e4m3fn, device=None) -> "Cache":
        dev = torch.device(device or "cuda")
        ints = dict(dtype=torch.int32, device=dev)
        return cls(torch.empty((layers, pages, 2, kv_heads, PAGE, HD), dtype=dtype, device=dev),
                   torch.empty((layers, pages, kv_heads, 2), dtype=torch.float32, device=dev),
                   torch.empty((layers, slots, 2, kv_heads, PAGE, HD), dtype=torch.float16,
                               device=dev),
                   torch.full((slots, max_pages), -1, **ints), torch.zeros(slots, **ints),
                   torch.zeros(pages, **ints))

    def reset(self):
        """Drop every sequence: all pages and slots are free again."""
        self.table.fill_(-1)
        self.tokens.zero_()
        self.refs.zero_()

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in
                   (self.codes, self.scales, self.tails, self.table, self.tokens, self.refs))


class Workspace:
    """Device scratch and fault word of the calls on caches up to this one's sizes, for
    batches up to `batch` sequences of `query_heads` heads.  One stream at a time."""

    def __init__(self, cache: Cache, batch: int, query_heads: int | None = None):
        self.device, self.index = cache.device, cache.index
        self.nbytes = int(abi.lib().pvlc_attn_kv8_workspace_bytes(
            int(batch), int(query_heads or cache.kv_heads), cache.kv_heads, cache.slots,
            cache.pages))
        if not self.nbytes:
            raise abi.PvlcError(abi.INVALID_DECODER_GEOMETRY, "pvlc_attn_kv8_workspace_bytes")
        self.buffer = torch.empty(self.nbytes, dtype=torch.uint8, device=self.device)
        self._p = self.buffer.data_ptr()
        with torch.cuda.device(self.device):
            abi.check(abi.lib().pvlc_attn_kv8_workspace_init(
                self._p, self.nbytes, _raw_stream(self.index)), "pvlc_attn_kv8_workspace_init")

    def errors(self) -> int:
        """Read and clear the fault word (FLAG_* bits); waits for the current stream.  After
        FLAG_TIMEOUT what decode() returned since is undefined, and the workspace is as new."""
        flags = ctypes.c_uint32(0)
        # a default stream's handle is the same on every device: it means the current one's
        with torch.cuda.device(self.device):
            st = abi.lib().pvlc_attn_kv8_errors(self._p, ctypes.byref(flags),
                                                _raw_stream(self.index))
        if st not in (abi.OK, abi.DEVICE_FAULT_FLAG):
            abi.check(st, "pvlc_attn_kv8_errors")
        return int(flags.value)


def _call(cache, workspace):
    """What every call checks: a cache and a workspace on the current device.  Returns it."""
    if not isinstance(cache, Cache) or not isinstance(workspace, Workspace):
        raise TypeError("expected a kv8.Cache and a kv8.Workspace")
    index = cache.index
    if workspace.index != index:
        raise ValueError(f"the workspace is on {workspace.device}, the cache on {cache.device}")
    if index != _current_device():
        raise ValueError(f"the cache is on {cache.device}, which is not the current device")
    return index


# Each function below first hands its arguments to the compiled checks (csrc/py_calls.cpp),
# which make the call when all is well and return None otherwise; then the checks here run
# and name what is wrong (or make the call, for what those do not know, a tensor subclass).


def _plain(cache, workspace):
    return type(cache) is Cache and type(workspace) is Workspace and abi.calls is not None


def store(cache: Cache, layer: int, k, v, begin, count, slot, max_count: int,
          workspace: Workspace):
    """Append rows to sequences in one layer (pvlc_attn_kv8_store).

    k, v: [rows, kv_heads, 128] fp16, keys rotated, rows the same distance apart in both;
    sequence b takes rows begin[b] : begin[b] + count[b] (int32 device tensors, count <=
    max_count) behind the rows its slot holds."""
    if _plain(cache, workspace):
        st = abi.calls.store(cache._p, cache.index, workspace._p, workspace.nbytes,
                             workspace.index, layer, slot, k, v, begin, count, max_count)
        if st is not None:
            return abi.check(st, "pvlc_attn_kv8_store")
    index = _call(cache, workspace)
    n, stride = _rows(k, cache.kv_heads, index, "k")
    if _rows(v, cache.kv_heads, index, "v") != (n, stride):
        raise ValueError("k and v must have the same rows, the same distance apart")
    B = _batch(slot)
    _need(slot, torch.int32, (B,), index, "slot")
    _need(begin, torch.int32, (B,), index, "begin")
    _need(count, torch.int32, (B,), index, "count")
    if not 0 <= layer < cache.layers or not 0 <= max_count < 1 << 32:
        raise ValueError("layer or max_count out of range")
    st = abi.lib().pvlc_attn_kv8_store(
        cache._p, layer, k.data_ptr(), v.data_ptr(), n, stride, begin.data_ptr(),
        count.data_ptr(), slot.data_ptr(), B, max_count, workspace._p, workspace.nbytes,
        _raw_stream(index))
    if st:
        abi.check(st, "pvlc_attn_kv8_store")


def decode(cache: Cache, layer: int, q, k_new, v_new, rope_cos, rope_sin, slot,
           workspace: Workspace, rope_row=None, out=None):
    """One token of every sequence in one layer, M-RoPE and append fused
    (pvlc_attn_kv8_decode).

    q [B, query_heads, 128], k_new, v_new [B, kv_heads, 128] fp16 before RoPE, each possibly a
    row-strided view (column blocks of one projection; k_new and v_new alike); rope tables
    [3, R, 128] f32; rope_row int32 [B] (None: the rows the slot holds); slot int32 [B] (None:
    sequence b is slot b).  Returns [B, query_heads, 128] fp16."""
    if _plain(cache, workspace):
        r = abi.calls.decode(cache._p, cache.index, workspace._p, workspace.nbytes,
                             workspace.index, layer, q, k_new, v_new, rope_cos, rope_sin, slot,
                             rope_row, out)
        if type(r) is int:
            abi.check(r, "pvlc_attn_kv8_decode")
        if r is not None:
            return r
    index, H = _call(cache, workspace), cache.kv_heads
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise TypeError("q must be a [B, query_heads, 128] CUDA tensor")
    if not isinstance(rope_cos, torch.Tensor) or rope_cos.dim() != 3:
        raise TypeError("rope_cos must be a [3, R, 128] CUDA tensor")
    QH, R = q.shape[1], rope_cos.shape[1]
    B, qs = _rows(q, QH, index, "q")
    kb, ks = _rows(k_new, H, index, "k_new")
    if kb != B or _rows(v_new, H, index, "v_new") != (B, ks):
        raise ValueError("k_new and v_new must have q's rows, the same distance apart")
    _need(rope_cos, torch.float32, (3, R, HD), index, "rope_cos")
    _need(rope_sin, torch.float32, (3, R, HD), index, "rope_sin")
    sp = rp = None
    if slot is not None:
        _need(slot, torch.int32, (B,), index, "slot")
        sp = slot.data_ptr()
    if rope_row is not None:
        _need(rope_row, torch.int32, (B,), index, "rope_row")
        rp = rope_row.data_ptr()
    if out is None:
        out = q.new_empty((B, QH, HD))
    else:
        _need(out, torch.float16, (B, QH, HD), index, "out")
    if not 0 <= layer < cache.layers:
        raise ValueError("layer out of range")
    st = abi.lib().pvlc_attn_kv8_decode(
        cache._p, layer, q.data_ptr(), qs, k_new.data_ptr(), v_new.data_ptr(), ks, QH,
        rope_cos.data_ptr(), rope_sin.data_ptr(), R, rp, sp, B, workspace._p, workspace.nbytes,
        out.data_ptr(), _raw_stream(index))
    if st:
        abi.check(st, "pvlc_attn_kv8_decode")
    return out


def _amount(x, B, index, name):
    """(device pointer, 0) of a per-sequence tensor, or (None, rows) of one number."""
    if isinstance(x, torch.Tensor):
        _need(x, torch.int32, (B,), index, name)
        return x.data_ptr(), 0
    if not 0 <= x < 1 << 31:
        raise ValueError(f"{name} out of range")
    return None, x


def grow(cache: Cache, slot, workspace: Workspace, advance=0, ahead=0):
    """Advance sequences by `advance` rows and give them the pages of their next `ahead` rows
    (each a number, or an int32 tensor per sequence; pvlc_attn_kv8_grow)."""
    if _plain(cache, workspace):
        st = abi.calls.grow(cache._p, cache.index, workspace._p, workspace.nbytes,
                            workspace.index, slot, advance, ahead)
        if st is not None:
            return abi.check(st, "pvlc_attn_kv8_grow")
    index, B = _call(cache, workspace), _batch(slot)
    _need(slot, torch.int32, (B,), index, "slot")
    ap, an = _amount(advance, B, index, "advance")
    hp, hn = _amount(ahead, B, index, "ahead")
    st = abi.lib().pvlc_attn_kv8_grow(cache._p, slot.data_ptr(), B, ap, an, hp, hn, workspace._p,
                                      workspace.nbytes, _raw_stream(index))
    if st:
        abi.check(st, "pvlc_attn_kv8_grow")


def fork(cache: Cache, slot, parent, workspace: Workspace, advance: int = 0, out=None):
    """Sequence b becomes a copy of sequence parent[b] (int32 [B], -1: none), after every
    sequence has grown by `advance` rows; returns the new slots (pvlc_attn_kv8_fork)."""
    if _plain(cache, workspace):
        r = abi.calls.fork(cache._p, cache.index, workspace._p, workspace.nbytes,
                           workspace.index, slot, parent, advance, out)
        if type(r) is int:
            abi.check(r, "pvlc_attn_kv8_fork")
        if r is not None:
            return r
    index, B = _call(cache, workspace), _batch(slot)
    _need(slot, torch.int32, (B,), index, "slot")
    _need(parent, torch.int32, (B,), index, "parent")
    if out is None:
        out = torch.empty_like(slot)
    else:
        _need(out, torch.int32, (B,), index, "out")
    if not 0 <= advance < 1 << 31:
        raise ValueError("advance out of range")
    st = abi.lib().pvlc_attn_kv8_fork(cache._p, slot.data_ptr(), parent.data_ptr(), B, advance,
                                      out.data_ptr(), workspace._p, workspace.nbytes,
                                      _raw_stream(index))
    if st:
        abi.check(st, "pvlc_attn_kv8_fork")
    return out


def compact(cache: Cache, into: Cache, workspace: Workspace, live=None):
    """Copy the live pages, in order, to the front of another cache with the same layers,
    heads and type, and make its tables match (pvlc_attn_kv8_compact).  live: optional int32
    [1] tensor that receives the number of live pages (-1: they do not fit)."""
    if _plain(cache, workspace) and type(into) is Cache:
        st = abi.calls.compact(cache._p, cache.index, workspace._p, workspace.nbytes,
                               workspace.index, into._p, into.index, live)
        if st is not None:
            return abi.check(st, "pvlc_attn_kv8_compact")
    index = _call(cache, workspace)
    if not isinstance(into, Cache):
        raise TypeError("into must be a kv8.Cache")
    if into.index != index:
        raise ValueError(f"into is on {into.device}, the cache on {cache.device}")
    if live is not None:
        _need(live, torch.int32, (1,), index, "live")
    st = abi.lib().pvlc_attn_kv8_compact(cache._p, into._p,
                                         live.data_ptr() if live is not None else None,
                                         workspace._p, workspace.nbytes, _raw_stream(index))
    if st:
        abi.check(st, "pvlc_attn_kv8_compact")
