"""Attention of a step's new tokens over a plain paged cache
(oscar_chunk_attention): decode, MTP verification, prompts and chunks of them,
in any mixture, for layers whose keys and values are kept as they are
(``append.PagedCache``).  What ``append.append_rotated`` has written of the
step's own tokens is part of what they see.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, decode, rotary as _rotary
from .append import PagedCache

HEAD_SIZES = (64, 128, 256)
MAX_HEADS = 1 << 16
MAX_KEYS = 1 << 30                          # of a request
MAX_INT32 = (1 << 31) - 1
_TOO_SMALL = -3                             # OSCAR_ERR_WORKSPACE_TOO_SMALL

_i32, _i64 = ctypes.c_int32, ctypes.c_int64


class ChunkStepArgs(ctypes.Structure):
    """struct oscar_chunk_step (include/oscar_amd.h)."""
    _fields_ = [("num_requests", _i32), ("num_tokens", _i32), ("num_heads", _i32), ("window", _i32),
                ("table_cols", _i32), ("narrow", _i32), ("wide", _i32), ("joins", _i32), ("few_joins", _i32),
                ("num_kv_heads", _i32), ("head_size", _i32), ("block_size", _i32), ("items_size", _i64),
                ("workspace_size", _i64)]


class ChunkStep:
    """A step's request layout and how its work is cut, for every layer of the
    step whose cache has the geometry of `cache`, whose heads are num_heads and
    whose window is the same (0: none): built once per step, like the block
    table.

    qsl [requests + 1] and seqs [requests] are host lists (query starts from the
    step's token 0; keys after the step); block_tables of integers
    [requests, pages] on the cache's device.  The block table is read at every call
    and replay where it is int32 with rows of their own, and else copied here.

    Building copies the step's arrays to the device on the current stream; calls
    on other streams wait for that by themselves.  A step is not built under graph
    capture.  A captured call keeps this step's lengths and needs the step to live
    as long as the graph, and its replays to come after that copy: torch.cuda.graph
    sees to it (it waits for the device before it captures), and a capture begun in
    another way has to, by a wait of its stream for the one the step was built on."""

    def __init__(self, qsl, seqs, block_tables: torch.Tensor, num_heads: int, cache: PagedCache, window: int = 0):
        layout = decode.request_layout(qsl, seqs)
        requests = len(layout.lengths)
        if num_heads < 1 or num_heads % cache.num_kv_heads:
            raise ValueError(f"{num_heads} query heads do not share {cache.num_kv_heads} kv heads")
        if num_heads > MAX_HEADS:
            raise ValueError(f"chunk attention takes at most {MAX_HEADS} query heads, got {num_heads}")
        if window < 0:
            raise ValueError("the window must be positive, or 0 for none")
        window = min(window, MAX_KEYS)      # (no request is longer; a larger integer would be taken modulo 2^32)
        if cache.head_size not in HEAD_SIZES:
            raise ValueError(f"chunk attention takes head sizes {HEAD_SIZES}, got {cache.head_size}")
        if cache.block_size % 16:
            raise ValueError("chunk attention needs a cache block size that is a multiple of 16")
        if layout.qsl and layout.qsl[0] < 0:
            raise ValueError("query starts are counted from the step's token 0")
        args = ChunkStepArgs()
        items = _plan(layout, requests, num_heads, window, cache, args)
        if block_tables.ndim != 2 or block_tables.shape[0] < requests or block_tables.shape[1] < args.table_cols:
            raise ValueError(f"block table must be [requests, pages] with the {args.table_cols} pages of the longest")
        if block_tables.dtype not in (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8):
            raise ValueError(f"block tables hold integers, got {block_tables.dtype}")
        if block_tables.device != cache.device:
            raise ValueError("the block table must be on the cache's device")
        device = cache.device
        if device.type != "cuda":
            raise ValueError("OSCAR kernels take device tensors")
        if (block_tables.dtype != torch.int32 or block_tables.stride(1) != 1
                or block_tables.stride(0) < block_tables.shape[1]):
            if block_tables.dtype == torch.int64:       # (what does not fit stays outside every cache)
                block_tables = block_tables.clamp(-1, MAX_INT32)
            block_tables = block_tables.to(torch.int32).clone(memory_format=torch.contiguous_format)
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("a step is built before its calls are captured")
        with torch.cuda.device(device):
            host = torch.empty(max(args.items_size, 16), dtype=torch.uint8, pin_memory=True)
            host.copy_(items[:host.numel()])
            self.items = host.to(device, non_blocking=True)
            self.ready = torch.cuda.Event()
            self.ready.record()
            self.stream = _lib.stream_handle(device)
        self.args = args
        self.address = ctypes.addressof(args)
        self.tokens = args.num_tokens
        self.num_heads = num_heads
        self.workspace_size = args.workspace_size
        self.geometry = cache.geometry
        self.device = device
        self.block_tables = block_tables
        self.items_ptr, self.table_ptr, self.table_stride = (self.items.data_ptr(), block_tables.data_ptr(),
                                                             block_tables.stride(0))

    def _join(self, device) -> None:
        """Order this step's arrays before the current stream, which is not the one it was built on."""
        stream = torch.cuda.current_stream(device)
        if not torch.cuda.is_current_stream_capturing():        # (a captured stream cannot wait for another's event)
            stream.wait_event(self.ready)
        self.items.record_stream(stream)
        self.block_tables.record_stream(stream)


def chunk_attention(query: torch.Tensor, cache: PagedCache, step: ChunkStep, scale: float, out=None) -> torch.Tensor:
    """Causal attention of query [N, Hq, D] (the cache's type; token t of the
    step in row t) over the cache; returns [N, Hq, D] of that type, a new tensor
    or `out` (query itself or apart from it), whose rows past the step's tokens and of
    tokens of no request are not written.  scale must be positive.  Keys on pages outside the cache
    are left out; a row that sees no key becomes zeros.  For serving: no autograd
    graph is recorded."""
    device = cache.device
    if cache.geometry != step.geometry or device != step.device:
        raise ValueError("the step was built for another cache geometry or device")
    d, dtype, tokens = cache.head_size, cache.dtype, step.tokens
    if not 0.0 < scale < 3.0e38:
        raise ValueError("scale must be positive and finite")
    q, hq = _rotary.heads(query, tokens, d, dtype, device, "query")
    if hq != step.num_heads:
        raise ValueError(f"query must have the step's {step.num_heads} heads")
    if _misaligned(query, tokens):
        query = query.clone(memory_format=torch.contiguous_format)
        q, _ = _rotary.heads(query, tokens, d, dtype, device, "query")
    if out is None:
        out, o = _rotary.new_heads(query, query.shape[0], hq, d)
    else:
        o = _rotary.out_heads(out, tokens, hq, d, dtype, device, "out")
        if _misaligned(out, tokens):
            raise ValueError("out must have rows at multiples of 16 bytes")
    if tokens == 0:
        return out
    if _lib.stream_handle(device) != step.stream:
        step._join(device)
    need = step.workspace_size
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _lib.call_on(device, "oscar_chunk_attention", step.address, step.items_ptr, step.table_ptr, step.table_stride,
                 cache.address, q, o, scale, None if ws is None else ws.data_ptr(), need)
    return out


def _plan(layout, requests: int, num_heads: int, window: int, cache: PagedCache, args: ChunkStepArgs) -> torch.Tensor:
    """The step's items (host bytes), its sizes in args.  Planned straight into
    128 KB, which most steps' items fit; a step that needs more is planned again."""
    size = 1 << 17
    while True:
        items = torch.empty(size, dtype=torch.uint8)
        status = _lib.load().oscar_chunk_plan(
            ctypes.addressof(layout.qstart), ctypes.addressof(layout.seq_t), requests, num_heads, window,
            cache.address, items.data_ptr(), size, ctypes.byref(args))
        if status != _TOO_SMALL:
            break
        size = args.items_size
    if status != 0:
        raise _lib.OscarKernelError(f"oscar_chunk_plan failed: {_lib.STATUS.get(status, status)}")
    return items


def _misaligned(x: torch.Tensor, tokens: int) -> bool:
    """Whether the first `tokens` rows of x begin off multiples of 16 bytes (8
    two-byte values).  Strides of axes of one entry mean nothing."""
    token, head, _ = x.stride()
    at = x.data_ptr() >> 1
    if tokens > 1:
        at |= token
    if x.shape[1] > 1:
        at |= head
    return at & 7 != 0
