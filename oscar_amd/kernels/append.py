"""Plain and 8-bit paged caches and their write (oscar_append_rotated,
oscar_append_normed, oscar_append_quantized), and the reading of the latter's
rows (oscar_read_back).

The layers the INT2 impl leaves native (MTP draft layers, sliding-window
layers) keep keys and values as they are, in bf16 or fp16 pages, or in half of
that: a byte a value and a power of two for each token and head.  One launch
turns a step's queries and keys by their positions (after their heads' norms,
where a model has them) and puts keys and values into their slots.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, rotary as _rotary

_p, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class PlainCacheArgs(ctypes.Structure):
    """struct oscar_plain_cache (include/oscar_amd.h)."""
    _fields_ = [("k", _p), ("v", _p), ("num_pages", _i64), ("k_stride_page", _i64), ("k_stride_token", _i64),
                ("k_stride_head", _i64), ("v_stride_page", _i64), ("v_stride_token", _i64), ("v_stride_head", _i64),
                ("block_size", _i32), ("num_kv_heads", _i32), ("head_size", _i32), ("dtype", _i32)]


class PagedCache:
    """A layer's plain K and V pages [pages, block_size, Hk, D] (bf16 or fp16),
    checked and packed once.  They may be views: of one tensor that holds both
    ([pages, 2, block_size, Hk, D] or [2, pages, ...]), or with heads before
    tokens.  Features are contiguous; rows start at multiples of 16 bytes."""

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor):
        if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or min(k_cache.shape) < 1:
            raise ValueError("K and V caches must share [pages, block_size, heads, head size]")
        if k_cache.dtype not in (torch.bfloat16, torch.float16) or v_cache.dtype != k_cache.dtype:
            raise ValueError("plain caches are bf16 or fp16, K and V alike")
        if k_cache.device != v_cache.device:
            raise ValueError("K and V caches must be on one device")
        pages, bs, hk, d = k_cache.shape
        if d % 8 or d > 256:
            raise ValueError(f"head size {d} must be a multiple of 8, at most 256")
        strides = []
        for x in (k_cache, v_cache):
            page, token, head, feature = x.stride()
            # strides of axes of one entry mean nothing
            token = token if bs > 1 else d
            head = head if hk > 1 else d
            tokens, heads = (bs - 1) * token + d, (hk - 1) * head + d
            page = page if pages > 1 else tokens + heads - d
            if feature != 1 or x.data_ptr() % 16 or page % 8 or token % 8 or head % 8 or min(page, token, head) < d:
                raise ValueError("cache rows must be contiguous features at multiples of 16 bytes")
            nested = heads <= token if token > head else tokens <= head
            if (bs > 1 and hk > 1 and not nested) or (pages > 1 and page < tokens + heads - d):
                raise ValueError("cache tokens, heads or pages overlap")
            if 2 * (tokens + heads - d) >= 1 << 31:
                raise ValueError("a cache page must span less than 2 GiB")
            strides += [2 * page, 2 * token, 2 * head]
        self.k_cache, self.v_cache = k_cache, v_cache
        self.device, self.dtype, self.on_gpu = k_cache.device, k_cache.dtype, k_cache.is_cuda
        self.pages, self.block_size, self.num_kv_heads, self.head_size = pages, bs, hk, d
        self.args = PlainCacheArgs(k_cache.data_ptr(), v_cache.data_ptr(), pages, *strides, bs, hk, d,
                                   _rotary.DTYPES[k_cache.dtype])
        self.address = ctypes.addressof(self.args)
        self.geometry = (hk, d, bs)


class QuantCacheArgs(ctypes.Structure):
    """struct oscar_quant_cache (include/oscar_amd.h)."""
    _fields_ = [("k", _p), ("v", _p), ("exponents", _p), ("num_pages", _i64), ("k_stride_page", _i64),
                ("k_stride_token", _i64), ("k_stride_head", _i64), ("v_stride_page", _i64), ("v_stride_token", _i64),
                ("v_stride_head", _i64), ("block_size", _i32), ("num_kv_heads", _i32), ("head_size", _i32),
                ("dtype", _i32)]


class QuantCache:
    """A layer's 8-bit K and V pages, checked and packed once: codes [pages,
    block_size, Hk, D] (float8_e4m3fn, or their bytes as uint8) that stand for
    code * 2^(b - 127), b the byte at exponents [pages, Hk, block_size, 2] (uint8,
    contiguous; K's, then V's): 47 to 227 in bf16, 112 to 135 in fp16 (135 with codes up
    to 240), of codes of zero any.  dtype (bf16 or fp16) is that of the rows that are
    written and read; the values are exact in it.  Codes may be views as PagedCache's may;
    D is a multiple of 16."""

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype):
        if k_codes.ndim != 4 or k_codes.shape != v_codes.shape or min(k_codes.shape) < 1:
            raise ValueError("K and V codes must share [pages, block_size, heads, head size]")
        if k_codes.dtype not in (torch.float8_e4m3fn, torch.uint8) or v_codes.dtype != k_codes.dtype:
            raise ValueError("codes are float8_e4m3fn or uint8, K and V alike")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"an 8-bit cache's rows are bf16 or fp16, got {dtype}")
        pages, bs, hk, d = k_codes.shape
        if d % 16 or d > 256:
            raise ValueError(f"head size {d} must be a multiple of 16, at most 256")
        if (exponents.shape != (pages, hk, bs, 2) or exponents.dtype != torch.uint8 or not exponents.is_contiguous()
                or exponents.data_ptr() % 16):
            raise ValueError("exponents must be a contiguous uint8 [pages, heads, block_size, 2] tensor at a multiple of "
                             "16 bytes")
        if k_codes.device != v_codes.device or exponents.device != k_codes.device:
            raise ValueError("codes and exponents must be on one device")
        strides = [s for x in (k_codes, v_codes) for s in _code_strides(x)]
        self.k_codes, self.v_codes, self.exponents = k_codes, v_codes, exponents
        self.device, self.dtype, self.on_gpu = k_codes.device, dtype, k_codes.is_cuda
        self.pages, self.block_size, self.num_kv_heads, self.head_size = pages, bs, hk, d
        self.args = QuantCacheArgs(k_codes.data_ptr(), v_codes.data_ptr(), exponents.data_ptr(), pages, *strides, bs, hk,
                                   d, _rotary.DTYPES[dtype])
        self.address = ctypes.addressof(self.args)
        self.geometry = (hk, d, bs, 8)     # (never a plain cache's)


def _code_strides(x: torch.Tensor) -> tuple[int, int, int]:
    """Page, token and head strides of codes, in bytes."""
    pages, bs, hk, d = x.shape
    page, token, head, feature = x.stride()
    # strides of axes of one entry mean nothing
    token = token if bs > 1 else d
    head = head if hk > 1 else d
    tokens, heads = (bs - 1) * token + d, (hk - 1) * head + d
    page = page if pages > 1 else tokens + heads - d
    if feature != 1 or x.data_ptr() % 16 or page % 16 or token % 16 or head % 16 or min(page, token, head) < d:
        raise ValueError("rows of codes must be contiguous features at multiples of 16 bytes")
    nested = heads <= token if token > head else tokens <= head
    if (bs > 1 and hk > 1 and not nested) or (pages > 1 and page < tokens + heads - d):
        raise ValueError("cache tokens, heads or pages overlap")
    if tokens + heads - d >= 1 << 31:
        raise ValueError("a cache page must span less than 2 GiB")
    return page, token, head


def quant_cache(pages: int, block_size: int, num_kv_heads: int, head_size: int, dtype: torch.dtype,
                device) -> QuantCache:
    """A new 8-bit cache of zeros."""
    codes = [torch.zeros(pages, block_size, num_kv_heads, head_size, dtype=torch.uint8, device=device)
             for _ in range(2)]
    exponents = torch.zeros(pages, num_kv_heads, block_size, 2, dtype=torch.uint8, device=device)
    return QuantCache(*codes, exponents, dtype)


def append_rotated(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                   rotary: _rotary.Rotary, cache: PagedCache, slot_mapping: torch.Tensor, query_out=None):
    """Write key (turned by its positions) and value [N, Hk, D] of the tokens of
    slot_mapping (int64 [N]) to their slots, and return query [N, Hq, D] turned
    (a new tensor, or query_out: query itself or apart from the call's rows; None
    without a query).  Rows are of the cache's type, with any token and head strides
    below 4 GiB; rows past the slots' count are not read.  Slots < 0 or past the cache are
    skipped, tokens with a position outside the table left out whole; slots of a
    call are distinct.  For serving: no autograd graph is recorded."""
    if not isinstance(cache, PagedCache):
        raise ValueError("append_rotated writes plain caches (append_quantized 8-bit ones)")
    return _append("oscar_append_rotated", (), query, key, value, positions, rotary, cache, slot_mapping, query_out)


def append_normed(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                  rotary: _rotary.Rotary, cache: PagedCache, slot_mapping: torch.Tensor, query_weight, key_weight,
                  eps: float = 1e-6, offset: float = 0.0, query_out=None):
    """append_rotated with queries and keys normed before they are turned, by weights
    [D] as ``rotary.norm_rotate`` takes them (None: that kind has no norm)."""
    if not isinstance(cache, PagedCache):
        raise ValueError("append_normed writes plain caches (append_quantized 8-bit ones)")
    norm = _rotary.pack_norm(query_weight if query is not None else None, key_weight, eps, offset, cache.head_size,
                             cache.device)
    return _append("oscar_append_normed", (norm,), query, key, value, positions, rotary, cache, slot_mapping, query_out)


def append_quantized(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                     rotary: _rotary.Rotary, cache: QuantCache, slot_mapping: torch.Tensor, query_weight=None,
                     key_weight=None, eps: float = 1e-6, offset: float = 0.0, query_out=None):
    """The same write to an 8-bit cache: queries and keys normed where they have a
    weight, and turned; keys and values rounded to e4m3 codes (to nearest, ties to even)
    times a power of two for each token and head, the smallest with which the row's
    largest finite magnitude is at most 448 times it (2^-80 to 2^100 in bf16, 2^-15 to
    2^8 in fp16; under the greatest, values past 240 times it become that).  What is not
    finite becomes NaN."""
    if not isinstance(cache, QuantCache):
        raise ValueError("append_quantized writes 8-bit caches (append_rotated and append_normed plain ones)")
    norm = _rotary.pack_norm(query_weight if query is not None else None, key_weight, eps, offset, cache.head_size,
                             cache.device)
    return _append("oscar_append_quantized", (norm,), query, key, value, positions, rotary, cache, slot_mapping,
                   query_out)


def _append(entry, norm, query, key, value, positions, rotary, cache, slot_mapping, query_out):
    if slot_mapping.ndim != 1 or slot_mapping.device != cache.device:
        raise ValueError("slot_mapping must be [tokens], on the cache's device")
    n, d, dtype, device = slot_mapping.shape[0], cache.head_size, cache.dtype, cache.device
    if d < rotary.rotary_dim:
        raise ValueError(f"head size {d} is below rotary_dim {rotary.rotary_dim}")
    k, hk = _rotary.heads(key, n, d, dtype, device, "key")
    v, hv = _rotary.heads(value, n, d, dtype, device, "value")
    if hk != cache.num_kv_heads or hv != cache.num_kv_heads:
        raise ValueError(f"key and value must have the cache's {cache.num_kv_heads} heads")
    q = qo = None
    if query is not None:
        q, hq = _rotary.heads(query, n, d, dtype, device, "query")
        if query_out is None:
            query_out, qo = _rotary.new_heads(query, n, hq, d)
        else:
            qo = _rotary.out_heads(query_out, n, hq, d, dtype, device, "query_out")
    slot_mapping = _slots(slot_mapping, n)
    positions, axis_stride = _rotary.positions_of(positions, rotary, n, device)
    if not cache.on_gpu:
        raise ValueError("OSCAR kernels take device tensors")
    if n:
        _lib.call_on(device, entry, rotary.address, *norm, positions.data_ptr(), axis_stride, n, q, qo, k, v,
                     cache.address, slot_mapping.data_ptr())
    return query_out if query is not None else None


def _slots(slots: torch.Tensor, n: int) -> torch.Tensor:
    if slots.dtype is not torch.int64 or (n > 1 and slots.stride(0) != 1):
        if slots.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"slot_mapping must be integers, got {slots.dtype}")
        slots = slots.to(torch.int64).contiguous()
    return slots


def read_back(cache: QuantCache, slot_mapping: torch.Tensor, dtype=None, key_out=None, value_out=None):
    """Keys and values [N, Hk, D] of the slots (int64 [N]) of an 8-bit cache, as the
    values they stand for, exactly: of the cache's type, or fp32 with dtype=torch.float32;
    new tensors, or the ones given (rows at multiples of 16 bytes, apart).  Slots < 0 or
    past the cache give zeros; a slot may come more than once."""
    if not isinstance(cache, QuantCache):
        raise ValueError("read_back reads 8-bit caches")
    if slot_mapping.ndim != 1 or slot_mapping.device != cache.device:
        raise ValueError("slot_mapping must be [tokens], on the cache's device")
    dtype = cache.dtype if dtype is None else dtype
    if dtype not in (cache.dtype, torch.float32):
        raise ValueError(f"rows are read as {cache.dtype} or float32, got {dtype}")
    n, d, hk, device = slot_mapping.shape[0], cache.head_size, cache.num_kv_heads, cache.device
    outs, packed = [], []
    for x, what in ((key_out, "key_out"), (value_out, "value_out")):
        if x is None:
            x = torch.empty((n, hk, d), dtype=dtype, device=device)
            packed.append(_rotary.pack_heads(x.data_ptr(), hk * d, d, hk, 0))
        else:
            packed.append(_rotary.out_heads(x, n, hk, d, dtype, device, what))
            token, head, _ = x.stride()
            at = x.data_ptr() | (token * x.element_size() if n > 1 else 0) | (head * x.element_size() if hk > 1 else 0)
            if at % 16:
                raise ValueError(f"{what} must have rows at multiples of 16 bytes")
        outs.append(x)
    slot_mapping = _slots(slot_mapping, n)
    if not cache.on_gpu:
        raise ValueError("OSCAR kernels take device tensors")
    if n:
        _lib.call_on(device, "oscar_read_back", cache.address, slot_mapping.data_ptr(), n, *packed, _rotary.DTYPES[dtype])
    return outs[0], outs[1]
