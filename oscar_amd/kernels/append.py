"""Plain paged caches and their write (oscar_append_rotated).

The layers the INT2 impl leaves native (MTP draft layers, sliding-window
layers) keep keys and values as they are, in bf16 or fp16 pages.  One launch
turns a step's queries and keys by their positions and puts keys and values
into their slots.
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


def append_rotated(query: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                   rotary: _rotary.Rotary, cache: PagedCache, slot_mapping: torch.Tensor, query_out=None):
    """Write key (turned by its positions) and value [N, Hk, D] of the tokens of
    slot_mapping (int64 [N]) to their slots, and return query [N, Hq, D] turned
    (a new tensor, or query_out: query itself or apart from the call's rows; None
    without a query).  Rows are of the cache's type, with any token and head strides
    below 4 GiB; rows past the slots' count are not read.  Slots < 0 or past the cache are
    skipped, tokens with a position outside the table left out whole; slots of a
    call are distinct.  For serving: no autograd graph is recorded."""
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
    if slot_mapping.dtype is not torch.int64 or (n > 1 and slot_mapping.stride(0) != 1):
        if slot_mapping.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"slot_mapping must be integers, got {slot_mapping.dtype}")
        slot_mapping = slot_mapping.to(torch.int64).contiguous()
    positions, axis_stride = _rotary.positions_of(positions, rotary, n, device)
    if not cache.on_gpu:
        raise ValueError("OSCAR kernels take device tensors")
    if n:
        _lib.call_on(device, "oscar_append_rotated", rotary.address, positions.data_ptr(), axis_stride, n, q, qo, k, v,
                     cache.address, slot_mapping.data_ptr())
    return query_out if query is not None else None
