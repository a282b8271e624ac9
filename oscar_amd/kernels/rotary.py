"""Position rotation of query and key heads (oscar_rotate_positions), and their
norms with it (oscar_norm_rotate).

The INT2 write and the attention impl take queries and keys that already carry
their positions; this is the rotation that puts them there, on one axis for
text or on several (time, height, width) for image and video prompts.  The
heads' first ``rotary_dim`` features turn in pairs by the cosines and sines of
a table (one row per position, cosines first: the layout serving engines keep),
in fp32 with one rounding; the rest pass through.  The map is orthogonal, so
``inverse=True`` both takes positions off and gives the gradient, which autograd
takes too.  Models that norm each head before its position have both in one pass
(``norm_rotate``), the gradients of heads and weights too.
"""
from __future__ import annotations

import ctypes
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_ROTARY_DIM = 256
MAX_AXES = 4

_p, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class RotaryArgs(ctypes.Structure):
    """struct oscar_rotary (include/oscar_amd.h)."""
    _fields_ = [("table", _p), ("positions", _i64), ("rotary_dim", _i32), ("adjacent", _i32), ("axes", _i32),
                ("reserved", _i32), ("pair_axis", ctypes.c_uint64 * 4)]


class HeadsArgs(ctypes.Structure):
    """struct oscar_heads (include/oscar_amd.h)."""
    _fields_ = [("data", _p), ("token_stride", _i64), ("head_stride", _i64), ("num_heads", _i32), ("reserved", _i32)]


def rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """fp32 [positions, rotary_dim]: the cosines, then the sines, of position *
    base^(-2j / rotary_dim), from angles in 64 bits (in 32, positions past 2^17
    would be off by more than the table's own rounding)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    turn = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * turn
    return torch.cat((angle.cos(), angle.sin()), -1).to(device=device, dtype=torch.float32)


def section_axes(sections, interleaved: bool = False) -> list:
    """The position axis of every feature pair, from how many pairs each axis
    has: in blocks (all of the first axis, then the next), or interleaved (the
    axes in turn until an axis but the first has had its share, the rest on the
    first)."""
    sections = [int(s) for s in sections]
    if not 1 <= len(sections) <= MAX_AXES or any(s < 0 for s in sections) or sum(sections) < 1:
        raise ValueError(f"sections are 1 to {MAX_AXES} pair counts")
    pairs, n = sum(sections), len(sections)
    if not interleaved:
        return [axis for axis, count in enumerate(sections) for _ in range(count)]
    axes = [j % n if j // n < sections[j % n] else 0 for j in range(pairs)]
    if any(axes.count(axis) != count for axis, count in enumerate(sections)):
        raise ValueError(f"sections {sections} cannot be interleaved: an axis but the first has too many pairs")
    return axes


class Rotary:
    """A model's position rotation, checked and packed once: the table (fp32
    [positions, rotary_dim]), whether pairs are adjacent features or halves of
    the rotary part, and, for positions on several axes, the axis of every pair
    (``section_axes``)."""

    def __init__(self, table: torch.Tensor, adjacent: bool = False, axes=None):
        if table.ndim != 2 or table.dtype != torch.float32 or not table.is_contiguous() or table.shape[0] < 1:
            raise ValueError("the rotary table must be a contiguous fp32 [positions, rotary_dim] tensor")
        rd = table.shape[1]
        if rd < 2 or rd % 2 or rd > MAX_ROTARY_DIM:
            raise ValueError(f"rotary_dim {rd} must be even, 2 to {MAX_ROTARY_DIM}")
        axes = [0] * (rd // 2) if axes is None else [int(a) for a in axes]
        if len(axes) != rd // 2 or min(axes) < 0 or max(axes) >= MAX_AXES:
            raise ValueError(f"axes must name one of {MAX_AXES} position axes for each of the {rd // 2} pairs")
        self.table = table
        self.device = table.device
        self.rotary_dim = rd
        self.axes = max(axes) + 1
        words = [0] * 4
        for j, a in enumerate(axes):
            words[j // 32] |= a << (2 * (j % 32))
        self.args = RotaryArgs(table.data_ptr(), table.shape[0], rd, int(adjacent), self.axes, 0,
                               (ctypes.c_uint64 * 4)(*words))
        self.address = ctypes.addressof(self.args)


# struct oscar_heads as bytes, which a call passes by their address: packing them
# takes a fifth of what filling a ctypes structure does.
pack_heads = struct.Struct("@Pqqii").pack


def heads(x: torch.Tensor, tokens: int, d: int, dtype, device, what: str) -> tuple[bytes, int]:
    """(struct oscar_heads, heads) of the first tokens of x [N, heads, d]."""
    shape = x.shape
    if len(shape) != 3 or shape[0] < tokens or shape[2] != d:
        raise ValueError(f"{what} must be [tokens, heads, {d}] with a row per token")
    if x.dtype is not dtype or x.device != device:
        raise ValueError(f"{what} must be {dtype} on {device} as the other rows are")
    token, head, feature = x.stride()
    if feature != 1:
        raise ValueError(f"{what}: a head's features must be contiguous")
    return pack_heads(x.data_ptr(), token, head, shape[1], 0), shape[1]


def out_heads(x: torch.Tensor, tokens: int, count: int, d: int, dtype, device, what: str) -> bytes:
    """heads() of an output of `count` heads, whose rows do not share memory."""
    packed, given = heads(x, tokens, d, dtype, device, what)
    if given != count:
        raise ValueError(f"{what} must have the {'key' if what == 'key_out' else 'query'}'s heads")
    token, head, _ = x.stride()
    token, head = token if tokens > 1 else d, head if count > 1 else d      # (of one entry they mean nothing)
    apart = head >= (tokens - 1) * token + d if token < head else token >= (count - 1) * head + d
    if min(token, head) < d or (tokens > 1 and count > 1 and not apart):
        raise ValueError(f"{what}: rows overlap")
    return packed


def new_heads(like: torch.Tensor, tokens: int, count: int, d: int) -> tuple[torch.Tensor, bytes]:
    """A new tensor [tokens, count, d] of like's type and device, and its struct oscar_heads."""
    x = like.new_empty((tokens, count, d))
    return x, pack_heads(x.data_ptr(), count * d, d, count, 0)


def positions_of(positions: torch.Tensor, rotary: Rotary, tokens: int, device) -> tuple[torch.Tensor, int]:
    """int64 positions [N], or [axes, N], and the stride between axes."""
    if positions.dtype is not torch.int64:
        if positions.dtype not in (torch.int32, torch.int16):
            raise ValueError(f"positions must be integers, got {positions.dtype}")
        positions = positions.to(torch.int64)
    if positions.device != device or rotary.device != device:
        raise ValueError("positions and rotary table must be on the rows' device")
    shape = positions.shape
    if (len(shape) not in (1, 2) or shape[-1] < tokens or (len(shape) == 1 and rotary.axes != 1)
            or (len(shape) == 2 and shape[0] != rotary.axes)):
        raise ValueError(f"positions must be [{rotary.axes}, tokens] with an entry per token"
                         + (" (or [tokens])" if rotary.axes == 1 else ""))
    if positions.stride(-1) != 1 and tokens > 1:
        positions = positions.contiguous()
    return positions, positions.stride(0) if len(shape) == 2 else 0


def rotate(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, query_out=None,
           key_out=None, inverse: bool = False):
    """query [N, Hq, D] and key [N, Hk, D] (or None) turned by their positions
    (int64 [N], or [axes, N]), bf16, fp16 or fp32 alike, with any token and head
    strides below 4 GiB.  Returns (query_out, key_out): new tensors, or the ones
    given, each its own input as it stands or apart from all rows of the call.
    New tensors carry a gradient to rows that require one (theirs, turned the
    other way); a call with a given output records no autograd graph.  Rows that carry
    forward mode's tangents are refused.  A token with a position outside the table is
    left out: its output rows keep what they held, and its inputs' gradient is zero."""
    _refuse_tangents(query, key)
    if ((query.requires_grad or (key is not None and key.requires_grad)) and torch.is_grad_enabled()
            and query_out is None and key_out is None):
        if key is not None and key.shape[0] > query.shape[0]:
            key = key[:query.shape[0]]
        return _Turned.apply(query, key, positions, rotary, inverse, False)
    return _rotate(query, key, positions, rotary, query_out, key_out, inverse)


def _refuse_tangents(*tensors) -> None:
    """Raise for dual tensors of forward mode, whose tangents a kernel's output would not have."""
    if getattr(forward_ad, "_current_level", -1) >= 0 and any(
            x is not None and forward_ad.unpack_dual(x).tangent is not None for x in tensors):
        raise ValueError("rows and weights carry tangents: there are no forward-mode gradients")


class _Turned(torch.autograd.Function):
    """rotate() into new tensors, zeros where a token is left out if `blank`.  Its
    gradient is such a rotation the other way, itself with a gradient."""

    @staticmethod
    def forward(ctx, query, key, positions, rotary, inverse, blank):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.back = (rotary, not inverse, True)
        outs = [torch.zeros_like(x, memory_format=torch.contiguous_format) if blank and x is not None else None
                for x in (query, key)]
        return _rotate(query, key, positions, rotary, *outs, inverse)

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        # (a sum's gradient is one number, expanded)
        rows = [g if g.stride(-1) == 1 else g.contiguous()
                for g, needed in zip(grads, ctx.needs_input_grad) if needed and g is not None]
        turned = iter(_Turned.apply(*rows, *(None,) * (2 - len(rows)), positions, *ctx.back) if rows else ())
        return (*(next(turned) if needed and g is not None else None
                  for g, needed in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def _rotate(query, key, positions, rotary, query_out, key_out, inverse):
    dtype, device = query.dtype, query.device
    if dtype not in DTYPES:
        raise ValueError(f"rotate takes bf16, fp16 or fp32 rows, got {dtype}")
    if query.ndim != 3:
        raise ValueError("query must be [tokens, heads, head size]")
    n, _, d = query.shape
    if d < rotary.rotary_dim or d % 2 or d > 256:
        raise ValueError(f"head size {d} must be even, {rotary.rotary_dim} (rotary_dim) to 256")
    q, hq = heads(query, n, d, dtype, device, "query")
    if query_out is None:
        query_out, qo = new_heads(query, n, hq, d)
    else:
        qo = out_heads(query_out, n, hq, d, dtype, device, "query_out")
    k = ko = None
    if key is not None:
        k, hk = heads(key, n, d, dtype, device, "key")
        if key_out is None:
            key_out, ko = new_heads(key, n, hk, d)
        else:
            ko = out_heads(key_out, n, hk, d, dtype, device, "key_out")
    positions, axis_stride = positions_of(positions, rotary, n, device)
    if not query.is_cuda:
        raise ValueError("OSCAR kernels take device tensors")
    if n:
        _lib.call_on(device, "oscar_rotate_positions", rotary.address, positions.data_ptr(), axis_stride, n, q, qo, k,
                     ko, d, DTYPES[dtype], int(inverse))
    return query_out, key_out if key is not None else None


# struct oscar_head_norm
_pack_norm = struct.Struct("@PPiffi").pack
MAX_FLOAT = 3.0e38


def pack_norm(query_weight, key_weight, eps: float, offset: float, d: int, device) -> bytes:
    """struct oscar_head_norm of weights [d] (None: that kind has no norm)."""
    if not 0.0 <= eps < MAX_FLOAT or not -MAX_FLOAT < offset < MAX_FLOAT:
        raise ValueError("eps must be finite and not negative, the offset finite")
    q, q_type = _weight(query_weight, d, device, "query_weight")
    k, k_type = _weight(key_weight, d, device, "key_weight")
    if q_type is not k_type and q and k:
        raise ValueError("query_weight and key_weight must be of one type")
    return _pack_norm(q, k, DTYPES.get(q_type or k_type, 0), eps, offset, 0)


def _weight(w, d: int, device, what: str):
    """(address, type) of a weight; (0, None) without one."""
    if w is None:
        return 0, None
    dtype = w.dtype
    if w.ndim != 1 or w.shape[0] != d or dtype not in DTYPES or w.device != device or not w.is_contiguous():
        raise ValueError(f"{what} must be a contiguous bf16, fp16 or fp32 [{d}] tensor on the rows' device")
    return w.data_ptr(), dtype


def norm_rotate(query: torch.Tensor, key: torch.Tensor | None, query_weight: torch.Tensor,
                key_weight: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, eps: float = 1e-6,
                offset: float = 0.0, query_out=None, key_out=None):
    """query [N, Hq, D] and key [N, Hk, D] (or None), each head normed and then turned
    by its token's position:
      x / sqrt(mean x^2 + eps) * (weight + offset), through ``rotate``,
    in fp32 with one rounding.  Weights are [D] of one type (bf16, fp16 or fp32), one
    for all query heads and one for all key heads; offset 1 is for models that keep
    them around zero.  Rows, positions and outputs are as ``rotate`` takes them.  New
    tensors carry a gradient to rows and weights that require one (a single time); a
    call with a given output records no autograd graph.  Rows and weights that carry
    forward mode's tangents are refused.  A token with a position outside the table is
    left out: its output rows keep what they held, and it adds nothing to a gradient."""
    _refuse_tangents(query, key, query_weight, key_weight)
    if query_weight is None or (key is not None and key_weight is None):
        raise ValueError("norm_rotate takes a weight for queries, and for keys where they are given")
    if key is None:
        key_weight = None
    if (query_out is None and key_out is None and torch.is_grad_enabled()
            and (query.requires_grad or query_weight.requires_grad
                 or (key is not None and (key.requires_grad or key_weight.requires_grad)))):
        if key is not None and key.shape[0] > query.shape[0]:
            key = key[:query.shape[0]]
        return _Normed.apply(query, key, query_weight, key_weight, positions, rotary, eps, offset)
    return _norm_rotate(query, key, query_weight, key_weight, positions, rotary, eps, offset, query_out, key_out)


class _Normed(torch.autograd.Function):
    """norm_rotate() into new tensors."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, rotary, eps, offset):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(query, key, query_weight, key_weight, positions)
        ctx.settings = rotary, eps, offset
        return _norm_rotate(query, key, query_weight, key_weight, positions, rotary, eps, offset, None, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        query, key, query_weight, key_weight, positions = ctx.saved_tensors
        rotary, eps, offset = ctx.settings
        n, _, d = query.shape
        device = query.device
        if n == 0:
            leaves = (query, key, query_weight, key_weight)
            return (*(torch.zeros_like(x) if needed else None for x, needed in zip(leaves, ctx.needs_input_grad)),
                    None, None, None, None)
        rows, back, weights, held = [], [None, None], [None, None], []
        for i, (x, w, g) in enumerate(((query, query_weight, grads[0]), (key, key_weight, grads[1]))):
            if g is None or not (ctx.needs_input_grad[i] or ctx.needs_input_grad[2 + i]):
                rows += [None, None, None]
                continue
            if g.stride(-1) != 1:           # (a sum's gradient is one number, expanded)
                g = g.contiguous()
            held.append(g)                  # (until the call: rows are addresses)
            rows += [heads(x, n, d, x.dtype, device, "rows")[0], heads(g, n, d, x.dtype, device, "gradient")[0], None]
            if ctx.needs_input_grad[i]:
                back[i], rows[-1] = new_heads(x, n, x.shape[1], d)
            if ctx.needs_input_grad[2 + i]:
                weights[i] = torch.empty_like(w)
        if any(x is not None for x in rows):
            positions, axis_stride = positions_of(positions, rotary, n, device)
            need = (_lib.load().oscar_norm_rotate_backward_workspace_bytes(n, d)
                    if any(w is not None for w in weights) else 0)
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            _lib.call_on(device, "oscar_norm_rotate_backward", rotary.address,
                         pack_norm(query_weight, key_weight, eps, offset, d, device), positions.data_ptr(), axis_stride,
                         n, *rows, *(_lib.ptr(w) for w in weights), d, DTYPES[query.dtype], _lib.ptr(ws), need)
        return (*back, *weights, None, None, None, None)


def _norm_rotate(query, key, query_weight, key_weight, positions, rotary, eps, offset, query_out, key_out):
    dtype, device = query.dtype, query.device
    if dtype not in DTYPES:
        raise ValueError(f"norm_rotate takes bf16, fp16 or fp32 rows, got {dtype}")
    if query.ndim != 3:
        raise ValueError("query must be [tokens, heads, head size]")
    n, _, d = query.shape
    if d < rotary.rotary_dim or d % 2 or d > 256:
        raise ValueError(f"head size {d} must be even, {rotary.rotary_dim} (rotary_dim) to 256")
    norm = pack_norm(query_weight, key_weight, eps, offset, d, device)
    q, hq = heads(query, n, d, dtype, device, "query")
    if query_out is None:
        query_out, qo = new_heads(query, n, hq, d)
    else:
        qo = out_heads(query_out, n, hq, d, dtype, device, "query_out")
    k = ko = None
    if key is not None:
        k, hk = heads(key, n, d, dtype, device, "key")
        if key_out is None:
            key_out, ko = new_heads(key, n, hk, d)
        else:
            ko = out_heads(key_out, n, hk, d, dtype, device, "key_out")
    positions, axis_stride = positions_of(positions, rotary, n, device)
    if not query.is_cuda:
        raise ValueError("OSCAR kernels take device tensors")
    if n:
        _lib.call_on(device, "oscar_norm_rotate", rotary.address, norm, positions.data_ptr(), axis_stride, n, q, qo, k,
                     ko, d, DTYPES[dtype])
    return query_out, key_out if key is not None else None
