"""Normed heads and the 8-bit cache without a GPU: geometry, and what is refused before
anything is launched."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from oscar_amd.kernels import _lib, append, rotary

FAKE = 1 << 20


def codes(shape=(3, 16, 2, 64), dtype=torch.uint8):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype)


def exponents(shape=(3, 2, 16, 2)):
    return torch.zeros(shape, dtype=torch.uint8)


def cache(**over):
    args = dict(k_codes=codes(), v_codes=codes(), exponents=exponents(), dtype=torch.bfloat16)
    args.update(over)
    return append.QuantCache(**args)


def test_geometries():
    c = cache()
    assert (c.args.k_stride_page, c.args.k_stride_token, c.args.k_stride_head) == (16 * 128, 128, 64)
    both = codes((3, 2, 16, 2, 64), torch.float8_e4m3fn)
    c = cache(k_codes=both[:, 0], v_codes=both[:, 1])
    assert c.args.k_stride_page == 2 * 16 * 128 and c.args.v == both.data_ptr() + 16 * 128
    heads_first = codes((3, 2, 16, 64)).transpose(1, 2)
    c = cache(k_codes=heads_first, v_codes=heads_first)
    assert (c.args.k_stride_token, c.args.k_stride_head) == (64, 16 * 64)
    one = cache(k_codes=codes((1, 1, 1, 16)), v_codes=codes((1, 1, 1, 16)), exponents=exponents((1, 1, 1, 2)))
    assert min(one.args.k_stride_page, one.args.k_stride_token, one.args.k_stride_head) >= 16
    new = append.quant_cache(3, 16, 2, 64, torch.float16, "cpu")
    assert new.geometry[:3] == (2, 64, 16) and new.exponents.shape == (3, 2, 16, 2)


@pytest.mark.parametrize("over, match", [
    ({"v_codes": codes((3, 16, 2, 128))}, "share"), ({"k_codes": codes()[0], "v_codes": codes()[0]}, "share"),
    ({"v_codes": codes(dtype=torch.float8_e4m3fn)}, "alike"), ({"dtype": torch.float32}, "bf16 or fp16"),
    ({"k_codes": codes(dtype=torch.int8), "v_codes": codes(dtype=torch.int8)}, "float8_e4m3fn"),
    ({"k_codes": codes((3, 16, 2, 72)), "v_codes": codes((3, 16, 2, 72))}, "multiple of 16"),
    ({"k_codes": codes((3, 16, 2, 272)), "v_codes": codes((3, 16, 2, 272))}, "at most 256"),
    ({"exponents": exponents((3, 16, 2, 2))}, "exponents"), ({"exponents": exponents().int()}, "exponents"),
    ({"exponents": exponents((3, 2, 2, 16)).transpose(2, 3)}, "exponents"),
    ({"exponents": torch.zeros(193, dtype=torch.uint8)[1:].view(3, 2, 16, 2)}, "exponents"),
    ({"k_codes": codes((3, 16, 2, 128))[..., ::2]}, "16 bytes"),
    ({"k_codes": codes((3, 16, 2, 65))[..., 1:]}, "16 bytes"),
    ({"k_codes": codes((3, 1, 2, 64)).expand(3, 16, 2, 64)}, "16 bytes"),
    ({"k_codes": torch.zeros(40000, dtype=torch.uint8).as_strided((3, 16, 2, 64), (4096, 64, 64, 1))}, "overlap"),
    ({"k_codes": torch.zeros(40000, dtype=torch.uint8).as_strided((3, 16, 2, 64), (1024, 128, 64, 1))}, "overlap"),
])
def test_cache_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        cache(**over)


def norm_args(**over):
    args = dict(query=torch.zeros(5, 4, 64), key=torch.zeros(5, 2, 64), query_weight=torch.ones(64),
                key_weight=torch.ones(64), positions=torch.zeros(5, dtype=torch.int64),
                rotary=rotary.Rotary(rotary.rotary_table(8, 32)))
    args.update(over)
    return args


@pytest.mark.parametrize("over, match", [
    ({"query_weight": None}, "weight"), ({"key_weight": None}, "weight"), ({"query_weight": torch.ones(32)}, "weight"),
    ({"query_weight": torch.ones(64, dtype=torch.float64)}, "weight"), ({"key_weight": torch.ones(128)[::2]}, "weight"),
    ({"key_weight": torch.ones(64).bfloat16()}, "one type"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"offset": float("inf")}, "offset"),
    ({"query": torch.zeros(5, 4, 64, dtype=torch.float64)}, "bf16, fp16 or fp32"),
    ({"query": torch.zeros(5, 256)}, "heads"), ({"query": torch.zeros(5, 4, 30), "key": None}, "head size"),
    ({"query": torch.zeros(5, 4, 128)[..., ::2]}, "contiguous"), ({"key": torch.zeros(4, 2, 64)}, "key"),
    ({"key": torch.zeros(5, 2, 64, dtype=torch.float16)}, "key"), ({"query_out": torch.zeros(5, 3, 64)}, "heads"),
    ({"query_out": torch.zeros(5, 1, 64).expand(5, 4, 64)}, "overlap"),
    ({"positions": torch.zeros(4, dtype=torch.int64)}, "positions"), ({}, "device tensors"),
    ({"query": torch.zeros(5, 4, 64, requires_grad=True)}, "device tensors")])
def test_norm_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        rotary.norm_rotate(**norm_args(**over))


def append_args(**over):
    bf = torch.bfloat16
    args = dict(query=torch.zeros(5, 4, 64, dtype=bf), key=torch.zeros(5, 2, 64, dtype=bf),
                value=torch.zeros(5, 2, 64, dtype=bf), positions=torch.zeros(5, dtype=torch.int64),
                rotary=rotary.Rotary(rotary.rotary_table(8, 32)), cache=cache(),
                slot_mapping=torch.zeros(5, dtype=torch.int64))
    args.update(over)
    return args


PLAIN = append.PagedCache(*(torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16) for _ in range(2)))


@pytest.mark.parametrize("over, match", [
    ({"cache": PLAIN}, "8-bit caches"), ({"slot_mapping": torch.zeros(5)}, "integers"),
    ({"slot_mapping": torch.zeros(6, dtype=torch.int64)}, "key"), ({"key": torch.zeros(5, 2, 64)}, "key"),
    ({"value": torch.zeros(5, 3, 64, dtype=torch.bfloat16)}, "2 heads"),
    ({"query": torch.zeros(4, 4, 64, dtype=torch.bfloat16)}, "query"),
    ({"rotary": rotary.Rotary(rotary.rotary_table(8, 128))}, "rotary_dim"),
    ({"query_weight": torch.ones(32)}, "weight"), ({"eps": -1.0}, "eps"), ({}, "device tensors")])
def test_append_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        append.append_quantized(**append_args(**over))


def test_caches_of_the_other_kind_are_refused():
    args = append_args()
    with pytest.raises(ValueError, match="plain caches"):
        append.append_rotated(**args)
    with pytest.raises(ValueError, match="plain caches"):
        append.append_normed(**args, query_weight=None, key_weight=None)
    with pytest.raises(ValueError, match="8-bit"):
        append.read_back(PLAIN, args["slot_mapping"])


@pytest.mark.parametrize("over, match", [
    ({"slot_mapping": torch.zeros(5)}, "integers"), ({"slot_mapping": torch.zeros(5, 1)}, "tokens"),
    ({"dtype": torch.float16}, "read as"), ({"key_out": torch.zeros(5, 2, 64)}, "key_out"),
    ({"value_out": torch.zeros(5, 2, 65, dtype=torch.bfloat16)[..., 1:]}, "16 bytes"),
    ({"value_out": torch.zeros(5, 1, 64, dtype=torch.bfloat16)}, "heads"), ({}, "device tensors")])
def test_read_back_refuses(over, match):
    args = dict(cache=cache(), slot_mapping=torch.zeros(5, dtype=torch.int64))
    args.update(over)
    with pytest.raises(ValueError, match=match):
        append.read_back(**args)


# ------------------------------------------------------------------ the C entries' own checks (nothing is launched)
def heads(at=FAKE, token=128, head=64, count=2):
    return rotary.HeadsArgs(at, token, head, count, 0)


def norm_status(norm=None, turn=None, q=None, qo=None, d=64, dtype=0, tokens=5, pos=FAKE, key=None, ko=None):
    turn = rotary.Rotary(rotary.rotary_table(8, 32)) if turn is None else turn
    norm = rotary._pack_norm(FAKE, FAKE, 2, 1e-6, 0.0, 0) if norm is None else norm
    q, qo = heads() if q is None else q, heads() if qo is None else qo
    ref = lambda x: None if x is None else ctypes.byref(x)       # noqa: E731
    return _lib.load().oscar_norm_rotate(turn.address, norm, pos, 0, tokens, ref(q), ref(qo), ref(key), ref(ko), d,
                                         dtype, None)


def test_norm_entry_refuses():
    pack = rotary._pack_norm
    assert norm_status(tokens=0) == 0 and norm_status(tokens=-1) == -1
    for norm in (pack(FAKE, FAKE, 3, 1e-6, 0.0, 0), pack(FAKE, FAKE, 2, -1e-6, 0.0, 0),
                 pack(FAKE, FAKE, 2, float("nan"), 0.0, 0), pack(FAKE, FAKE, 2, 0.0, float("inf"), 0)):
        assert norm_status(norm=norm) == -1
    assert norm_status(dtype=3) == -1 and norm_status(d=30) == -2 and norm_status(d=258) == -2
    assert norm_status(pos=None) == -1 and norm_status(q=heads(at=None)) == -1
    assert norm_status(qo=heads(count=1)) == -1 and norm_status(q=heads(token=-128)) == -5
    assert norm_status(q=heads(token=1 << 32)) == -5 and norm_status(q=heads(token=1 << 61)) == -5
    assert norm_status(qo=heads(at=FAKE + 64)) == -6
    assert norm_status(key=heads(at=FAKE + 4096), ko=heads()) == -6


def test_backward_entry_refuses():
    turn = rotary.Rotary(rotary.rotary_table(8, 32))
    norm = rotary._pack_norm(FAKE, 0, 2, 1e-6, 0.0, 0)
    size = _lib.load().oscar_norm_rotate_backward_workspace_bytes(5, 64)
    assert size == 5 * 2 * 64 * 4
    for args in ((0, 64), (-1, 64), (5, 0), (5, 258)):
        assert _lib.load().oscar_norm_rotate_backward_workspace_bytes(*args) == 0

    def status(x=heads(), g=heads(at=FAKE + 4096), dx=heads(at=FAKE + 8192), key=None, dw=FAKE, ws=FAKE, need=size,
               dtype=0, norm=norm):
        ref = lambda x: None if x is None else ctypes.byref(x)   # noqa: E731
        return _lib.load().oscar_norm_rotate_backward(turn.address, norm, FAKE, 0, 5, ref(x), ref(g), ref(dx), ref(key),
                                                      ref(key), None, dw, None, 64, dtype, ws, need, None)

    assert status(need=size - 1) == -3 and status(ws=None) == -3 and status(ws=FAKE + 2) == -5
    assert status(g=None) == -1 and status(g=heads(count=1)) == -1 and status(dx=heads(at=FAKE + 9000, count=1)) == -1
    assert status(dx=heads()) == -6 and status(dx=heads(at=FAKE + 4096)) == -6
    assert status(key=heads(at=FAKE + 16384)) == -1      # (keys have no weight)
    assert status(dtype=3) == -1


def quant_status(entry="append", over=None, **change):
    c = append.QuantCacheArgs.from_buffer_copy(cache().args)
    for name, value in change.items():
        setattr(c, name, value)
    args = dict(key=heads(), value=heads(at=FAKE + 4096), slots=FAKE, dtype=0, tokens=5)
    args.update(over or {})
    k, v = args["key"], args["value"]
    if entry == "append":
        turn = rotary.Rotary(rotary.rotary_table(8, 32))
        return _lib.load().oscar_append_quantized(turn.address, rotary._pack_norm(0, 0, 0, 0.0, 0.0, 0), FAKE, 0,
                                                  args["tokens"], None, None, ctypes.byref(k), ctypes.byref(v),
                                                  ctypes.byref(c), args["slots"], None)
    return _lib.load().oscar_read_back(ctypes.byref(c), args["slots"], args["tokens"], ctypes.byref(k), ctypes.byref(v),
                                       args["dtype"], None)


@pytest.mark.parametrize("entry", ["append", "read"])
def test_quant_entries_refuse(entry):
    assert quant_status(entry, {"tokens": 0}) == 0 and quant_status(entry, {"tokens": -1}) == -1
    for change in ({"k": None}, {"exponents": None}, {"num_pages": 0}, {"block_size": 0}, {"dtype": 2}):
        assert quant_status(entry, **change) == -1
    for change in ({"head_size": 24}, {"head_size": 272}, {"head_size": 0}):
        assert quant_status(entry, **change) == -2
    for change in ({"k": FAKE + 8}, {"exponents": FAKE + 8}, {"k_stride_token": 136}, {"v_stride_head": 48},
                   {"k_stride_page": 1024}, {"k_stride_token": 64}, {"v_stride_token": 1 << 31}):
        assert quant_status(entry, **change) == -5
    assert quant_status(entry, {"key": heads(count=1)}) == -1 and quant_status(entry, {"slots": None}) == -1
    assert quant_status(entry, {"key": heads(token=-128)}) == -5


def test_read_entry_refuses():
    assert quant_status("read", {"dtype": 1}) == -1
    assert quant_status("read", {"key": heads(at=FAKE + 8)}) == -5
    assert quant_status("read", {"key": heads(token=132)}) == -5
    assert quant_status("read", {"key": heads(token=1 << 60)}) == -5
    assert quant_status("read", {"value": heads(at=FAKE + 128)}) == -6


@pytest.mark.parametrize("name, mirror", [("oscar_quant_cache", append.QuantCacheArgs)])
def test_structs_match_the_header(tmp_path, name, mirror):
    header = Path(__file__).resolve().parents[1] / "include" / "oscar_amd.h"
    text = re.sub(r"/\*.*?\*/", "", header.read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    fields = [f for f, _ in mirror._fields_]
    assert [re.findall(r"\w+", d)[-1] for d in body.split(";") if d.strip()] == fields
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oscar_amd.h"',
             'int main(void) { printf("%%zu\\n", sizeof(%s));' % name]
    lines += ['  printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f in fields]
    lines += ['  printf("%zu %zu %zu %zu\\n", sizeof(oscar_head_norm), offsetof(oscar_head_norm, weight_dtype),'
              ' offsetof(oscar_head_norm, eps), offsetof(oscar_head_norm, offset));']
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(header.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    want = [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]
    assert [int(x) for x in got] == want + [32, 16, 20, 24] and len(rotary._pack_norm(0, 0, 0, 0.0, 0.0, 0)) == 32
