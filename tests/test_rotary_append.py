"""Position rotation and the plain cache's write without a GPU: tables, axis
layouts, cache geometry, and what is refused before anything is launched."""
import ctypes
import math

import pytest
import torch

from oscar_amd.kernels import _lib, append, rotary


def test_table_holds_cosines_then_sines_of_64_bit_angles():
    table = rotary.rotary_table(70001, 8, base=100.0)
    assert table.shape == (70001, 8) and table.dtype == torch.float32
    for pos in (0, 1, 777, 70000):
        for j in range(4):
            angle = pos * 100.0 ** (-2 * j / 8)
            assert table[pos, j].item() == pytest.approx(math.cos(angle), abs=2.0 ** -24)
            assert table[pos, 4 + j].item() == pytest.approx(math.sin(angle), abs=2.0 ** -24)
    with pytest.raises(ValueError, match="even"):
        rotary.rotary_table(4, 7)


def test_section_axes():
    assert rotary.section_axes((2, 1, 1)) == [0, 0, 1, 2]
    assert rotary.section_axes((4, 2, 2), interleaved=True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rotary.section_axes((11, 11, 10), interleaved=True)[-3:] == [2, 0, 1]
    assert rotary.section_axes((5,)) == [0] * 5
    for bad in ((), (1, 2, 3, 4, 5), (0, 0), (3, -1)):
        with pytest.raises(ValueError, match="sections"):
            rotary.section_axes(bad)
    with pytest.raises(ValueError, match="interleaved"):
        rotary.section_axes((1, 5, 2), interleaved=True)


def test_rotary_packs_two_bits_a_pair():
    turn = rotary.Rotary(rotary.rotary_table(4, 128), axes=rotary.section_axes((16, 24, 24)))
    got = [(turn.args.pair_axis[j // 32] >> (2 * (j % 32))) & 3 for j in range(64)]
    assert got == [0] * 16 + [1] * 24 + [2] * 24 and turn.axes == 3
    assert rotary.Rotary(rotary.rotary_table(4, 128)).axes == 1


@pytest.mark.parametrize("table, axes", [
    (torch.zeros(4), None), (torch.zeros(4, 7), None), (torch.zeros(4, 258), None), (torch.zeros(0, 8), None),
    (torch.zeros(4, 8, dtype=torch.float16), None), (torch.zeros(8, 4).t(), None),
    (torch.zeros(4, 8), [0, 1]), (torch.zeros(4, 8), [0, 1, 2, 4]), (torch.zeros(4, 8), [0, 0, -1, 0])])
def test_rotary_refuses(table, axes):
    with pytest.raises(ValueError):
        rotary.Rotary(table, axes=axes)


def _cache(shape=(3, 16, 2, 64), dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_cache_geometries():
    c = append.PagedCache(_cache(), _cache())
    assert (c.args.k_stride_page, c.args.k_stride_token, c.args.k_stride_head) == (16 * 256, 256, 128)
    both = _cache((3, 2, 16, 2, 64))
    c = append.PagedCache(both[:, 0], both[:, 1])
    assert c.args.k_stride_page == 2 * 16 * 256 and c.args.v == both.data_ptr() + 16 * 256
    heads_first = _cache((3, 2, 16, 64)).transpose(1, 2)
    c = append.PagedCache(heads_first, heads_first)
    assert (c.args.k_stride_token, c.args.k_stride_head) == (128, 16 * 128)
    one = append.PagedCache(_cache((1, 1, 1, 64)), _cache((1, 1, 1, 64)))
    assert min(one.args.k_stride_page, one.args.k_stride_token, one.args.k_stride_head) >= 128


@pytest.mark.parametrize("k, v, match", [
    (_cache(), _cache((3, 16, 2, 128)), "share"), (_cache()[0], _cache()[0], "share"),
    (_cache(), _cache(dtype=torch.float16), "alike"),
    (_cache(dtype=torch.float32), _cache(dtype=torch.float32), "bf16 or fp16"),
    (_cache((3, 16, 2, 60)), _cache((3, 16, 2, 60)), "multiple of 8"),
    (_cache((3, 16, 2, 264)), _cache((3, 16, 2, 264)), "at most 256"),
    (_cache((3, 16, 2, 128))[..., ::2], _cache(), "16 bytes"),
    (_cache((3, 16, 2, 65))[..., 1:], _cache(), "16 bytes"),
    (_cache((3, 1, 2, 64)).expand(3, 16, 2, 64), _cache(), "16 bytes"),
    (_cache((1, 16, 2, 64)).expand(3, 16, 2, 64), _cache(), "16 bytes"),
    (torch.zeros(40000, dtype=torch.bfloat16).as_strided((3, 16, 2, 64), (4096, 64, 64, 1)), _cache(), "overlap"),
    (torch.zeros(40000, dtype=torch.bfloat16).as_strided((3, 16, 2, 64), (1024, 128, 64, 1)), _cache(), "overlap"),
])
def test_cache_refuses(k, v, match):
    with pytest.raises(ValueError, match=match):
        append.PagedCache(k, v)


def _rotate_args(**over):
    args = dict(query=torch.zeros(5, 4, 64), key=torch.zeros(5, 2, 64), positions=torch.zeros(5, dtype=torch.int64),
                rotary=rotary.Rotary(rotary.rotary_table(8, 32)))
    args.update(over)
    return args


@pytest.mark.parametrize("over, match", [
    ({"query": torch.zeros(5, 4, 64, dtype=torch.float64)}, "bf16, fp16 or fp32"),
    ({"query": torch.zeros(5, 256)}, "heads"),
    ({"query": torch.zeros(5, 4, 30), "key": None}, "head size"),
    ({"query": torch.zeros(5, 4, 258), "key": None}, "head size"),
    ({"query": torch.zeros(5, 4, 128)[..., ::2]}, "contiguous"),
    ({"key": torch.zeros(4, 2, 64)}, "key"), ({"key": torch.zeros(5, 2, 128)}, "key"),
    ({"key": torch.zeros(5, 2, 64, dtype=torch.float16)}, "key"),
    ({"query_out": torch.zeros(5, 3, 64)}, "heads"), ({"query_out": torch.zeros(4, 4, 64)}, "query_out"),
    ({"key_out": torch.zeros(5, 1, 64)}, "heads"),
    ({"query_out": torch.zeros(5, 1, 64).expand(5, 4, 64)}, "overlap"),
    ({"query_out": torch.zeros(1, 4, 64).expand(5, 4, 64)}, "overlap"),
    ({"key_out": torch.zeros(400).as_strided((5, 2, 64), (66, 64, 1))}, "overlap"),
    ({"key_out": torch.zeros(600).as_strided((5, 2, 64), (64, 256, 1))}, "overlap"),
    ({"positions": torch.zeros(4, dtype=torch.int64)}, "positions"),
    ({"positions": torch.zeros(5)}, "integers"), ({"positions": torch.zeros(3, 5, dtype=torch.int64)}, "positions"),
    ({"positions": torch.zeros(5, dtype=torch.int64), "rotary": rotary.Rotary(rotary.rotary_table(8, 32),
                                                                              axes=[0, 1] * 8)}, "positions"),
    ({}, "device tensors"),
])
def test_rotate_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        rotary.rotate(**_rotate_args(**over))


def _append_args(**over):
    bf = torch.bfloat16
    args = dict(query=torch.zeros(5, 4, 64, dtype=bf), key=torch.zeros(5, 2, 64, dtype=bf),
                value=torch.zeros(5, 2, 64, dtype=bf), positions=torch.zeros(5, dtype=torch.int64),
                rotary=rotary.Rotary(rotary.rotary_table(8, 32)), cache=append.PagedCache(_cache(), _cache()),
                slot_mapping=torch.zeros(5, dtype=torch.int64))
    args.update(over)
    return args


@pytest.mark.parametrize("over, match", [
    ({"slot_mapping": torch.zeros(5, 1, dtype=torch.int64)}, "slot_mapping"),
    ({"slot_mapping": torch.zeros(5)}, "integers"),
    ({"slot_mapping": torch.zeros(6, dtype=torch.int64)}, "key"),
    ({"key": torch.zeros(5, 2, 64)}, "key"), ({"value": torch.zeros(5, 2, 64, dtype=torch.float16)}, "value"),
    ({"key": torch.zeros(5, 1, 64, dtype=torch.bfloat16)}, "2 heads"),
    ({"value": torch.zeros(5, 3, 64, dtype=torch.bfloat16)}, "2 heads"),
    ({"query": torch.zeros(4, 4, 64, dtype=torch.bfloat16)}, "query"),
    ({"query_out": torch.zeros(5, 5, 64, dtype=torch.bfloat16)}, "query's heads"),
    ({"query_out": torch.zeros(5, 1, 64, dtype=torch.bfloat16).expand(5, 4, 64)}, "overlap"),
    ({"positions": torch.zeros(4, dtype=torch.int64)}, "positions"),
    ({"rotary": rotary.Rotary(rotary.rotary_table(8, 128))}, "rotary_dim"),
    ({}, "device tensors"),
])
def test_append_refuses(over, match):
    with pytest.raises(ValueError, match=match):
        append.append_rotated(**_append_args(**over))


# ------------------------------------------------------------------ the C entries' own checks (nothing is launched)
FAKE = 1 << 20


def _c_rotary(**over):
    args = rotary.RotaryArgs(FAKE, 8, 32, 0, 1, 0, (ctypes.c_uint64 * 4)())
    for name, value in over.items():
        if name == "pair_axis":
            args.pair_axis[0] = value
        else:
            setattr(args, name, value)
    return args


def _c_heads(n, data=FAKE):
    return rotary.HeadsArgs(data, n * 64, 64, n, 0)


def _c_cache(**over):
    args = append.PlainCacheArgs(FAKE, FAKE, 3, 4096, 256, 128, 4096, 256, 128, 16, 2, 64, 0)
    for name, value in over.items():
        setattr(args, name, value)
    return args


def _status(fn, *args):
    keep = [ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args]
    return getattr(_lib.load(), fn)(*keep)


INVALID, HEAD, GEOMETRY = -1, -2, -5


@pytest.mark.parametrize("over, head_size, dtype, status", [
    ({"rotary_dim": 31}, 64, 0, INVALID), ({"rotary_dim": 0}, 64, 0, INVALID), ({"rotary_dim": 258}, 256, 0, INVALID),
    ({"axes": 0}, 64, 0, INVALID), ({"axes": 5}, 64, 0, INVALID), ({"positions": 0}, 64, 0, INVALID),
    ({"table": None}, 64, 0, INVALID), ({"pair_axis": 4}, 64, 0, INVALID), ({}, 64, 3, INVALID), ({}, 64, -1, INVALID),
    ({}, 30, 0, HEAD), ({}, 258, 0, HEAD), ({}, 63, 0, HEAD)])
def test_rotate_entry_refuses(over, head_size, dtype, status):
    q = _c_heads(2)
    assert _status("oscar_rotate_positions", _c_rotary(**over), FAKE, 0, 5, q, q, None, None, head_size, dtype, 0,
                   None) == status


def test_rotate_entry_refuses_rows():
    q, r = _c_heads(2), _c_rotary()
    for query, out, key, key_out in ((q, None, None, None), (q, _c_heads(3), None, None), (q, q, q, None),
                                     (_c_heads(2, None), q, None, None), (q, _c_heads(2, None), None, None),
                                     (_c_heads(-1), _c_heads(-1), None, None)):
        assert _status("oscar_rotate_positions", r, FAKE, 0, 5, query, out, key, key_out, 64, 0, 0, None) == INVALID
    assert _status("oscar_rotate_positions", r, None, 0, 5, q, q, None, None, 64, 0, 0, None) == INVALID
    assert _status("oscar_rotate_positions", r, FAKE, 0, -1, q, q, None, None, 64, 0, 0, None) == INVALID
    assert _status("oscar_rotate_positions", None, FAKE, 0, 5, q, q, None, None, 64, 0, 0, None) == INVALID
    assert _status("oscar_rotate_positions", r, FAKE, 0, 0, q, q, None, None, 64, 0, 0, None) == 0
    assert _status("oscar_rotate_positions", r, FAKE, 0, 5, None, None, None, None, 64, 0, 0, None) == 0


@pytest.mark.parametrize("over, status", [
    ({"k": None}, INVALID), ({"num_pages": 0}, INVALID), ({"block_size": 0}, INVALID), ({"num_kv_heads": 0}, INVALID),
    ({"dtype": 2}, INVALID), ({"head_size": 60}, HEAD), ({"head_size": 264}, HEAD), ({"k": FAKE + 8}, GEOMETRY),
    ({"k_stride_token": 264}, GEOMETRY), ({"v_stride_head": 64}, GEOMETRY), ({"k_stride_token": 128}, GEOMETRY),
    ({"v_stride_page": 2048}, GEOMETRY), ({"v_stride_page": 1 << 33, "v_stride_token": 1 << 28}, GEOMETRY),
    ({"num_kv_heads": 3}, INVALID)])
def test_append_entry_refuses(over, status):
    h = _c_heads(2)
    if over == {"num_kv_heads": 3}:
        over = {"num_kv_heads": 3, "k_stride_token": 384, "v_stride_token": 384, "k_stride_page": 6144,
                "v_stride_page": 6144}
    assert _status("oscar_append_rotated", _c_rotary(), FAKE, 0, 5, None, None, h, h, _c_cache(**over), FAKE,
                   None) == status


def test_append_entry_refuses_rows():
    h, c, r = _c_heads(2), _c_cache(), _c_rotary()
    for query, out, key, value, slots in ((None, None, None, h, FAKE), (None, None, h, None, FAKE),
                                          (None, None, h, h, None), (h, None, h, h, FAKE),
                                          (None, None, _c_heads(1), h, FAKE)):
        assert _status("oscar_append_rotated", r, FAKE, 0, 5, query, out, key, value, c, slots, None) == INVALID
    assert _status("oscar_append_rotated", r, FAKE, 0, 5, None, None, h, h, None, FAKE, None) == INVALID
    assert _status("oscar_append_rotated", _c_rotary(rotary_dim=128), FAKE, 0, 5, None, None, h, h, c, FAKE,
                   None) == HEAD
    assert _status("oscar_append_rotated", r, FAKE, 0, 0, None, None, h, h, c, None, None) == 0


def test_argument_structs_match_the_header(tmp_path):
    import re
    import subprocess
    from pathlib import Path

    header = Path(__file__).resolve().parents[1] / "include" / "oscar_amd.h"
    structs = {"oscar_rotary": rotary.RotaryArgs, "oscar_heads": rotary.HeadsArgs,
               "oscar_plain_cache": append.PlainCacheArgs}
    text = re.sub(r"/\*.*?\*/", "", header.read_text(), flags=re.S)
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oscar_amd.h"', "int main(void) {"]
    want = []
    for cname, cls in structs.items():
        body = re.search(r"typedef struct " + cname + r" \{(.*?)\} " + cname + ";", text, flags=re.S).group(1)
        declared = [re.findall(r"\w+", d.split("[")[0])[-1] for d in body.split(";") if d.strip()]
        assert declared == [f for f, _ in cls._fields_], cname
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {field}));')
            want.append(getattr(cls, field).offset)
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(header.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no device memory")
def test_strides_of_single_rows_are_not_looked_at():
    """Without a GPU what passes the checks ends at the launch (-4)."""
    r, far = _c_rotary(), 1 << 40

    def status(tokens, token, heads, head):
        x = rotary.HeadsArgs(FAKE, token, head, heads, 0)
        return _status("oscar_rotate_positions", r, FAKE, 0, tokens, x, x, None, None, 64, 0, 0, None)

    assert status(1, far, 2, 64) == status(1, -1, 2, 64) == status(5, 64, 1, far) == status(5, 64, 1, -1) == -4
    assert status(2, far, 2, 64) == status(2, -64, 2, 64) == status(5, 64, 2, far) == GEOMETRY


# ------------------------------------------------------------------ outputs and the rows they may lie among
OVERLAP, LAUNCHED = -6, -4          # (without a GPU what passes the checks ends at the launch)
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are host memory")


def _view(x):
    token, head, _ = x.stride()
    return rotary.HeadsArgs(x.data_ptr(), token, head, x.shape[1], 0)


def _rotate_views(q, qo, k=None, ko=None):
    views = [None if x is None else _view(x) for x in (q, qo, k, ko)]
    return _status("oscar_rotate_positions", _c_rotary(rotary_dim=2), FAKE, 0, len(q), *views, q.shape[2], 2, 0, None)


def _memory(x):
    token, head, _ = x.stride()
    return {x.storage_offset() + t * token + h * head + f for t in range(x.shape[0]) for h in range(x.shape[1])
            for f in range(x.shape[2])}


@no_gpu
def test_rows_that_share_memory_never_count_as_apart():
    """Random views of one store as output and input: refused whenever they share a
    value, and, all but the tangled ones, only then."""
    import random

    rng, store, passed, apart = random.Random(1), torch.zeros(4096), 0, 0
    for _ in range(4000):
        tokens, d = rng.choice((1, 2, 3, 5)), rng.choice((2, 4, 8))
        strides = [rng.choice((0, 2, 4, 8, 12, 16, 24, 40)) for _ in range(4)]
        if rng.random() < 0.5:
            strides[2:] = strides[:2]
        heads = rng.choice((1, 2, 4))
        x, y = (store.as_strided((tokens, heads, d), (*strides[2 * i:2 * i + 2], 1), rng.randint(0, 60))
                for i in range(2))
        same = all(a == b for a, b, n in zip((x.data_ptr(), *x.stride()), (y.data_ptr(), *y.stride()),
                                             (9, tokens, heads)) if n > 1)
        truth, status = not _memory(x) & _memory(y), _rotate_views(x, y)
        assert status in (OVERLAP, LAUNCHED) and (status == OVERLAP or truth or same)
        passed, apart = passed + (status == LAUNCHED and not same), apart + truth
    assert passed > 0.9 * apart > 1000


@no_gpu
@pytest.mark.parametrize("views, status", [
    (lambda x: (x[:, :2], x[:, 2:4], x[:, 2:4], x[:, :2]), OVERLAP),                     # exchanged
    (lambda x: (x[:, :4], x[:, 2:6], None, None), OVERLAP),                              # two heads further on
    (lambda x: (x[:4], x[1:5], None, None), OVERLAP),                                    # a token further on
    (lambda x: (x[:4], x[:8:2], None, None), OVERLAP),                                   # another stride
    (lambda x: (x[:, :4], x[:, 6:10], x[:, 10:], x[:, 2:4]), OVERLAP),                   # keys onto queries
    (lambda x: (x[:, :4], x[:, 9:11].repeat(1, 2, 1), x[:, 4:6], x[:, 3:5]), OVERLAP),
    (lambda x: (x[:, :2], x[:, 4:6], x[:, 6:8], x[:, 4:6]), OVERLAP),                    # both to one place
    (lambda x: (x[:, :2], x[:, 4:6], x[:, 4:6], x[:, 6:8]), OVERLAP),                    # queries onto keys
    (lambda x: (x[:, :4], x[:, :4], x[:, 4:6], x[:, 4:6]), LAUNCHED),                    # in place
    (lambda x: (x[:, :4], x[:, 6:10], x[:, 4:6], x[:, 10:]), LAUNCHED),                  # slices of one projection
    (lambda x: (x[:4, :4], x[4:, :4], x[:4, 4:6], x[4:, 4:6]), LAUNCHED),                # tokens of one tensor
    (lambda x: (x[:1, :4], x[:1, :4].as_strided((1, 4, 64), (1, 64, 1)), None, None), LAUNCHED),
    (lambda x: (x[:, ::3], x[:, ::3], x[:, 1::3], x[:, 1::3]), LAUNCHED),                # heads in turn
    (lambda x: (x[:, ::3], x[:, 2::3], x[:, 1::3], None), INVALID),
    (lambda x: (x.transpose(0, 1)[:, :3], x.transpose(0, 1)[:, 3:6], None, None), LAUNCHED)])     # heads first
def test_outputs_among_the_calls_rows(views, status):
    assert _rotate_views(*views(torch.zeros(8, 12, 64))) == status


@no_gpu
@pytest.mark.parametrize("first, status", [(0, LAUNCHED), (8, LAUNCHED), (1, OVERLAP), (4, OVERLAP), (6, OVERLAP)])
def test_append_refuses_outputs_among_its_rows(first, status):
    x = torch.zeros(5, 12, 64, dtype=torch.bfloat16)       # queries, 2 heads of keys, 2 of values, 4 more
    q, k, v, out = (_view(x[:, a:b]) for a, b in ((0, 4), (4, 6), (6, 8), (first, first + 4)))
    assert _status("oscar_append_rotated", _c_rotary(), FAKE, 0, 5, q, out, k, v, _c_cache(), FAKE, None) == status
