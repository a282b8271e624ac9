"""The plan of the attention over the 8-bit cache, and what is refused, without a GPU."""
import ctypes
import re
import struct
import subprocess
from pathlib import Path

import pytest
import torch

from oscar_amd.kernels import _lib, append, chunk, rotary
from tests.test_chunk_attention import JOIN, PIECE, ints
from tests.test_shared_prefix import PART, STEPS

SOURCE = struct.Struct("4i")


def quant_cache(pages=4, page=16, hk=2, d=128, dtype=torch.bfloat16):
    return append.quant_cache(pages, page, hk, d, dtype, "cpu")


def plan(starts, seqs, heads, cache, window=0, prefixes=(), status=0):
    args, q, s, flat = chunk.QuantStepArgs(), ints(starts), ints(seqs), ints([x for p in prefixes for x in p])
    call = [ctypes.addressof(q), ctypes.addressof(s), len(seqs), heads, window, ctypes.addressof(flat), len(prefixes),
            cache.address]
    assert _lib.load().oscar_quant_plan(*call, None, 0, ctypes.byref(args)) == status
    if status:
        return None
    size = args.chunk.items_size
    items = ctypes.create_string_buffer(max(size, 1))
    _lib.call("oscar_quant_plan", *call, ctypes.addressof(items), size, ctypes.byref(args))
    if size:
        assert _lib.load().oscar_quant_plan(*call, ctypes.addressof(items), size - 1, ctypes.byref(args)) == -3
    a = args.chunk
    at = PIECE.size * (a.narrow + a.wide)
    end = at + JOIN.size * a.joins + PART.size * a.parts
    assert size == end + SOURCE.size * args.sources
    return (args, [PIECE.unpack_from(items, PIECE.size * i) for i in range(a.narrow + a.wide)],
            [SOURCE.unpack_from(items, end + SOURCE.size * i) for i in range(args.sources)])


@pytest.mark.parametrize("d, hk, group", [(64, 4, 4), (256, 1, 6), (128, 2, 40)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("reqs, prefixes", [([(1, 0)], ()), ([(9256, 15360)], ()),
                                            ([(4, 5000), (0, 7), (1024, 4096), (4, 333), (300, 31)], ()), *STEPS])
def test_wide_pieces_find_their_keys(reqs, prefixes, window, d, hk, group):
    if window and prefixes:
        return
    starts, seqs = [0], []
    for n, h in reqs:
        starts.append(starts[-1] + n)
        seqs.append(n + h)
    args, pieces, sources = plan(starts, seqs, hk * group, quant_cache(d=d, hk=hk), window, prefixes)
    a = args.chunk
    owner = {}
    for row, group0, groups, page0 in sources:
        assert groups > 0 and page0 == len(owner)
        for i in range(groups):
            owner[page0 + i] = (row, group0 + i)
    assert args.pages == len(owner) and (a.wide > 0) == (args.pages > 0)
    for piece in pieces[a.narrow:]:
        token0, _, base, _, _, _, key0, key1 = piece[:8]
        request = owner[base + key0 // 16][0]
        # (of a prefix: the first of its requests that has tokens)
        assert starts[request] == token0
        for group in (key0 // 16, (key1 - 1) // 16):
            assert owner[base + group] == (request, group)
    for piece in pieces[:a.narrow]:
        assert 0 <= piece[2] < len(reqs)
    assert args.partials_size % 256 == 0
    if args.pages:
        table = (4 * args.pages + 255) // 256 * 256
        assert a.workspace_size == args.partials_size + table + args.pages * 2 * 16 * hk * d * 2
    else:
        assert a.workspace_size <= args.partials_size


def test_plan_entry_refuses():
    for over in ({"status": -2, "cache": quant_cache(d=80)}, {"status": -5, "cache": quant_cache(page=24)}):
        plan([0, 4], [9], 8, **over)
    for starts, seqs, heads, window in (([0, 4], [3], 8, 0), ([4, 0], [9], 8, 0), ([0, 4], [9], 7, 0),
                                        ([0, 4], [9], 8, -1), ([0, 4], [(1 << 30) + 1], 8, 0)):
        plan(starts, seqs, heads, quant_cache(), window, status=-1)
    plan([0, 4], [9], 8, quant_cache(), 0, [(0, 1, 6)], status=-1)


def test_attention_entry_refuses():
    cache = quant_cache()
    args, _, _ = plan([0, 4, 200], [9000, 300], 8, cache)
    need = args.chunk.workspace_size
    fake = 1 << 20

    def status(step=args, items=fake, table=fake, stride=1000, q=None, o=None, scale=0.1, ws=fake, size=need, cache=cache):
        q = rotary.HeadsArgs(fake, 8 * 128, 128, 8, 0) if q is None else q
        o = rotary.HeadsArgs(fake, 8 * 128, 128, 8, 0) if o is None else o
        return _lib.load().oscar_quant_attention(None if step is None else ctypes.byref(step), items, table, stride,
                                                 cache.address, ctypes.byref(q), ctypes.byref(o), scale, ws, size, None)

    heads = rotary.HeadsArgs
    assert status(step=None) == -1 and status(items=None) == -1 and status(table=None) == -1
    assert status(stride=args.chunk.table_cols - 1) == -1
    for field, value in (("num_kv_heads", 4), ("head_size", 64), ("block_size", 32), ("parts", -1), ("joins", -1),
                         ("wide", 0)):
        other = chunk.QuantStepArgs.from_buffer_copy(args)
        setattr(other.chunk, field, value)
        assert status(step=other) == -1
    for field, value in (("sources", 0), ("pages", 0), ("pages", -1), ("partials_size", -256)):
        other = chunk.QuantStepArgs.from_buffer_copy(args)
        setattr(other, field, value)
        assert status(step=other) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert status(scale=scale) == -1
    assert status(q=heads(fake, 1024, 128, 4, 0)) == -1 and status(o=heads(None, 1024, 128, 8, 0)) == -1
    assert status(ws=None) == -3 and status(size=need - 1) == -3
    assert status(q=heads(fake + 8, 1024, 128, 8, 0)) == -5 and status(o=heads(fake, 1028, 128, 8, 0)) == -5
    assert status(ws=fake + 8) == -5 and status(items=fake + 4) == -5
    assert status(o=heads(fake + 256, 1024, 128, 8, 0)) == -6
    empty, _, _ = plan([0, 0], [9], 8, cache)
    assert status(step=empty, size=0, ws=None) == 0


@pytest.mark.parametrize("over, match", [
    ({"seqs": [3]}, "lengths"), ({"num_heads": 7}, "share"), ({"window": -1}, "window"),
    ({"cache": quant_cache(d=80)}, "head sizes"), ({"cache": quant_cache(page=24)}, "multiple of 16"),
    ({"block_tables": torch.zeros(1, 0, dtype=torch.int32)}, "block table"), ({"prefixes": [(0, 2, 1)]}, "request"),
    ({}, "device tensors")])
def test_step_refuses(over, match):
    args = dict(qsl=[0, 4], seqs=[9], block_tables=torch.zeros(1, 1, dtype=torch.int32), num_heads=8,
                cache=quant_cache(), window=0)
    args.update(over)
    with pytest.raises(ValueError, match=match):
        chunk.ChunkStep(**args)


def test_step_struct_matches_the_header(tmp_path):
    header = Path(__file__).resolve().parents[1] / "include" / "oscar_amd.h"
    text = re.sub(r"/\*.*?\*/", "", header.read_text(), flags=re.S)
    body = re.search(r"typedef struct oscar_quant_step \{(.*?)\} oscar_quant_step;", text, flags=re.S).group(1)
    fields = [f for f, _ in chunk.QuantStepArgs._fields_]
    assert [re.findall(r"\w+", d)[-1] for d in body.split(";") if d.strip()] == fields
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oscar_amd.h"',
             'int main(void) { printf("%zu\\n", sizeof(oscar_quant_step));']
    lines += [f'  printf("%zu\\n", offsetof(oscar_quant_step, {f}));' for f in fields]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(header.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(chunk.QuantStepArgs)] + [getattr(chunk.QuantStepArgs, f).offset
                                                                            for f in fields]


@pytest.mark.parametrize("d, hk, group", [(64, 4, 4), (64, 3, 2), (256, 1, 6), (128, 2, 16)])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("reqs", [[(1, 32768)] * 8, [(4, 5000), (0, 7), (12, 4096), (4, 333), (5, 31)],
                                  [(1, 37 * i) for i in range(300)], [(9, 700)] * 11])
def test_narrow_pieces_cover_every_row_and_key_once(reqs, window, d, hk, group):
    """In whatever order they stand; pieces of the same lines 8 apart."""
    starts, seqs = [0], []
    for n, h in reqs:
        starts.append(starts[-1] + n)
        seqs.append(n + h)
    args, pieces, _ = plan(starts, seqs, hk * group, quant_cache(d=d, hk=hk), window)
    assert args.chunk.wide == 0
    parts = {}
    for token0, pos0, row, head, row0, rows, key0, key1, *_ in pieces:
        n, h = reqs[row]
        assert token0 == starts[row] and pos0 == h and row0 % 32 == 0 and rows == min(32, n * group - row0)
        parts.setdefault((row, head, row0), []).append((key0, key1))
    assert len(parts) == sum(hk * -(-n * group // 32) for n, _ in reqs)
    for (row, _, row0), keys in parts.items():
        n, h = reqs[row]
        first, last = h + row0 // group, h + (min(row0 + 32, n * group) - 1) // group
        keys.sort()
        lo = max(0, first - window + 1) if window else 0
        assert keys[0][0] == lo // 32 * 32 and keys[-1][1] == last + 1
        assert all(a[1] == b[0] for a, b in zip(keys, keys[1:]))
    if d == 64 and hk == 4 and len({n for n, _ in reqs}) == 1 and not window:
        at = {p[:8]: i for i, p in enumerate(pieces)}
        pairs = [at[p[:3] + (p[3] + 1,) + p[4:8]] - i for i, p in enumerate(pieces) if p[3] % 2 == 0 and p[4] == 0]
        assert all(x > 0 for x in pairs) and sum(x == 8 for x in pairs) >= len(pairs) - 8


@pytest.mark.parametrize("d, hk, group", [(64, 4, 4), (256, 2, 6), (128, 8, 4)])
def test_a_much_longer_request_is_cut_where_the_others_fill_the_gpu(d, hk, group):
    keys = [1000] * 300 + [60000]
    args, pieces, _ = plan(list(range(302)), keys, hk * group, quant_cache(d=d, hk=hk))
    mean = -(-sum(-(-n // 32) for n in keys) * hk // (3 * 256))           # tiles of 32 keys
    assert max(p[7] - p[6] for p in pieces) <= 32 * mean and args.chunk.narrow <= 301 * hk + 3 * 256 and args.chunk.wide == 0
    args, pieces, _ = plan(list(range(302)), [100 + 2 * i for i in range(301)], hk * group, quant_cache(d=d, hk=hk))
    assert args.chunk.narrow == 301 * hk and args.chunk.joins == 0


@pytest.mark.parametrize("d, hk, group", [(64, 1, 6), (128, 1, 6), (256, 1, 6), (256, 2, 4)])
@pytest.mark.parametrize("prompt", [0, 1200])
@pytest.mark.parametrize("others", [100, 160, 165, 168, 169, 170, 171, 200, 249, 254, 255, 256, 400, 490, 500, 510, 511, 512,
                                    600])
def test_a_much_longer_request_is_cut_however_many_others_there_are(d, hk, group, prompt, others):
    """Also where they nearly fill the GPU: pieces are at most twice the mean length of those
    that reside at once, or 32 key tiles above it."""
    keys = [1000] * (others // hk) + [60000] + ([prompt] if prompt else [])
    starts = list(range(len(keys) + 1))
    starts[-1] += max(prompt - 1, 0)
    args, pieces, _ = plan(starts, keys, hk * group, quant_cache(d=d, hk=hk))
    assert (args.chunk.wide > 0) == (prompt > 0)
    tiles = hk * sum(-(-n // 32) for n in keys[:others // hk + 1])
    mean = max(4, -(-tiles // (170 if prompt else 512)))                 # (the fewest that may reside)
    assert max(p[7] - p[6] for p in pieces[:args.chunk.narrow]) <= 32 * max(2 * mean, mean + 32)
