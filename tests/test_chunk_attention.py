"""The chunk attention's plan, and what is refused, without a GPU."""
import ctypes
import struct
import time

import pytest
import torch

from oscar_amd.kernels import _lib, append, chunk, decode, rotary

PIECE, JOIN = struct.Struct("12i"), struct.Struct("8i")
NARROW, WIDE, TILE = 32, 128, 32


def plain_cache(pages=4, page=16, hk=2, d=128, dtype=torch.bfloat16):
    return append.PagedCache(*(torch.zeros(pages, page, hk, d, dtype=dtype) for _ in range(2)))


def ints(values):
    return (ctypes.c_int32 * max(len(values), 1))(*values)


def plan(starts, seqs, heads, window, cache):
    args, q, s = chunk.ChunkStepArgs(), ints(starts), ints(seqs)
    call = [ctypes.addressof(q), ctypes.addressof(s), len(seqs), heads, window, cache.address]
    _lib.call("oscar_chunk_plan", *call, None, 0, ctypes.byref(args))
    size = args.items_size
    items = ctypes.create_string_buffer(max(size, 1))
    _lib.call("oscar_chunk_plan", *call, ctypes.addressof(items), size, ctypes.byref(args))
    if size > 0:
        assert _lib.load().oscar_chunk_plan(*call, ctypes.addressof(items), size - 1, ctypes.byref(args)) == -3
    at = PIECE.size * (args.narrow + args.wide)
    assert size == at + JOIN.size * args.joins
    pieces = [PIECE.unpack_from(items, PIECE.size * i) for i in range(args.narrow + args.wide)]
    return args, pieces, [JOIN.unpack_from(items, at + JOIN.size * i) for i in range(args.joins)]


@pytest.mark.parametrize("d, hk, group", [(64, 4, 4), (128, 1, 6), (256, 1, 6), (256, 2, 1), (128, 2, 40)])
@pytest.mark.parametrize("window", [0, 1, 100, 1 << 31 - 1])
@pytest.mark.parametrize("reqs", [
    [(1, 0)], [(1, 32768)] * 8, [(4, 24579)], [(9256, 15360)], [(4, 5000), (0, 7), (1024, 4096), (4, 333)],
    [(2049, 0), (33, 12), (1, 1), (16, 16)], [(1, 37 * i) for i in range(300)], [(5, 0), (300, 31)]])
def test_pieces_cover_every_row_and_key_once(reqs, window, group, d, hk):
    cache = plain_cache(d=d, hk=hk)
    starts, seqs = [3], []
    for n, h in reqs:
        starts.append(starts[-1] + n)
        seqs.append(n + h)
    window = min(window, (1 << 31) - 1)
    args, pieces, joins = plan(starts, seqs, hk * group, window, cache)
    assert args.num_tokens == starts[-1] and args.num_requests == len(reqs) and args.num_heads == hk * group
    assert args.table_cols == max(-(-s // 16) for s, (n, _) in zip(seqs, reqs) if n)
    left = {}
    slots = {}
    for i, (token0, pos0, row, head, row0, rows, key0, key1, slot, *_) in enumerate(pieces):
        n, h = reqs[row]
        assert token0 == starts[row] and pos0 == h and 0 <= head < hk
        assert 0 < rows <= (NARROW if i < args.narrow else WIDE) and row0 + rows <= n * group and key0 % TILE == 0
        assert 0 <= key0 < key1 <= n + h
        left.setdefault((row, head, row0, rows), []).append((key0, key1, slot))
        if slot >= 0:
            for g in range(-(-rows // NARROW)):
                assert slots.setdefault(slot + g, (token0, head, row0 + NARROW * g)) == (token0, head,
                                                                                          row0 + NARROW * g)
    if slots:
        assert sorted(slots) == list(range(len(slots)))
    assert args.workspace_size == len(slots) * NARROW * (d + 2) * 4
    covered = {}
    for (row, head, row0, rows), parts in left.items():
        parts.sort()
        n, h = reqs[row]
        first, last = h + row0 // group, h + (row0 + rows - 1) // group
        lo = max(0, first - window + 1) if window else 0
        assert parts[0][0] == lo // TILE * TILE and parts[-1][1] == last + 1
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        assert (len(parts) > 1) == (parts[0][2] >= 0)
        covered[(row, head)] = covered.get((row, head), 0) + rows
        if len(parts) > 1:
            for g in range(-(-rows // NARROW)):
                want = sorted(p[2] + g for p in parts)
                found = [j for j in joins if j[:4] == (starts[row], head, row0 + NARROW * g,
                                                        min(NARROW, rows - NARROW * g))]
                # (requests of no new tokens share a start with the next one)
                assert len(found) == 1
                _, _, _, _, slot0, step, count, _ = found[0]
                assert [slot0 + step * k for k in range(count)] == want
    assert covered == {(i, head): n * group for i, (n, _) in enumerate(reqs) for head in range(hk) if n}
    keys = [p[7] - p[6] for p in pieces[args.narrow:]]          # the longest first, the first 256 the other way round
    first = min(256, len(keys))
    keys[:first] = keys[:first][::-1]
    assert keys == sorted(keys, reverse=True)
    assert [j[6] <= 8 for j in joins] == [True] * args.few_joins + [False] * (args.joins - args.few_joins)


def test_an_empty_step():
    args, pieces, joins = plan([0], [], 8, 0, plain_cache())
    assert not pieces and not joins and args.items_size == 0 and args.num_tokens == 0
    args, pieces, joins = plan([0, 0, 0], [5, 0], 8, 0, plain_cache())
    assert not pieces and args.workspace_size == 0


@pytest.mark.parametrize("requests", [1, 3000])
def test_a_step_plans_its_items(requests):
    """Items that fit the first buffer, and those (144 KB) that need another."""
    cache, starts, seqs = plain_cache(hk=1), list(range(requests + 1)), [9] * requests
    args, pieces, _ = plan(starts, seqs, 4, 0, cache)
    own = chunk.ChunkStepArgs()
    items = chunk._plan(decode.request_layout(starts, seqs), requests, 4, 0, cache, own)
    assert own.items_size == args.items_size == PIECE.size * requests and (own.items_size > 1 << 17) == (requests > 1)
    assert [PIECE.unpack_from(items.numpy().tobytes(), PIECE.size * i) for i in range(requests)] == pieces


def _plan_status(starts=(0, 4), seqs=(9,), heads=8, window=0, cache=None, requests=None):
    q, s = ints(starts), ints(seqs)
    args = chunk.ChunkStepArgs()
    cache = plain_cache() if cache is None else cache
    return _lib.load().oscar_chunk_plan(ctypes.addressof(q), ctypes.addressof(s),
                                        len(seqs) if requests is None else requests, heads, window,
                                        cache.address if hasattr(cache, "address") else ctypes.byref(cache), None, 0,
                                        ctypes.byref(args))


@pytest.mark.parametrize("over, status", [
    ({}, 0), ({"seqs": (3,)}, -1), ({"starts": (4, 0)}, -1), ({"starts": (-1, 4)}, -1), ({"heads": 7}, -1),
    ({"heads": 0}, -1), ({"window": -1}, -1), ({"requests": -1}, -1), ({"seqs": ((1 << 30) + 1,)}, -1),
    ({"seqs": (1 << 30,)}, 0), ({"starts": (0, 1 << 30), "seqs": (1 << 30,)}, -1)])
def test_plan_entry_refuses(over, status):
    assert _plan_status(**over) == status


def test_plan_entry_refuses_caches():
    assert _plan_status(cache=plain_cache(d=80)) == -2
    assert _plan_status(cache=plain_cache(page=24)) == -5
    bad = append.PlainCacheArgs.from_buffer_copy(plain_cache().args)
    bad.k = None
    assert _plan_status(cache=bad) == -1


def test_attention_entry_refuses():
    cache = plain_cache()
    args, _, _ = plan([0, 4], [9000], 8, 0, cache)
    assert args.workspace_size > 0
    fake = 1 << 20

    def status(step=args, items=fake, table=fake, stride=1000, q=None, o=None, scale=0.1, ws=fake,
               size=args.workspace_size):
        q = rotary.HeadsArgs(fake, 8 * 128, 128, 8, 0) if q is None else q
        o = rotary.HeadsArgs(fake, 8 * 128, 128, 8, 0) if o is None else o
        return _lib.load().oscar_chunk_attention(None if step is None else ctypes.byref(step), items, table, stride,
                                                 cache.address, ctypes.byref(q), ctypes.byref(o), scale, ws, size,
                                                 None)

    heads = rotary.HeadsArgs
    assert status(step=None) == -1 and status(items=None) == -1 and status(table=None) == -1
    assert status(stride=args.table_cols - 1) == -1
    for field, value in (("num_kv_heads", 4), ("head_size", 64), ("block_size", 32)):        # another cache's step
        other = chunk.ChunkStepArgs.from_buffer_copy(args)
        setattr(other, field, value)
        assert status(step=other) == -1
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert status(scale=scale) == -1
    assert status(q=heads(fake, 1024, 128, 4, 0)) == -1 and status(o=heads(fake, 1024, 128, 4, 0)) == -1
    assert status(q=heads(None, 1024, 128, 8, 0)) == -1 and status(o=heads(None, 1024, 128, 8, 0)) == -1
    assert status(ws=None) == -3 and status(size=args.workspace_size - 1) == -3
    assert status(q=heads(fake + 8, 1024, 128, 8, 0)) == -5 and status(o=heads(fake, 1028, 128, 8, 0)) == -5
    assert status(q=heads(fake, -1024, 128, 8, 0)) == -5 and status(o=heads(fake, 1024, -128, 8, 0)) == -5
    assert status(ws=fake + 8) == -5 and status(items=fake + 4) == -5
    empty, _, _ = plan([0, 0], [9], 8, 0, cache)
    assert status(step=empty, size=0, ws=None) == 0


@pytest.mark.parametrize("over, match", [
    ({"seqs": [3]}, "lengths"), ({"seqs": [9, 9]}, "lengths"), ({"qsl": [-4, 0]}, "token 0"),
    ({"num_heads": 7}, "share"), ({"num_heads": 0}, "share"), ({"window": -1}, "window"),
    ({"cache": plain_cache(d=80)}, "head sizes"), ({"cache": plain_cache(page=24)}, "multiple of 16"),
    ({"block_tables": torch.zeros(1, dtype=torch.int32)}, "block table"),
    ({"block_tables": torch.zeros(1, 0, dtype=torch.int32)}, "block table"),
    ({"block_tables": torch.zeros(0, 4, dtype=torch.int32)}, "block table"), ({}, "device tensors")])
def test_step_refuses(over, match):
    args = dict(qsl=[0, 4], seqs=[9], block_tables=torch.zeros(1, 1, dtype=torch.int32), num_heads=8,
                cache=plain_cache(), window=0)
    args.update(over)
    with pytest.raises(ValueError, match=match):
        chunk.ChunkStep(**args)


def test_step_struct_matches_the_header(tmp_path):
    import re
    import subprocess
    from pathlib import Path

    header = Path(__file__).resolve().parents[1] / "include" / "oscar_amd.h"
    text = re.sub(r"/\*.*?\*/", "", header.read_text(), flags=re.S)
    body = re.search(r"typedef struct oscar_chunk_step \{(.*?)\} oscar_chunk_step;", text, flags=re.S).group(1)
    fields = [f for f, _ in chunk.ChunkStepArgs._fields_]
    assert [re.findall(r"\w+", d)[-1] for d in body.split(";") if d.strip()] == fields
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "oscar_amd.h"',
             'int main(void) { printf("%zu\\n", sizeof(oscar_chunk_step));']
    lines += [f'  printf("%zu\\n", offsetof(oscar_chunk_step, {f}));' for f in fields]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", str(header.parent), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [ctypes.sizeof(chunk.ChunkStepArgs)] + [getattr(chunk.ChunkStepArgs, f).offset
                                                                            for f in fields]


@pytest.mark.parametrize("window, planned", [
    (5, 5), (1 << 30, 1 << 30), ((1 << 30) + 1, 1 << 30), ((1 << 31) - 1, 1 << 30), (1 << 31, 1 << 30),
    ((1 << 32) + 5, 1 << 30), (1 << 64, 1 << 30)])
def test_windows_of_any_size(monkeypatch, window, planned):
    """A window past the longest request is that of all keys, past 32 bits too."""
    seen = []
    plan_step = chunk._plan

    def keep(*args):
        items = plan_step(*args)
        seen.append(args[-1])
        return items

    monkeypatch.setattr(chunk, "_plan", keep)
    with pytest.raises(ValueError, match="device tensors"):       # (planned, then refused without a GPU)
        chunk.ChunkStep([0, 4], [9], torch.zeros(1, 1, dtype=torch.int32), 8, plain_cache(), window)
    assert seen[0].window == planned


@pytest.mark.parametrize("window", [(1 << 30) + 1, (1 << 31) - 1])
def test_plan_clamps_the_window(window):
    reqs = ([0, 4, 300], [9000, 300], 8)
    none, pieces, joins = plan(*reqs, 0, plain_cache())
    args, same_pieces, same_joins = plan(*reqs, window, plain_cache())
    assert args.window == 1 << 30 and none.window == 0 and (same_pieces, same_joins) == (pieces, joins)


@pytest.mark.parametrize("qsl, seqs", [([0, 4], [(1 << 32) + 9]), ([0, 4], [1 << 31]), ([1 << 32, (1 << 32) + 4], [9]),
                                       ([0, 1 << 31], [1 << 31]), ([-(1 << 32), 4 - (1 << 32)], [9])])
def test_lengths_past_32_bits_are_refused(qsl, seqs):
    with pytest.raises(ValueError, match="32-bit"):
        decode.RequestLayout(qsl, seqs)
    with pytest.raises(ValueError, match="32-bit"):
        chunk.ChunkStep(qsl, seqs, torch.zeros(1, 1, dtype=torch.int32), 8, plain_cache())


@pytest.mark.parametrize("heads, match", [((1 << 32) + 8, "at most"), ((1 << 16) + 2, "at most"), (1 << 16, "device")])
def test_more_heads_than_the_plan_takes_are_refused(heads, match):
    with pytest.raises(ValueError, match=match):
        chunk.ChunkStep([0, 4], [9], torch.zeros(1, 1, dtype=torch.int32), heads, plain_cache())


@pytest.mark.parametrize("short, long, pieces", [(254, 1 << 30, 2), (250, 1 << 20, 6), (255, 1 << 20, 1),
                                                 (100, 1 << 25, 156)])
def test_one_long_row_among_short_ones_is_planned_at_once(short, long, pieces):
    """The fewest key tiles a piece with which there are at most 256 pieces (one wide
    cache head of 256 features), found in time that does not go by the keys: 50 us each
    (a second here, for a machine with other work)."""
    cache = plain_cache(d=256, hk=1)
    began = time.perf_counter()
    args, items, joins = plan(list(range(short + 2)), [11] * short + [long], 6, 0, cache)
    assert time.perf_counter() - began < 1.0
    parts = sorted((p[6], p[7]) for p in items if p[2] == short)
    assert len(items) == short + pieces and len(parts) == pieces and len(joins) == (pieces > 1)
    tiles = [-(-(b - a) // TILE) for a, b in parts]
    assert parts[0][0] == 0 and parts[-1][1] == long and max(tiles) - min(tiles) <= 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.bool], ids=str)
def test_block_tables_of_other_types_are_refused(dtype):
    with pytest.raises(ValueError, match="integers"):
        chunk.ChunkStep([0, 4], [9], torch.zeros(1, 1, dtype=dtype), 8, plain_cache())


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no device memory")
def test_strides_of_single_rows_are_not_looked_at():
    """Without a GPU what passes the checks ends at the launch (-4)."""
    fake, heads = 1 << 20, rotary.HeadsArgs

    def status(tokens, hq, q, o):
        cache = plain_cache(hk=1)
        args, _, _ = plan([0, tokens], [40], hq, 0, cache)
        return _lib.load().oscar_chunk_attention(ctypes.byref(args), fake, fake, 10, cache.address,
                                                 ctypes.byref(heads(fake, *q, hq, 0)),
                                                 ctypes.byref(heads(fake, *o, hq, 0)), 0.1, fake, args.workspace_size,
                                                 None)

    good, odd = (512, 128), (513, 128)
    assert status(1, 4, good, odd) == status(1, 4, odd, good) == status(1, 4, good, (-1, 128)) == -4
    assert status(2, 4, good, odd) == status(2, 4, odd, good) == -5
    assert status(2, 1, (128, 128), (128, 129)) == status(2, 1, (128, -5), (128, 128)) == -4
    assert status(2, 2, good, (512, 129)) == -5
