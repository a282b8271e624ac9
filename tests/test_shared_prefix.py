"""The plan of a step whose requests share prefixes, and what is refused, without a GPU."""
import ctypes
import struct

import pytest
import torch

from oscar_amd.kernels import _lib, chunk
from tests.test_chunk_attention import JOIN, NARROW, PIECE, TILE, WIDE, ints, plain_cache

PART = struct.Struct("4i")


def plan(starts, seqs, heads, prefixes, cache, window=0, status=0):
    args, q, s = chunk.ChunkStepArgs(), ints(starts), ints(seqs)
    flat = ints([x for p in prefixes for x in p])
    call = [ctypes.addressof(q), ctypes.addressof(s), len(seqs), heads, window, ctypes.addressof(flat), len(prefixes),
            cache.address]
    got = _lib.load().oscar_chunk_plan_shared(*call, None, 0, ctypes.byref(args))
    assert got == status
    if status:
        return None
    size = args.items_size
    items = ctypes.create_string_buffer(max(size, 1))
    _lib.call("oscar_chunk_plan_shared", *call, ctypes.addressof(items), size, ctypes.byref(args))
    at = PIECE.size * (args.narrow + args.wide)
    end = at + JOIN.size * args.joins
    assert size == end + PART.size * args.parts
    if size:
        assert _lib.load().oscar_chunk_plan_shared(*call, ctypes.addressof(items), size - 1, ctypes.byref(args)) == -3
    return (args, [PIECE.unpack_from(items, PIECE.size * i) for i in range(args.narrow + args.wide)],
            [JOIN.unpack_from(items, at + JOIN.size * i) for i in range(args.joins)],
            [PART.unpack_from(items, end + PART.size * i) for i in range(args.parts)])


STEPS = [
    ([(1, 4200), (1, 4100), (1, 4099)], [(0, 3, 4099)]),
    ([(4, 24600 + i) for i in range(32)], [(0, 32, 24579)]),
    ([(1, 100), (2, 500), (0, 3), (3, 600), (1, 40), (7, 999), (5, 800), (1, 31)], [(1, 3, 500), (5, 2, 777)]),
    ([(300, 900), (1, 900), (64, 950)], [(0, 3, 900)]),
    ([(0, 4), (2, 70), (2, 64)], [(0, 3, 64)]),
    ([(1, 31), (1, 31)], [(0, 2, 31)]),                       # (less than a key tile: each reads its own)
    ([(1, 500), (0, 500)], [(0, 2, 500)]),                    # (one request with tokens)
    ([(1, 300)] * 300, [(0, 150, 256), (150, 150, 33)]),
]


@pytest.mark.parametrize("d, hk, group", [(64, 4, 4), (128, 1, 6), (256, 1, 6), (128, 2, 40)])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_every_row_meets_every_key_once(case, d, hk, group):
    reqs, prefixes = STEPS[case]
    starts, seqs = [2], []
    for n, h in reqs:
        starts.append(starts[-1] + n)
        seqs.append(n + h)
    args, pieces, joins, parts = plan(starts, seqs, hk * group, prefixes, plain_cache(d=d, hk=hk))
    used = []
    for first, count, keys in prefixes:
        members = [i for i in range(first, first + count) if reqs[i][0]]
        if len(members) > 1 and keys >= TILE:
            used.append((members, first, keys // TILE * TILE))
    group_of = {i: u for u in used for i in u[0]}
    assert (args.parts > 0) == bool(used)
    # what each slot holds: rows by (token, head of the kv head) of a kv head, over keys
    slots, finished = {}, {}
    for i, (token0, pos0, row, head, row0, rows, key0, key1, slot, *_) in enumerate(pieces):
        assert 0 < rows <= (NARROW if i < args.narrow else WIDE) and key0 % TILE == 0 and key0 < key1
        n, h = reqs[row]
        end = starts[row] + n
        if row in group_of and key1 <= group_of[row][2]:      # of the prefix
            members, first, keys = group_of[row]
            assert row == members[0] and token0 == starts[first] and pos0 >= keys and slot >= 0
            end = starts[members[-1]] + reqs[members[-1]][0]
        else:
            assert token0 == starts[row] and pos0 == h
            assert key0 >= (group_of[row][2] if row in group_of else 0) and key1 <= n + h
        assert (row0 + rows - 1) // group + token0 < end
        for r in range(rows):
            at = (token0 + (row0 + r) // group, (row0 + r) % group, head)
            if slot >= 0:
                assert slots.setdefault((slot + r // NARROW, r % NARROW), (at, key0, key1)) == (at, key0, key1)
            else:
                assert finished.setdefault(at, (key0, key1)) == (key0, key1)
    held = {s for s, _ in slots}
    assert held == set(range(len(held))) and args.workspace_size == len(held) * NARROW * (d + 2) * 4
    met = {at: [keys] for at, keys in finished.items()}
    few = []
    for token0, head, row0, rows, slot0, step, count, shared in joins:
        total = count
        for r in range(rows):
            at = (token0 + (row0 + r) // group, (row0 + r) % group, head)
            assert at not in met
            met[at] = []
            places = [(slot0 + step * k, r) for k in range(count)]
            if shared:
                pslot, pstep, pcount, prow = parts[shared - 1]
                places += [(pslot + pstep * k + (prow + r) // NARROW, (prow + r) % NARROW) for k in range(pcount)]
                total = count + pcount
            for place in places:
                owner, key0, key1 = slots.pop(place)
                assert owner == at
                met[at].append((key0, key1))
        few.append(total <= 8)
    assert not slots                                           # (every partial is joined)
    assert few == [True] * args.few_joins + [False] * (args.joins - args.few_joins)
    want = {}
    for i, (n, h) in enumerate(reqs):
        for t in range(n):
            for x in range(group):
                for head in range(hk):
                    want[(starts[i] + t, x, head)] = h + t
    assert met.keys() == want.keys()
    for at, keys in met.items():
        keys.sort()
        assert keys[0][0] == 0 and all(a[1] == b[0] for a, b in zip(keys, keys[1:]))
        assert want[at] < keys[-1][1] <= want[at] + WIDE


def test_without_prefixes_the_plan_is_the_plain_one():
    cache = plain_cache(d=256, hk=1)
    args, pieces, joins, parts = plan([0, 4, 1000], [9000, 2000], 6, [], cache)
    plain = chunk.ChunkStepArgs()
    q, s = ints([0, 4, 1000]), ints([9000, 2000])
    items = ctypes.create_string_buffer(args.items_size)
    _lib.call("oscar_chunk_plan", ctypes.addressof(q), ctypes.addressof(s), 2, 6, 0, cache.address,
              ctypes.addressof(items), args.items_size, ctypes.byref(plain))
    assert bytes(plain) == bytes(args) and not parts
    assert [PIECE.unpack_from(items, PIECE.size * i) for i in range(len(pieces))] == pieces


@pytest.mark.parametrize("prefixes, window", [
    ([(0, 2, 40)], 5), ([(0, 2, 101)], 0), ([(-1, 2, 40)], 0), ([(0, 4, 40)], 0), ([(0, -1, 40)], 0),
    ([(0, 2, -1)], 0), ([(0, 2, 40), (1, 1, 40)], 0), ([(1, 2, 40), (0, 1, 40)], 0), ([(3, 1, 0)], 0)])
def test_plan_entry_refuses(prefixes, window):
    plan([0, 1, 2, 3], [101, 102, 400], 4, prefixes, plain_cache(), window, status=-1)


def test_plan_entry_refuses_no_array():
    args, q, s = chunk.ChunkStepArgs(), ints([0, 1]), ints([9])
    for count in (1, -1):
        assert _lib.load().oscar_chunk_plan_shared(ctypes.addressof(q), ctypes.addressof(s), 1, 4, 0, None, count,
                                                   plain_cache().address, None, 0, ctypes.byref(args)) == -1


@pytest.mark.parametrize("over, match", [
    ({"prefixes": [(0, 2, 40)], "window": 8}, "window"), ({"prefixes": [(0, 4, 40)]}, "no request in two"),
    ({"prefixes": [(0, 2, 40), (1, 2, 40)]}, "no request in two"), ({"prefixes": [(0, 2, 101)]}, "fewer keys"),
    ({"prefixes": [(0, 2, -1)]}, "prefixes are"), ({"prefixes": [(-1, 2, 40)]}, "no request in two"),
    ({"prefixes": [(2, 1, 40), (0, 2, 100)]}, "device tensors")])
def test_step_refuses(over, match):
    args = dict(qsl=[0, 1, 2, 3], seqs=[101, 102, 400], block_tables=torch.zeros(3, 25, dtype=torch.int32), num_heads=4,
                cache=plain_cache())
    args.update(over)
    with pytest.raises(ValueError, match=match):
        chunk.ChunkStep(**args)


def test_a_step_of_a_bad_count_is_refused():
    """The attention's entry looks at the parts as it does at the joins."""
    from oscar_amd.kernels import rotary

    cache = plain_cache()
    args, *_ = plan([0, 1, 2], [5000, 5000], 8, [(0, 2, 4096)], cache)
    bad = chunk.ChunkStepArgs.from_buffer_copy(args)
    bad.parts = -1
    h = rotary.HeadsArgs(1 << 20, 8 * 128, 128, 8, 0)
    assert _lib.load().oscar_chunk_attention(ctypes.byref(bad), 1 << 20, 1 << 20, 1000, cache.address, ctypes.byref(h),
                                             ctypes.byref(h), 0.1, 1 << 20, args.workspace_size, None) == -1


FULL = [
    ([(4096, 1024)] * 8, [(0, 8, 1024)]),
    ([(2048, 64)] * 16, [(0, 16, 64)]),
    ([(0, 900), (4, 1900), (3, 1930), (3000, 1900), (2, 1905), (0, 9), (4000, 2000), (1, 1900), (5, 2011), (1, 1950),
      (9, 400), (1, 400)], [(0, 10, 1900), (10, 2, 400)]),
    ([(4000, 500), (1, 500), (2, 500), (4000, 0), (2, 100), (2, 96)], [(0, 3, 500), (4, 2, 96)]),
    ([(9256, 32), (9256, 32), (1, 70)], [(0, 3, 32)]),
    ([(10, 64)] * 128 + [(2000, 500)] * 6, [(0, 128, 64)]),
    ([(10, 4096)] * 128 + [(2000, 500)] * 6, [(0, 128, 4096)]),
]


@pytest.mark.parametrize("d, hk, group", [(64, 4, 4), (128, 8, 4), (256, 1, 6)])
@pytest.mark.parametrize("case", range(len(FULL)))
def test_prompts_that_fill_the_gpu_share_no_sums(case, d, hk, group):
    """Those that gain nothing by sharing compute the prefix themselves, on the first one's pages,
    and leave no partials for it; the requests between them share theirs.  Every row meets every
    key once."""
    reqs, prefixes = FULL[case]
    starts, seqs = [0], []
    for n, h in reqs:
        starts.append(starts[-1] + n)
        seqs.append(n + h)
    narrow_rows = 32
    assert sum(n * group for n, _ in reqs if n * group > narrow_rows) * hk >= 256 * WIDE
    alone = []
    for i, (n, _) in enumerate(reqs):
        keys = sum(k // TILE * TILE for first, count, k in prefixes if first <= i < first + count)
        alone.append(n * group > narrow_rows and keys * (-n * group % WIDE) < 800 * n * group)
    args, pieces, joins, parts = plan(starts, seqs, hk * group, prefixes, plain_cache(d=d, hk=hk))
    head, keys_of, run = {}, {}, {}
    for first, count, keys in prefixes:
        members = [i for i in range(first, first + count) if reqs[i][0]]
        runs = [[]]
        for i in members:
            head[i], keys_of[i] = members[0], keys // TILE * TILE
            if alone[i]:
                runs.append([])
            else:
                runs[-1].append(i)
        for r in runs:
            run.update({i: r for i in r if len(r) > 1})
    met = {}                                # (request, kv head, row0): ranges of keys, by table row
    slots = set()
    for i, (token0, pos0, row, kv, row0, rows, key0, key1, slot, head_keys, head_row, pad) in enumerate(pieces):
        request = max(r for r in range(len(reqs)) if starts[r] <= token0 and reqs[r][0])
        assert rows <= (NARROW if i < args.narrow else WIDE) and pad == 0
        if slot >= 0:
            slots.add(slot)
        if request in run and key1 <= keys_of[request] and pos0 == keys_of[request] and token0 == starts[run[request][0]]:
            assert row == head[request] and head_keys == 0 and slot >= 0
            n = sum(reqs[r][0] for r in run[request])
            at = ("run", run[request][0], kv, row0)
            assert rows == min(NARROW if i < args.narrow else WIDE, n * group - row0)
        else:
            assert token0 == starts[request] and row == request and pos0 == reqs[request][1]
            at = (request, kv, row0)
            if request in head and request not in run and head[request] != request:
                assert (head_keys, head_row) == (keys_of[request], head[request])
            else:
                assert head_keys == 0
            if alone[request] and args.joins == 0:
                assert slot < 0
        met.setdefault(at, []).append((key0, key1))
    for at, keys in met.items():
        keys.sort()
        assert all(a[1] == b[0] for a, b in zip(keys, keys[1:]))
        if at[0] == "run":
            assert keys[0][0] == 0 and keys[-1][1] == keys_of[at[1]]
        else:
            n, h = reqs[at[0]]
            assert keys[0][0] == (keys_of[at[0]] if at[0] in run else 0) and keys[-1][1] <= n + h
    assert {a[:2] for a in met if a[0] != "run"} == {(i, kv) for i, (n, _) in enumerate(reqs) if n for kv in range(hk)}
    assert sum(a[0] == "run" for a in met) > 0 if run else args.parts == 0
    # partials: of the requests that share, and a bounded number of others
    own = sum(-(-reqs[i][0] * group // NARROW) for i in run) * hk
    assert args.parts == own and (run or args.joins == 0 and args.workspace_size == 0)
