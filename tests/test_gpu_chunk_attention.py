"""Chunk attention over a plain paged cache, against the formula in 64 bits.

Tolerance of an output o = sum p_t v_t (p the normalised weights, inputs taken
as they are), eps the type's, B = sum p_t |v_t|:
  the weights are rounded to the type before the product and summed as rounded:
    each is off by eps / 2 relative, the mean by eps / 2 (B + |o|) at most;
  the scores are fp32 sums of D products, off by at most (D + 2) 2^-24 sum |q k|
    scale; a weight by that, relatively, and the mean by twice that times B;
    the exponential and the lazy maximum (weights up to 2^8 of the largest
    possible 1) add 2^-21 of a weight;
  fp16 weights below 2^-14 of the maximum are subnormal: off by 2^-25 each, of a
    sum that is at least 1: t 2^-25 max |v|;
  the output's own rounding: eps / 2 |o| and half a subnormal step."""
import math

import pytest
import torch

from oscar_amd.kernels import _lib, append, chunk, rotary

pytestmark = pytest.mark.gpu


def expected(q, keys, values, first, window, scale, hidden=None):
    """(o, bound) of one request: q [n, Hq, D] at positions first .., keys / values
    [t, Hk, D]; hidden [t]: keys that no row sees."""
    n, hq, d = q.shape
    hk = keys.shape[1]
    dtype = q.dtype
    eps = torch.finfo(dtype).eps
    q, keys, values = q.double(), keys.double(), values.double()
    pos = first + torch.arange(n, device=q.device)
    at = torch.arange(keys.shape[0], device=q.device)
    seen = at[None] <= pos[:, None]
    if window:
        seen &= at[None] > pos[:, None] - window
    if hidden is not None:
        seen &= ~hidden[None]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(hq):
        k, v = keys[:, h // (hq // hk)], values[:, h // (hq // hk)]
        s = (q[:, h] @ k.t()) * scale
        reach = (q[:, h].abs() @ k.abs().t()) * scale
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, (s - torch.where(top.isinf(), 0.0, top)).exp(), 0.0)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        v = torch.where(seen.any(0)[:, None], v, 0.0)
        o = p @ v
        mean = p @ v.abs()
        off = (torch.where(seen, reach, 0.0).amax(-1, keepdim=True)) * (d + 2) * 2.0 ** -24
        b = eps / 2 * (mean + o.abs()) + (2 * off + 2.0 ** -20) * mean + eps / 2 * o.abs() * (1 + eps)
        b += torch.finfo(dtype).smallest_normal * eps / 2
        if dtype == torch.float16:
            b += seen.sum(-1, keepdim=True) * 2.0 ** -25 * v.abs().amax()
        out[:, h], bound[:, h] = o, b
    return out, bound


def make(g, reqs, hq, hk, d, page, dtype, layout="apart", spread=1.0):
    """Caches with shuffled pages, block table, queries of a step of (new, history) requests."""
    need = [max(1, -(-(n + h) // page)) for n, h in reqs]
    pages = sum(need) + 2
    shape = (page, hk, d)
    if layout == "joint":
        both = torch.randn(pages, 2, *shape, generator=g, device="cuda:0").to(dtype)
        caches = [both[:, 0], both[:, 1]]
    elif layout == "heads_first":
        caches = [torch.randn(pages, hk, page, d, generator=g, device="cuda:0").to(dtype).transpose(1, 2)
                  for _ in range(2)]
    else:
        caches = [torch.randn(pages, *shape, generator=g, device="cuda:0").to(dtype) for _ in range(2)]
    order = torch.randperm(pages, generator=g, device="cuda:0").to(torch.int32)
    table = torch.full((len(reqs), max(need)), -1, dtype=torch.int32, device="cuda:0")
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    q = (torch.randn(sum(n for n, _ in reqs), hq, d, generator=g, device="cuda:0") * spread).to(dtype)
    starts = [0]
    for n, _ in reqs:
        starts.append(starts[-1] + n)
    return q, caches, table, starts, [n + h for n, h in reqs]


def gather(caches, row, seq, page):
    at = torch.arange(seq, device=row.device)
    slot = row[at // page].long() * page + at % page
    return [c.reshape(-1, *c.shape[2:])[slot] for c in caches]


def check(got, q, caches, table, starts, seqs, window, scale, page):
    for i, seq in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        keys, values = gather(caches, table[i], seq, page)
        o, bound = expected(q[a:b], keys, values, seq - (b - a), window, scale)
        off = (got[a:b].double() - o).abs() - bound
        assert off.max().item() <= 0, f"request {i}: off by {off.max().item():.3e} more than the bound"


DECODE = [[(1, 0)], [(1, 1)], [(1, 31)], [(1, 32)], [(1, 4099)], [(4, 700), (1, 15), (3, 0), (2, 5000)],
          [(16, 33), (0, 100), (5, 127), (1, 128), (7, 1000)], [(1, 40 * i) for i in range(70)]]
PROMPTS = [[(17, 0)], [(33, 1)], [(257, 0)], [(300, 777)], [(129, 2000), (1, 900), (64, 0)], [(1100, 333)]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(DECODE + PROMPTS)))
def test_against_the_formula(device, dtype, d, case):
    reqs = (DECODE + PROMPTS)[case]
    g = torch.Generator(device=device).manual_seed(100 * case + d)
    for hq, hk, page, window, layout in ((6, 1, 128, 0, "apart"), (4, 4, 16, 0, "joint"), (8, 2, 48, 100, "heads_first"),
                                         (16, 1, 32, 1, "apart"), (7, 1, 64, 33, "joint")):
        q, caches, table, starts, seqs = make(g, reqs, hq, hk, d, page, dtype, layout, spread=2.0)
        cache = append.PagedCache(*caches)
        step = chunk.ChunkStep(starts, seqs, table, hq, cache, window)
        got = chunk.chunk_attention(q, cache, step, d ** -0.5)
        check(got, q, caches, table, starts, seqs, window, d ** -0.5, page)


def test_scores_of_any_size(device):
    """One key dominates, or all weigh alike; maxima that rise along the keys."""
    g = torch.Generator(device=device).manual_seed(5)
    for scale, spread in ((1.0, 8.0), (1e-6, 1.0), (0.3, 30.0)):
        q, caches, table, starts, seqs = make(g, [(3, 900), (40, 300)], 8, 2, 128, 32, torch.bfloat16, spread=spread)
        ramp = torch.linspace(0, 4, 32, device=device)[None, :, None, None]
        caches[0].mul_(ramp.to(torch.bfloat16))
        cache = append.PagedCache(*caches)
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 8, cache), scale)
        check(got, q, caches, table, starts, seqs, 0, scale, 32)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_do_not_depend_on_their_neighbours(device, d):
    """Scores that grow along the keys at another pace for every row: a row's result is
    the same among the others and among copies of itself."""
    g = torch.Generator(device=device).manual_seed(14)
    n, h = 64, 700
    q, caches, table, starts, seqs = make(g, [(n, h)], 2, 1, d, 16, torch.bfloat16)
    caches[0].mul_(0.125)
    keys = torch.arange(n + h, device=device)
    caches[0][table[0][keys // 16].long(), keys % 16, 0, 0] = (keys / 16).bfloat16()
    q[..., 0] = torch.arange(2 * n, device=device).view(n, 2).flip(0) / 64       # (a score rises by 2 along the keys, or 80)
    cache = append.PagedCache(*caches)
    step = chunk.ChunkStep(starts, seqs, table, 2, cache)
    got = chunk.chunk_attention(q, cache, step, 1.0)
    check(got, q, caches, table, starts, seqs, 0, 1.0, 16)
    for row in (0, 17, 40, 63):
        alone = chunk.chunk_attention(q[row:row + 1].expand(n, 2, d), cache, step, 1.0)
        assert torch.equal(alone[row], got[row])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_lies_in_unseen_slots_does_not_matter(device, d):
    """Slots past a request's keys, other requests' pages: NaN and infinities."""
    g = torch.Generator(device=device).manual_seed(6)
    reqs = [(1, 40), (4, 90), (50, 100), (1, 0), (130, 3)]
    q, caches, table, starts, seqs = make(g, reqs, 6, 1, d, 64, torch.bfloat16)
    cache = append.PagedCache(*caches)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    want = chunk.chunk_attention(q, cache, step, 0.1)
    used = torch.zeros(caches[0].shape[0] * 64, dtype=torch.bool, device=device)
    for i, seq in enumerate(seqs):
        at = torch.arange(seq, device=device)
        used[table[i][at // 64].long() * 64 + at % 64] = True
    for c, bad in zip(caches, (math.nan, math.inf)):
        c.view(-1, 1, d)[~used] = bad
    assert torch.equal(chunk.chunk_attention(q, cache, step, 0.1), want)
    check(want, q, caches, table, starts, seqs, 0, 0.1, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_what_a_row_does_not_see_does_not_reach_it(device, dtype, d, window):
    """NaN and infinities in keys and values of single positions: rows that do not
    see them are as without them, rows that do have the formula's NaN or infinity."""
    g = torch.Generator(device=device).manual_seed(16)
    for reqs in ([(16, 100), (3, 70)], [(200, 90)], [(260, 0), (2, 33)]):
        q, caches, table, starts, seqs = make(g, reqs, 4, 2, d, 32, dtype)
        table[0, 0] = -1 if reqs[0][1] == 90 else table[0, 0]     # (a tile that is whole, but half unmapped)
        cache = append.PagedCache(*caches)
        step = chunk.ChunkStep(starts, seqs, table, 4, cache, window)
        clean = chunk.chunk_attention(q, cache, step, 0.1)
        n, h = reqs[0]
        at = {h + n // 2: (1, math.nan, 5), h + n - 2: (1, math.inf, 7), h + n - 5: (1, -math.inf, 7),
              h + 3: (0, math.inf, 1), max(h - 20, 0) + 16: (1, math.inf, 2)}
        for pos, (which, value, feature) in at.items():
            caches[which][table[0, pos // 32].long(), pos % 32, 0, feature] = value
        got = chunk.chunk_attention(q, cache, step, 0.1)
        pos = h + torch.arange(n, device=device)
        touched = torch.zeros(n, 2, d, dtype=torch.bool, device=device)      # (kv head 0: query heads 0 and 1)
        without = torch.zeros(n, 2, 1, dtype=torch.bool, device=device)      # rows whose score of the infinite key is
        for p, (which, value, feature) in at.items():                        # -inf: its weight is 0
            sees = ((pos >= p) & ((pos < p + window) if window else True))[:, None, None]
            if which == 0:
                hidden = torch.arange(n + h, device=device) == p
                touched |= sees & (q[:n, :2, 1:2] > 0)                       # +inf: no number in the whole row
                without |= sees & (q[:n, :2, 1:2] < 0)
            else:
                touched[..., feature] |= sees[..., 0]
        mine, were = got[:n, :2], clean[:n, :2]
        assert torch.equal(got[:, 2:], clean[:, 2:]) and torch.equal(got[n:], clean[n:])
        same = ~touched & ~without
        assert torch.equal(mine[same], were[same])
        assert not mine[touched].isfinite().any()
        if reqs[0][1] != 90:
            keys, values = gather(caches, table[0], n + h, 32)
            values = torch.where(values.isfinite(), values, 0.0)
            keys = torch.where(keys.isfinite(), keys, 0.0)
            o, bound = expected(q[:n], keys, values, h, window, 0.1, hidden)
            rest = (without & ~touched).expand_as(mine)
            assert ((mine.double() - o[:, :2]).abs() <= bound[:, :2])[rest].all()
        # a single infinity stays one
        row = touched[..., 2] & ~touched[..., 1]
        assert (mine[row][..., 2] == math.inf).all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_decodes_beside_prompts(device, d):
    """More short row tiles than CUs, and wide ones cut in many pieces."""
    g = torch.Generator(device=device).manual_seed(30 + d)
    reqs = [(1, 3000)] * 40 + [(40, 0), (50, 9000)]
    q, caches, table, starts, seqs = make(g, reqs, 4, 4, d, 32, torch.bfloat16)
    cache = append.PagedCache(*caches)
    for window in (0, 700):
        step = chunk.ChunkStep(starts, seqs, table, 4, cache, window)
        assert step.args.wide > 0 and (window or step.args.narrow > 256)
        got = chunk.chunk_attention(q, cache, step, 0.1)
        check(got, q, caches, table, starts, seqs, window, 0.1, 32)


@pytest.mark.parametrize("hq, hk, page", [(64, 1, 1024), (40, 1, 16), (33, 1, 240), (66, 2, 128), (1, 1, 4096)])
def test_large_groups_and_pages(device, hq, hk, page):
    """Groups of more heads than a narrow tile's rows; pages of many tiles, or of 15 groups of 16 keys."""
    g = torch.Generator(device=device).manual_seed(hq + page)
    q, caches, table, starts, seqs = make(g, [(1, 1500), (3, 40), (0, 7), (9, 5000)], hq, hk, 128, page, torch.float16)
    cache = append.PagedCache(*caches)
    for window in (0, 333):
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, hq, cache, window), 0.09)
        check(got, q, caches, table, starts, seqs, window, 0.09, page)


def test_unmapped_pages_are_left_out(device):
    g = torch.Generator(device=device).manual_seed(7)
    reqs = [(2, 200), (40, 200), (1, 10), (3, 300)]
    q, caches, table, starts, seqs = make(g, reqs, 4, 2, 128, 32, torch.float16)
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 6], bad[2, 0], bad[3, 9] = -1, caches[0].shape[0], 1 << 30, -(1 << 31), -7
    cache = append.PagedCache(*caches)
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, bad, 4, cache), 0.09)
    for i, seq in enumerate(seqs):
        hidden = torch.zeros(seq, dtype=torch.bool, device=device)
        for c in range(-(-seq // 32)):
            if bad[i, c] != table[i, c]:
                hidden[32 * c:32 * (c + 1)] = True
        keys, values = gather(caches, table[i], seq, 32)
        o, bound = expected(q[starts[i]:starts[i + 1]], keys, values, reqs[i][1], 0, 0.09, hidden)
        assert ((got[starts[i]:starts[i + 1]].double() - o).abs() <= bound).all()
    assert (got[starts[2]:starts[3]] == 0).all()          # nothing left to see


def test_rows_of_no_request_are_left_alone(device):
    g = torch.Generator(device=device).manual_seed(8)
    q, caches, table, _, seqs = make(g, [(4, 50), (3, 60)], 6, 1, 64, 16, torch.bfloat16)
    cache = append.PagedCache(*caches)
    starts = [0, 4, 7]
    padded = torch.cat((q, torch.full((5, 6, 64), math.nan, device=device).bfloat16()))
    out = torch.full((14, 6, 64), 3.0, device=device).bfloat16()[:12]
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    assert chunk.chunk_attention(padded, cache, step, 0.125, out=out) is out
    assert (out[7:] == 3.0).all()
    check(out, q, caches, table, starts, seqs, 0, 0.125, 16)
    # a step that begins past token 0 (rows before it are another call's)
    out2 = torch.full_like(out, 3.0)
    shifted = torch.cat((padded[:2], padded))
    chunk.chunk_attention(shifted[:9], cache, chunk.ChunkStep([2, 6, 9], seqs, table, 6, cache), 0.125, out=out2[:9])
    assert (out2[:2] == 3.0).all() and torch.equal(out2[2:9], out[:7])


def test_strided_queries_and_outputs(device):
    g = torch.Generator(device=device).manual_seed(9)
    q, caches, table, starts, seqs = make(g, [(40, 50), (1, 600)], 6, 2, 64, 16, torch.float16)
    cache = append.PagedCache(*caches)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    want = chunk.chunk_attention(q, cache, step, 0.125)
    fused = torch.zeros(41, 10, 64, device=device, dtype=torch.float16)
    fused[:, 2:8] = q
    out = torch.zeros(41, 9, 64, device=device, dtype=torch.float16)
    chunk.chunk_attention(fused[:, 2:8], cache, step, 0.125, out=out[:, 1:7])
    assert torch.equal(out[:, 1:7], want) and (out[:, 0] == 0).all() and (out[:, 7:] == 0).all()
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(chunk.chunk_attention(heads_first, cache, step, 0.125), want)
    odd = torch.zeros(41, 6, 65, device=device, dtype=torch.float16)[..., 1:]
    odd.copy_(q)
    assert torch.equal(chunk.chunk_attention(odd, cache, step, 0.125), want)
    with pytest.raises(ValueError, match="16 bytes"):
        chunk.chunk_attention(q, cache, step, 0.125, out=odd)
    with pytest.raises(ValueError, match="overlap"):
        chunk.chunk_attention(q, cache, step, 0.125, out=out[:, :1].expand(41, 6, 64))
    early = torch.zeros(41 * 6 * 64 + 1, device=device, dtype=torch.float16)[1:].view(41, 6, 64)       # 2 bytes off
    early.copy_(q)
    assert torch.equal(chunk.chunk_attention(early, cache, step, 0.125), want)
    mine = q.clone()
    assert chunk.chunk_attention(mine, cache, step, 0.125, out=mine) is mine and torch.equal(mine, want)


@pytest.mark.parametrize("kind", ["int64", "columns first", "one row for all"])
def test_block_tables_of_other_layouts(device, kind):
    g = torch.Generator(device=device).manual_seed(21)
    q, caches, table, starts, seqs = make(g, [(40, 50), (40, 50)], 4, 2, 64, 16, torch.bfloat16)
    cache = append.PagedCache(*caches)
    if kind == "one row for all":
        table[1] = table[0]
    want = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 4, cache), 0.125)
    other = {"int64": table.long(), "columns first": table.t().contiguous().t(),
             "one row for all": table[:1].expand(2, -1)}[kind]
    assert torch.equal(chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, other, 4, cache), 0.125), want)


@pytest.mark.parametrize("new", [3, 300])
def test_pages_past_32_bits(device, new):
    """A cache of 6 GB (K and V pages in turn) whose last pages are used, at both tile sizes."""
    base = torch.empty(3 << 30, dtype=torch.bfloat16, device=device)
    joint = base.view(-1, 2, 16, 2, 128)
    cache = append.PagedCache(joint[:, 0], joint[:, 1])
    g = torch.Generator(device=device).manual_seed(new)
    q, caches, table, starts, seqs = make(g, [(new, 350)], 4, 2, 128, 16, torch.bfloat16)
    high = torch.where(table % 2 == 0, joint.shape[0] - 1 - table, table)
    for c in range(2):
        joint[high[0].long(), c] = caches[c][table[0].long()]
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, high, 4, cache), 0.1)
    small = append.PagedCache(*caches)
    assert torch.equal(got, chunk.chunk_attention(q, small, chunk.ChunkStep(starts, seqs, table, 4, small), 0.1))


def test_a_long_row_of_tokens(device):
    """One token of a request of 2^18 keys, and a window at its end."""
    g = torch.Generator(device=device).manual_seed(8)
    n = 1 << 18
    q, caches, table, starts, seqs = make(g, [(1, n - 1)], 2, 1, 64, 64, torch.float16)
    cache = append.PagedCache(*caches)
    for window in (0, 5, n):
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 2, cache, window), 0.125)
        check(got, q, caches, table, starts, seqs, window, 0.125, 64)


def test_streams_and_replays(device):
    g = torch.Generator(device=device).manual_seed(10)
    q, caches, table, starts, seqs = make(g, [(4, 5000), (100, 900)], 6, 1, 128, 128, torch.bfloat16)
    cache = append.PagedCache(*caches)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    assert step.workspace_size > 0
    want = chunk.chunk_attention(q, cache, step, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chunk.chunk_attention(q, cache, step, 0.1)
        own = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 6, cache), 0.1)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(own, want)
    graphs = []
    for _ in range(2):                # two graphs of one step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chunk.chunk_attention(q, cache, step, 0.1)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        junk = chunk.chunk_attention(q, cache, step, 0.2)
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out in graphs) and not torch.equal(junk, want)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(ValueError, match="before its calls are captured"):
            chunk.ChunkStep(starts, seqs, table, 6, cache)
        out.zero_()


def test_a_captured_step_reads_its_inputs_anew(device):
    """Write and attention of a mixed step in one graph: rows, positions, slots and
    block table change between replays; two streams run the step at once."""
    g = torch.Generator(device=device).manual_seed(12)
    hq, hk, d, page, dtype = 6, 2, 128, 32, torch.float16
    turn = rotary.Rotary(rotary.rotary_table(900, d, device=device))
    lengths, history = (4, 90), (500, 300)
    starts, seqs, n = [0, 4, 94], [504, 390], 94
    caches = [torch.randn(60, page, hk, d, generator=g, device=device).to(dtype) for _ in range(2)]
    cache = append.PagedCache(*caches)
    x = torch.zeros(n, hq + 2 * hk, d, device=device, dtype=dtype)
    q, k, v = x.split((hq, hk, hk), 1)
    pos, slots = torch.zeros(n, dtype=torch.int64, device=device), torch.zeros(n, dtype=torch.int64, device=device)
    table = torch.zeros(2, 16, dtype=torch.int32, device=device)
    step = chunk.ChunkStep(starts, seqs, table, hq, cache)

    def run(cache):
        return chunk.chunk_attention(append.append_rotated(q, k, v, pos, turn, cache, slots), cache, step, 0.1)

    def change():
        x.copy_(torch.randn(x.shape, generator=g, device=device))
        pos.copy_(torch.randint(0, 900, (n,), generator=g, device=device))
        table.copy_(torch.randperm(60, generator=g, device=device)[:32].view(2, 16))
        slots.copy_(torch.cat([table[i].long()[(h + torch.arange(m, device=device)) // page] * page
                               + (h + torch.arange(m, device=device)) % page
                               for i, (m, h) in enumerate(zip(lengths, history))]))

    change()
    run(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(cache)
    side = torch.cuda.Stream()
    for _ in range(3):
        change()
        copies = [c.clone() for c in caches]
        other = append.PagedCache(*copies)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            want = run(other)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(caches, copies))
        keys, values = gather(caches, table[1], seqs[1], page)
        o, bound = expected(rotary.rotate(q, None, pos, turn)[0][4:], keys, values, history[1], 0, 0.1)
        assert ((out[4:].double() - o).abs() <= bound).all()


def test_append_then_attend(device):
    """A prompt, its follow-up chunk and MTP steps of two requests, rotated on
    image positions, written and read; against the formula over all tokens."""
    g = torch.Generator(device=device).manual_seed(11)
    hq, hk, d, page, rd, dtype = 6, 2, 128, 32, 64, torch.bfloat16
    axes = rotary.section_axes((11, 11, 10), interleaved=True)
    turn = rotary.Rotary(rotary.rotary_table(2000, rd, device=device), axes=axes)
    caches = [torch.full((40, page, hk, d), math.nan, dtype=dtype, device=device) for _ in range(2)]
    cache = append.PagedCache(*caches)
    table = torch.randperm(40, generator=g, device=device).to(torch.int32).view(2, 20)
    total = [0, 0]
    kept = [[[], []], [[], []]]
    for lengths in ((100, 37), (200, 1), (4, 4), (1, 130), (4, 2)):
        n = sum(lengths)
        x = torch.randn(n, hq + 2 * hk, d, generator=g, device=device).to(dtype)
        q, k, v = x.split((hq, hk, hk), 1)
        pos = torch.randint(0, 2000, (3, n), generator=g, device=device)
        slots = []
        for i, m in enumerate(lengths):
            at = torch.arange(total[i], total[i] + m, device=device)
            slots.append(table[i][at // page].long() * page + at % page)
        q_turned = append.append_rotated(q, k, v, pos, turn, cache, torch.cat(slots))
        k_turned = rotary.rotate(k, None, pos, turn)[0]
        starts, seqs = [0, lengths[0], n], [t + m for t, m in zip(total, lengths)]
        got = chunk.chunk_attention(q_turned, cache, chunk.ChunkStep(starts, seqs, table, hq, cache), d ** -0.5)
        for i, m in enumerate(lengths):
            a, b = starts[i], starts[i + 1]
            kept[i][0].append(k_turned[a:b])
            kept[i][1].append(v[a:b])
            o, bound = expected(rotary.rotate(q, None, pos, turn)[0][a:b], torch.cat(kept[i][0]), torch.cat(kept[i][1]),
                                total[i], 0, d ** -0.5)
            assert ((got[a:b].double() - o).abs() <= bound).all()
            total[i] += m


@pytest.mark.parametrize("d, reqs, hq, hk", [(256, [(1, 32767)] * 300, 2, 1), (128, [(1, 32767)] * 600, 2, 1),
                                             (64, [(1, 32767)] * 1100, 2, 1), (64, [(2048, 32768)], 32, 4),
                                             (128, [(2048, 32768)], 32, 4), (256, [(1024, 24576)], 32, 4)])
@pytest.mark.parametrize("below", [24.59375, 22.40625])
def test_many_faint_keys_beside_one_keep_their_share(device, d, reqs, hq, hk, below):
    """fp16: the first key outweighs each of the others by 2^below, and those together
    are half a percent of a row and more.  (All requests read the same pages.)  The
    weights are rounded in fp16 relative to 2^7 of the largest's, so one below 2^-14 is
    off by 2^-25, which is 2^-32 of the row's sum; else the bounds above, with B = |o|."""
    n, h = reqs[0]
    seq, page = n + h, 128
    pages = -(-seq // page)
    keys = torch.zeros(pages, page, hk, d, device=device, dtype=torch.float16)
    keys[..., 0] = -below
    keys[0, 0, :, 0] = 0
    feature = 1 + torch.arange(d, device=device) / d                     # (exact in fp16)
    values = feature.half().expand(pages, page, hk, d).clone()
    values[0, 0] = 0
    cache = append.PagedCache(keys, values)
    starts = [n * i for i in range(len(reqs) + 1)]
    table = torch.arange(pages, device=device, dtype=torch.int32).expand(len(reqs), pages)
    q = torch.zeros(starts[-1], hq, d, device=device, dtype=torch.float16)
    q[..., 0] = 1
    scale = math.log(2)
    step = chunk.ChunkStep(starts, [seq] * len(reqs), table, hq, cache)
    got = chunk.chunk_attention(q, cache, step, scale).double()
    others = (seq - n + torch.arange(n, device=device, dtype=torch.float64)).repeat(len(reqs))[:, None, None]
    weight = math.exp(-below * scale)
    o = others * weight / (1 + others * weight) * feature.double()
    eps = 2.0 ** -10
    bound = eps / 2 * 2 * o + eps / 2 * o * (1 + eps) + (2 * below * scale * (d + 2) * 2.0 ** -24 + 2.0 ** -20) * o
    bound += others * 2.0 ** -32 * 2 + torch.finfo(torch.float16).smallest_normal * eps / 2
    off = (got - o).abs() - bound
    assert off.max().item() <= 0, f"off by {off.max().item():.3e} more than the bound"


@pytest.mark.parametrize("dtype, above", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_at_the_edge_of_a_raise_do_not_depend_on_their_neighbours(device, dtype, above, d):
    """A score so little above the limit for raising the maximum (2^8 of it) that its
    weight rounds to the limit, beside rows whose scores go far beyond: the row is the
    same among copies of itself."""
    n, h, page = 32, 64, 32
    keys, values = (torch.zeros(3, page, 1, d, device=device, dtype=dtype) for _ in range(2))
    keys[1, :4, 0, 0], keys[1, :4, 0, 1] = 8, above                      # the second tile, the third is not seen:
    keys[2, :, 0, 0] = -60
    values[0, :, 0] = (1 + torch.arange(d, device=device) / d).to(dtype)
    cache = append.PagedCache(keys, values)
    table = torch.arange(3, device=device, dtype=torch.int32)[None]
    q = torch.ones(n, 2, d, device=device, dtype=dtype)
    q[1::2, :, 0] = 10
    step = chunk.ChunkStep([0, n], [n + h], table, 2, cache)
    assert step.args.wide == 1
    got = chunk.chunk_attention(q, cache, step, math.log(2))
    alone = chunk.chunk_attention(q[:1].expand(n, 2, d), cache, step, math.log(2))
    assert torch.equal(got[0], alone[0]) and torch.equal(got[::2], alone[::2])


def test_pages_past_32_bits_of_an_int64_table_are_left_out(device):
    """Entries that name pages of the cache modulo 2^32, and those at the ends of both types."""
    g = torch.Generator(device=device).manual_seed(23)
    q, caches, table, starts, seqs = make(g, [(3, 230)], 4, 2, 64, 32, torch.bfloat16)
    cache = append.PagedCache(*caches)
    for far in ((1 << 32) + 1, -(1 << 32), (1 << 31) + 2, (1 << 63) - 1, -(1 << 63), -1):
        bad = table.clone()
        bad[0, 2] = -1
        wide = table.long()
        wide[0, 2] = far
        want = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, bad, 4, cache), 0.1)
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, wide, 4, cache), 0.1)
        assert torch.equal(got, want)
    want = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 4, cache), 0.1)
    for dtype in (torch.uint8, torch.int16):
        step = chunk.ChunkStep(starts, seqs, table.to(dtype), 4, cache)
        assert torch.equal(chunk.chunk_attention(q, cache, step, 0.1), want)


def test_strides_of_single_tokens_and_heads_mean_nothing(device):
    """One token's query and output of any token stride, one head's of any head stride."""
    g = torch.Generator(device=device).manual_seed(24)
    for (n, hq, hk), token, head in (((1, 6, 2), 6 * 64 + 1, 64), ((5, 1, 1), 64, 67), ((1, 1, 1), 3, 5)):
        q, caches, table, starts, seqs = make(g, [(n, 50)], hq, hk, 64, 16, torch.bfloat16)
        cache = append.PagedCache(*caches)
        step = chunk.ChunkStep(starts, seqs, table, hq, cache)
        want = chunk.chunk_attention(q, cache, step, 0.125)
        store = torch.zeros(2, 4000, device=device, dtype=torch.bfloat16)
        mine, out = (x.as_strided((n, hq, 64), (token, head, 1)) for x in store)
        mine.copy_(q)
        assert chunk.chunk_attention(mine, cache, step, 0.125, out=out) is out and torch.equal(out, want)
        assert torch.equal(chunk.chunk_attention(mine, cache, step, 0.125), want)


def test_outputs_that_overlap_the_queries_are_refused(device):
    g = torch.Generator(device=device).manual_seed(26)
    q, caches, table, starts, seqs = make(g, [(40, 50)], 4, 2, 64, 16, torch.bfloat16)
    cache = append.PagedCache(*caches)
    step = chunk.ChunkStep(starts, seqs, table, 4, cache)
    want = chunk.chunk_attention(q, cache, step, 0.125)
    x = torch.zeros(41, 8, 64, device=device, dtype=torch.bfloat16)
    x[:40, :4] = q
    for out in (x[1:, :4], x[:40, 2:6], x[:40, 1:5]):
        with pytest.raises(_lib.OscarKernelError, match="overlaps"):
            chunk.chunk_attention(x[:40, :4], cache, step, 0.125, out=out)
    assert torch.equal(x[:40, :4], q)
    assert torch.equal(chunk.chunk_attention(x[:40, :4], cache, step, 0.125, out=x[:40, 4:]), want)
    assert torch.equal(chunk.chunk_attention(x[:40, :4], cache, step, 0.125, out=x[:40, :4]), want)


@pytest.mark.parametrize("kind", ["int32", "int64"])
def test_a_capture_that_waits_for_the_step(device, kind):
    """A step built on one stream just before another one, which waits for it, begins
    to capture a call by hand; replays there and on the first stream."""
    g = torch.Generator(device=device).manual_seed(31)
    q, caches, table, starts, seqs = make(g, [(4, 5000), (100, 900)], 6, 1, 128, 128, torch.bfloat16)
    table = table.to(getattr(torch, kind))
    cache = append.PagedCache(*caches)
    want = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 6, cache), 0.1)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    big = torch.ones(1 << 28, device=device)
    for _ in range(10):
        big.mul_(1.0)                       # (a millisecond and more of other work ahead of the copy)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        out = chunk.chunk_attention(q, cache, step, 0.1)
        graph.capture_end()
        graph.replay()
    side.synchronize()
    assert torch.equal(out, want)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
