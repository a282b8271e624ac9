"""Chunk attention over the 8-bit cache, against the formula in 64 bits over the values
the codes stand for, with the tolerance of the chunk attention.  What differs from the
plain cache stays within it: weights are rounded with V's power in them, so each is off
by eps / 2 of itself as there, and the sum they are divided by is of unrounded ones
(the tolerance grants both).  In fp16 the largest weight is at least 2^7, so one below
2^-14 is off by 2^-25 of a unit in which that key's largest value is at least 2^7 * 224:
far below the 2^-25 max |v| a key that is granted.
Weights and products below fp32's smallest normal number, 2^-126, may be taken as zero:
in units in which the heaviest key's weight is at least 1, so each key may be off by
2^-126 of its |v|, and where V's power is in the weight by 2^-126 * 448 of the heaviest
key's power, less than 2^-126 * 2 max |v|: t * 2^-125 max |v| in all.  (Scores of 100 and
more show it: a first run without this term was off by 5e-36 over 340 keys, |v| up to
14000, which it grants 1e-31.)"""
import math

import pytest
import torch

from oscar_amd.kernels import append, chunk, rotary
from tests.test_gpu_chunk_attention import DECODE, PROMPTS, expected
from tests.test_gpu_norm_rotary import weights
from tests.test_gpu_shared_prefix import STEPS

pytestmark = pytest.mark.gpu


def powers(g, shape, dtype, spread):
    """Exponents around those of values near 1, and some far off."""
    e = torch.randint(-8, -4, shape, generator=g, device="cuda:0")
    far = torch.rand(shape, generator=g, device="cuda:0") < 0.05
    return torch.where(far, e + torch.randint(-spread, 3, shape, generator=g, device="cuda:0"), e)


def make(g, reqs, hq, hk, d, page, dtype, layout="apart", spread=7, scale=1.0):
    """A cache of shuffled pages, its block table, queries of a step of (new, history) requests."""
    need = [max(1, -(-(n + h) // page)) for n, h in reqs]
    pages = sum(need) + 2
    shape = {"joint": (pages, 2, page, hk, d), "heads_first": (2, pages, hk, page, d)}.get(layout, (2, pages, page, hk, d))
    codes = torch.randint(0, 256, shape, generator=g, device="cuda:0").to(torch.uint8)
    codes = torch.where((codes & 0x7F) == 0x7F, 0x35, codes)       # (no NaN)
    k, v = ((codes[:, 0], codes[:, 1]) if layout == "joint" else (codes[0].transpose(1, 2), codes[1].transpose(1, 2))
            if layout == "heads_first" else (codes[0], codes[1]))
    exponents = (powers(g, (pages, hk, page, 2), dtype, spread) + 127).to(torch.uint8)
    cache = append.QuantCache(k, v, exponents, dtype)
    order = torch.randperm(pages, generator=g, device="cuda:0").to(torch.int32)
    table = torch.full((len(reqs), max(need)), -1, dtype=torch.int32, device="cuda:0")
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c]
        at += c
    q = (torch.randn(sum(n for n, _ in reqs), hq, d, generator=g, device="cuda:0") * scale).to(dtype)
    starts = [0]
    for n, _ in reqs:
        starts.append(starts[-1] + n)
    return q, cache, table, starts, [n + h for n, h in reqs]


def values(cache, row, seq):
    """Keys and values [seq, Hk, D] in 64 bits, by the definition."""
    at = torch.arange(seq, device=row.device)
    page, place = row[at // cache.block_size].long(), at % cache.block_size
    out = []
    for i, codes in enumerate((cache.k_codes, cache.v_codes)):
        c = codes.view(torch.uint8)[page, place].contiguous().view(torch.float8_e4m3fn).double()
        e = cache.exponents[page, :, place, i].int() - 127
        out.append(c * torch.ldexp(torch.ones((), dtype=torch.float64, device=row.device), e)[..., None])
    return out


def check(got, q, cache, table, starts, seqs, window, scale, hidden=None):
    for i, seq in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        keys, vals = values(cache, table[i], seq)
        o, bound = expected(q[a:b], keys, vals, seq - (b - a), window, scale, None if hidden is None else hidden[i])
        off = (got[a:b].double() - o).abs() - bound - seq * 2.0 ** -125 * vals.abs().amax()
        assert off.max().item() <= 0, f"request {i}: off by {off.max().item():.3e} more than the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(DECODE + PROMPTS)))
def test_against_the_formula(device, dtype, d, case):
    reqs = (DECODE + PROMPTS)[case]
    g = torch.Generator(device=device).manual_seed(100 * case + d)
    for hq, hk, page, window, layout in ((6, 1, 128, 0, "apart"), (4, 4, 16, 0, "joint"), (8, 2, 48, 100, "heads_first"),
                                         (16, 1, 32, 1, "apart"), (7, 1, 64, 33, "joint")):
        q, cache, table, starts, seqs = make(g, reqs, hq, hk, d, page, dtype, layout)
        step = chunk.ChunkStep(starts, seqs, table, hq, cache, window)
        got = chunk.chunk_attention(q, cache, step, d ** -0.5)
        check(got, q, cache, table, starts, seqs, window, d ** -0.5)
        assert torch.equal(got, chunk.chunk_attention(q, cache, step, d ** -0.5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_shared_prefixes(device, dtype, case):
    reqs, prefixes = STEPS[case]
    g = torch.Generator(device=device).manual_seed(case)
    for hq, hk, d, page, layout in ((6, 1, 256, 128, "apart"), (8, 2, 128, 48, "heads_first"), (4, 4, 64, 16, "joint")):
        q, cache, table, starts, seqs = make(g, reqs, hq, hk, d, page, dtype, layout)
        for first, count, keys in prefixes:
            table[first:first + count, :keys // page] = table[first, :keys // page]
            if keys % page:
                own, whole = table[first:first + count, keys // page].long(), keys % page
                for c in (cache.k_codes, cache.v_codes):
                    c[own, :whole] = c[own[0], :whole].clone()
                cache.exponents[own, :, :whole] = cache.exponents[own[0], :, :whole].clone()
        step = chunk.ChunkStep(starts, seqs, table, hq, cache, prefixes=prefixes)
        got = chunk.chunk_attention(q, cache, step, d ** -0.5)
        check(got, q, cache, table, starts, seqs, 0, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompts_are_those_of_a_plain_cache(device, d):
    """A step of wide pieces alone gives the bits of the same values in 16-bit pages.
    (Requests of 400 rows and more a kv head: those of at most 96 are narrow.)"""
    g = torch.Generator(device=device).manual_seed(d)
    q, cache, table, starts, seqs = make(g, [(200, 333), (1000, 0), (300, 2000)], 4, 2, d, 32, torch.bfloat16)
    slots = torch.arange(cache.pages * 32, device=device)
    plain = append.PagedCache(*(x.view(cache.pages, 32, 2, d) for x in append.read_back(cache, slots)))
    for window in (0, 70):
        got, want = (chunk.chunk_attention(q, c, chunk.ChunkStep(starts, seqs, table, 4, c, window), 0.1)
                     for c in (cache, plain))
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_scores_and_powers_of_any_size(device, dtype):
    """One key dominates, or all weigh alike; values of very different powers, and rows of zeros."""
    g = torch.Generator(device=device).manual_seed(5)
    low, high = ((-80, 100) if dtype == torch.bfloat16 else (-15, 7))
    for scale, spread in ((1.0, 4.0), (1e-6, 1.0), (0.3, 8.0)):
        q, cache, table, starts, seqs = make(g, [(3, 900), (40, 300), (1, 40)], 8, 2, 128, 32, dtype, scale=spread)
        cache.exponents[..., 1] = torch.randint(-12, 6, cache.exponents.shape[:3], generator=g, device=device) + 127
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 8, cache), scale)
        check(got, q, cache, table, starts, seqs, 0, scale)
        # zeros, as a write leaves them, beside any others
        zero = torch.rand(cache.exponents.shape[:3], generator=g, device=device) < 0.4
        cache.exponents[..., 1] = torch.where(zero, low + 127, cache.exponents[..., 1].int()).to(torch.uint8)
        cache.v_codes[zero.transpose(1, 2)] = 0
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 8, cache), scale)
        check(got, q, cache, table, starts, seqs, 0, scale)
    # all zeros, and all of the greatest power
    cache.v_codes.zero_()
    assert (chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 8, cache), 0.1) == 0).all()
    cache.v_codes.fill_(0x30)                # 0.5
    cache.exponents[..., 1] = high + 127
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 8, cache), 0.1)
    check(got, q, cache, table, starts, seqs, 0, 0.1)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_faint_keys_keep_their_share(device, d):
    """24000 keys of 2^-24.6 of one key's weight, fp16, their values 2^4 larger than its."""
    n = 24000
    g = torch.Generator(device=device).manual_seed(2)
    q, cache, table, starts, seqs = make(g, [(1, n)], 2, 1, d, 16, torch.float16)
    q.zero_()
    q[..., 0] = 1.0
    cache.k_codes.zero_()
    cache.exponents.fill_(127)
    cache.v_codes.fill_(0x38)                # 1
    cache.exponents[..., 1] = 127 + 1
    slot = int(table[0, 0]), 3
    cache.k_codes[slot] = torch.tensor([0x7E] + [0] * (d - 1), dtype=torch.uint8, device=device)[None]      # 448
    cache.exponents[slot[0], :, slot[1], 1] = 127 - 3
    scale = 24.6 * math.log(2) / 448
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 2, cache), scale)
    share = n * 2.0 ** -24.6
    want = (0.125 + 2 * share) / (1 + share)
    # the scale is rounded to fp32: 2^-24 of 24.6 binary orders
    assert (got.double() - want).abs().max().item() <= 2.0 ** -11 * want + 2 * share * 24.6 * 2.0 ** -22


@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_lies_in_unseen_slots_does_not_matter(device, d):
    """Slots past a request's keys, other requests' pages: NaN codes, powers of all bytes."""
    g = torch.Generator(device=device).manual_seed(6)
    reqs = [(1, 40), (4, 90), (50, 100), (1, 0), (130, 3)]
    q, cache, table, starts, seqs = make(g, reqs, 6, 1, d, 64, torch.bfloat16)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    want = chunk.chunk_attention(q, cache, step, 0.1)
    used = torch.zeros(cache.pages * 64, dtype=torch.bool, device=device)
    for i, seq in enumerate(seqs):
        at = torch.arange(seq, device=device)
        used[table[i][at // 64].long() * 64 + at % 64] = True
    for c in (cache.k_codes, cache.v_codes):
        c.view(-1, 1, d)[~used] = torch.tensor([0x7F, 0xFF] * (d // 2), dtype=torch.uint8, device=device)
    for byte in (255, 0):
        cache.exponents.view(-1, 2)[~used] = byte
        assert torch.equal(chunk.chunk_attention(q, cache, step, 0.1), want)
    check(want, q, cache, table, starts, seqs, 0, 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_nan_reaches_the_rows_that_see_it(device, dtype, d, window):
    g = torch.Generator(device=device).manual_seed(16)
    for reqs in ([(16, 100), (3, 70)], [(200, 90)], [(8, 90), (2, 33)]):
        q, cache, table, starts, seqs = make(g, reqs, 4, 2, d, 32, dtype)
        table[0, 0] = -1 if reqs[0][1] == 90 else table[0, 0]     # (a tile that is whole, but unmapped)
        step = chunk.ChunkStep(starts, seqs, table, 4, cache, window)
        clean = chunk.chunk_attention(q, cache, step, 0.1)
        n, h = reqs[0]
        at = {h + n // 2: 5, h + n - 2: 7, h + 3: d - 1, max(h - 20, 0) + 16: 2}
        for pos, feature in at.items():
            cache.v_codes[table[0, pos // 32].long(), pos % 32, 0, feature] = 0xFF if feature == 7 else 0x7F
        got = chunk.chunk_attention(q, cache, step, 0.1)
        pos = h + torch.arange(n, device=device)
        touched = torch.zeros_like(got[:n], dtype=torch.bool)
        for p, feature in at.items():
            sees = (pos >= p) & ((pos < p + window) if window else True)
            touched[:, :2, feature] |= sees[:, None]
        assert got[:n][touched].isnan().all()
        assert torch.equal(got[:n][~touched], clean[:n][~touched]) and torch.equal(got[n:], clean[n:])
        # a key that is NaN takes the whole row
        cache.k_codes[table[0, (h + 1) // 32].long(), (h + 1) % 32, 0, 0] = 0x7F
        got = chunk.chunk_attention(q, cache, step, 0.1)
        sees = (pos >= h + 1) & ((pos < h + 1 + window) if window else True)
        assert got[:n][sees][:, :2].isnan().all() and torch.equal(got[:n][~sees][:, 2:], clean[:n][~sees][:, 2:])


def test_unmapped_pages_are_left_out(device):
    g = torch.Generator(device=device).manual_seed(7)
    reqs = [(2, 200), (40, 200), (1, 10), (3, 300)]
    q, cache, table, starts, seqs = make(g, reqs, 4, 2, 128, 32, torch.float16)
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 6], bad[2, 0], bad[3, 9] = -1, cache.pages, 1 << 30, -(1 << 31), -7
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, bad, 4, cache), 0.09)
    hidden = []
    for i, seq in enumerate(seqs):
        gone = (bad[i] != table[i]).repeat_interleave(32)[:seq]
        hidden.append(gone)
    check(got, q, cache, table, starts, seqs, 0, 0.09, hidden)
    assert (got[starts[2]:starts[3]] == 0).all()          # nothing left to see


def test_rows_of_no_request_are_left_alone(device):
    g = torch.Generator(device=device).manual_seed(8)
    for reqs in ([(4, 50), (3, 60)], [(40, 50), (3, 60)]):
        q, cache, table, starts, seqs = make(g, reqs, 6, 1, 64, 16, torch.bfloat16)
        n = len(q)
        padded = torch.cat((q, torch.full((5, 6, 64), math.nan, device=device).bfloat16()))
        out = torch.full((n + 7, 6, 64), 3.0, device=device).bfloat16()
        step = chunk.ChunkStep(starts, seqs, table, 6, cache)
        assert chunk.chunk_attention(padded, cache, step, 0.125, out=out) is out
        assert (out[n:] == 3.0).all()
        check(out, q, cache, table, starts, seqs, 0, 0.125)
        fused = torch.zeros(n, 10, 64, device=device, dtype=torch.bfloat16)
        fused[:, 2:8] = q
        assert torch.equal(chunk.chunk_attention(fused[:, 2:8], cache, step, 0.125), out[:n])
        assert chunk.chunk_attention(q, cache, step, 0.125, out=q) is q and torch.equal(q, out[:n])


@pytest.mark.parametrize("hq, hk, page", [(64, 1, 1024), (40, 1, 16), (33, 1, 240), (66, 2, 128), (1, 1, 4096)])
def test_large_groups_and_pages(device, hq, hk, page):
    g = torch.Generator(device=device).manual_seed(hq + page)
    q, cache, table, starts, seqs = make(g, [(1, 1500), (3, 40), (0, 7), (9, 5000)], hq, hk, 128, page, torch.float16)
    for window in (0, 333):
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, hq, cache, window), 0.09)
        check(got, q, cache, table, starts, seqs, window, 0.09)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_decodes_beside_prompts(device, d):
    g = torch.Generator(device=device).manual_seed(30 + d)
    reqs = [(1, 3001)] * 40 + [(40, 0), (50, 9000)]
    q, cache, table, starts, seqs = make(g, reqs, 4, 4, d, 32, torch.bfloat16)
    for window in (0, 700):
        step = chunk.ChunkStep(starts, seqs, table, 4, cache, window)
        got = chunk.chunk_attention(q, cache, step, 0.1)
        check(got, q, cache, table, starts, seqs, window, 0.1)


@pytest.mark.parametrize("new", [3, 300])
def test_pages_past_32_bits(device, new):
    """A cache of 6 GB (K and V pages in turn) whose last pages are used, at both tile sizes."""
    base = torch.empty(6 << 30, dtype=torch.uint8, device=device)
    joint = base.view(-1, 2, 16, 2, 128)
    pages = joint.shape[0]
    cache = append.QuantCache(joint[:, 0], joint[:, 1],
                              torch.full((pages, 2, 16, 2), 120, dtype=torch.uint8, device=device), torch.bfloat16)
    g = torch.Generator(device=device).manual_seed(new)
    used = torch.tensor([pages - 1 - 3 * i for i in range(40)], dtype=torch.int32, device=device)
    joint[used.long()] = torch.randint(0, 120, (40, 2, 16, 2, 128), generator=g, device=device).to(torch.uint8)
    q = torch.randn(new, 4, 128, generator=g, device=device).bfloat16()
    table = used[None]
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep([0, new], [640], table, 4, cache), 0.01)
    check(got, q, cache, table, [0, new], [640], 0, 0.01)


def test_a_step_of_the_other_cache_is_refused(device):
    g = torch.Generator(device=device).manual_seed(1)
    q, cache, table, starts, seqs = make(g, [(1, 100)], 4, 2, 64, 16, torch.bfloat16)
    plain = append.PagedCache(*(torch.zeros(cache.pages, 16, 2, 64, dtype=torch.bfloat16, device=device) for _ in "kv"))
    for a, b in ((cache, plain), (plain, cache)):
        with pytest.raises(ValueError, match="geometry"):
            chunk.chunk_attention(q, a, chunk.ChunkStep(starts, seqs, table, 4, b), 0.1)


@pytest.mark.parametrize("norm", [False, True])
def test_a_layer_of_both_kinds_of_requests(device, norm):
    """Heads normed and turned, written, and attended to: a prompt, then tokens of users who
    share it, captured and replayed, against the formula over what the cache holds."""
    g = torch.Generator(device=device).manual_seed(11)
    hq, hk, d, page, long = 6, 1, 256, 16, 400
    turn = rotary.Rotary(rotary.rotary_table(2000, 64, device=device))
    w = weights(g, d, torch.bfloat16, 1.0) if norm else [None, None]
    cache = append.quant_cache(64, page, hk, d, torch.bfloat16, device)
    fused = torch.randn(long + 20, hq + 2 * hk, d, generator=g, device=device).bfloat16()
    q, k, v = fused.split((hq, hk, hk), 1)
    # the prompt
    first = torch.arange(25, dtype=torch.int32, device=device)
    slots = torch.arange(long, device=device)
    turned = append.append_quantized(q[:long], k[:long], v[:long], slots, turn, cache, slots, *w, offset=1.0 * norm)
    out = chunk.chunk_attention(turned, cache, chunk.ChunkStep([0, long], [long], first[None], hq, cache), 0.0625)
    check(out, turned, cache, first[None], [0, long], [long], 0, 0.0625)
    # five users of it, four tokens each
    table = torch.cat((first.expand(5, 25), (25 + torch.arange(5, dtype=torch.int32, device=device))[:, None]), 1)
    place = torch.arange(4, device=device)
    slots = ((25 + torch.arange(5, device=device))[:, None] * page + place).flatten()
    pos = (long + place).repeat(5)
    starts, seqs = [4 * i for i in range(6)], [long + 4] * 5
    step = chunk.ChunkStep(starts, seqs, table, hq, cache, prefixes=[(0, 5, long)])
    rows = [x[long:].contiguous() for x in (q, k, v)]

    def layer():
        turned = append.append_quantized(*rows, pos, turn, cache, slots, *w, offset=1.0 * norm)
        return turned, chunk.chunk_attention(turned, cache, step, 0.0625)

    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer()
    side = torch.cuda.Stream()
    for seed in range(3):
        g.manual_seed(seed)
        for x in rows:
            x.copy_(torch.randn(x.shape, generator=g, device=device))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        check(got[1], got[0], cache, table, starts, seqs, 0, 0.0625)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = layer()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_two_graphs_of_a_step(device):
    """Replayed in turn: each has its own workspace."""
    g = torch.Generator(device=device).manual_seed(12)
    q, cache, table, starts, seqs = make(g, [(2, 5000), (60, 700)], 6, 1, 256, 64, torch.bfloat16)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache)
    other = q.flip(0).contiguous()
    want = [chunk.chunk_attention(x, cache, step, 0.1) for x in (q, other)]
    graphs, held = [], []
    for x in (q, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(chunk.chunk_attention(x, cache, step, 0.1))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 300])
def test_rows_of_zeros_whatever_their_power(device, dtype, d, new):
    """Slots that hold zeros with a power below the type's least, as fresh memory of zeros
    does, weigh as any key of zeros: alone, and beside keys of large negative scores,
    where exp2(score - maximum of score + power) would pass fp32 if the power counted."""
    g = torch.Generator(device=device).manual_seed(d)
    q, cache, table, starts, seqs = make(g, [(new, 900), (new, 100)], 4, 2, d, 32, dtype)
    for x in (cache.k_codes, cache.v_codes, cache.exponents):
        x.zero_()
    step = chunk.ChunkStep(starts, seqs, table, 4, cache)
    assert chunk.chunk_attention(q, cache, step, 0.1).eq(0).all()
    page = table[0, 3].long()               # keys 96 .. 127 of request 0, against the queries
    q.copy_(q.abs() + 1)
    cache.k_codes[page], cache.v_codes[page], cache.exponents[page] = 0xF8, 0x70, 127 - 3
    got = chunk.chunk_attention(q, cache, step, 1.0 / d)
    check(got, q, cache, table, starts, seqs, 0, 1.0 / d)


def test_a_much_longer_request_among_many(device):
    """It is cut where the others fill the GPU; nothing else of the step is."""
    g = torch.Generator(device=device).manual_seed(12)
    reqs = [(1, 7 * i % 97) for i in range(260)] + [(2, 8000)] + [(1, 50)] * 3
    for dtype, hq, hk, d, page in ((torch.bfloat16, 6, 2, 256, 128), (torch.float16, 8, 2, 64, 16)):
        q, cache, table, starts, seqs = make(g, reqs, hq, hk, d, page, dtype)
        step = chunk.ChunkStep(starts, seqs, table, hq, cache)
        assert step.args.chunk.joins == hk and step.args.chunk.narrow > len(reqs) * hk + 8
        got = chunk.chunk_attention(q, cache, step, d ** -0.5)
        check(got, q, cache, table, starts, seqs, 0, d ** -0.5)


def test_two_calls_of_a_step_at_once(device):
    """On two streams, into the queries themselves: prompts, cut decodes and a prefix."""
    g = torch.Generator(device=device).manual_seed(13)
    reqs = [(300, 700), (1, 20000), (4, 3000), (4, 3100), (4, 3050)]
    q, cache, table, starts, seqs = make(g, reqs, 4, 2, 128, 32, torch.bfloat16)
    table[3, :93] = table[4, :93] = table[2, :93]
    step = chunk.ChunkStep(starts, seqs, table, 4, cache, prefixes=[(2, 3, 2976)])
    want = chunk.chunk_attention(q, cache, step, 0.1)
    check(want, q, cache, table, starts, seqs, 0, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        rows = [q.clone() for _ in streams]
        torch.cuda.synchronize()
        for x, stream in zip(rows, streams):
            with torch.cuda.stream(stream):
                chunk.chunk_attention(x, cache, step, 0.1, out=x)
        torch.cuda.synchronize()
        for x in rows:
            assert torch.equal(x, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("reqs, gone, prefixes, window", [
    ([(1, 3999)], (), (), 0), ([(1, 4099), (3, 4001)], (), (), 0), ([(2, 1030)], (0, 21, 45, 63), (), 0),
    ([(3, 2000)], (124,), (), 900), ([(1, 1700), (2, 1650), (1, 1633)], (), [(0, 3, 1632)], 0)])
def test_nan_beside_keys_that_are_not_there(device, dtype, d, reqs, gone, prefixes, window):
    """One in every 32 keys, a feature each, where pieces end inside a tile of codes and where
    a page of 16 keys in a tile is outside the cache: each reaches the rows that see it."""
    g = torch.Generator(device=device).manual_seed(len(reqs) + d)
    q, cache, table, starts, seqs = make(g, reqs, 4, 2, d, 16, dtype)
    for first, count, keys in prefixes:
        table[first:first + count, :keys // 16] = table[first, :keys // 16]
    for page in gone:
        table[0, page] = -1
    step = chunk.ChunkStep(starts, seqs, table, 4, cache, window, prefixes=prefixes)
    clean = chunk.chunk_attention(q, cache, step, 0.1)
    assert clean.isfinite().all()
    held = cache.v_codes.clone()
    tiles = range(seqs[0] // 32)
    for at in range(0, len(tiles), d):
        touched = torch.zeros_like(clean, dtype=torch.bool)
        for tile in tiles[at:at + d]:
            feature = tile - at
            pos = 32 * tile + (7 * tile) % 32
            page = table[0, pos // 16].long()
            if page < 0:
                continue
            cache.v_codes[page, pos % 16, 1, feature] = 0x7F if tile % 2 else 0xFF
            for i, (n, h) in enumerate(reqs):
                if i == 0 or any(pos < keys for _, _, keys in prefixes):
                    rows = h + torch.arange(n, device=device)
                    sees = (rows >= pos) & ((rows < pos + window) if window else True)
                    touched[starts[i]:starts[i + 1], 2:, feature] |= sees[:, None]
        got = chunk.chunk_attention(q, cache, step, 0.1)
        assert touched.any()
        assert torch.equal(got.isnan(), touched) and torch.equal(got[~touched], clean[~touched])
        cache.v_codes.copy_(held)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 300])
def test_rows_of_zeros_of_powers_past_the_types(device, dtype, d, new):
    """Codes of zero are zeros under any power byte: they take no other key's weight away."""
    g = torch.Generator(device=device).manual_seed(d + new)
    for byte in (228 if dtype == torch.bfloat16 else 136, 200 if dtype == torch.float16 else 240, 254, 255):
        q, cache, table, starts, seqs = make(g, [(new, 900), (new, 100)], 4, 2, d, 32, dtype)
        cache.exponents[..., 1] = torch.randint(-12, 6, cache.exponents.shape[:3], generator=g, device=device) + 127
        zero = torch.rand(cache.exponents.shape[:3], generator=g, device=device) < 0.4
        cache.exponents[..., 1] = torch.where(zero, byte, cache.exponents[..., 1].int()).to(torch.uint8)
        cache.v_codes[zero.transpose(1, 2)] = 0
        cache.k_codes[3], cache.exponents[3, :, :, 0] = 0, byte          # (keys of zero too)
        got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 4, cache), d ** -0.5)
        check(got, q, cache, table, starts, seqs, 0, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [40, 260, 1000, 30000])
@pytest.mark.parametrize("order", ["rising", "falling", "stripes"])
def test_sums_of_powers_far_apart(device, d, n, order):
    """Keys of equal scores share the sum of weights alike, whatever the powers of their values:
    rows of zeros of the least power, as a write leaves them, and rows of 2^60, in one tile of
    codes or several, one wave or four, one piece or many."""
    g = torch.Generator(device=device).manual_seed(n)
    q, cache, table, starts, seqs = make(g, [(1, n - 1)], 4, 2, d, 16, torch.bfloat16)
    q.zero_()
    key = torch.arange(n, device=device)
    large = {"rising": key >= n // 2, "falling": key < n // 2, "stripes": key // 32 % 2 == 1}[order]
    page, place = table[0][key // 16].long(), key % 16
    cache.exponents[page, :, place, 1] = torch.where(large, 127 + 60, 127 - 80)[:, None].to(torch.uint8)
    cache.v_codes[page[~large], place[~large]] = 0
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 4, cache), 0.1)
    check(got, q, cache, table, starts, seqs, 0, 0.1)


def test_sums_of_powers_far_apart_of_a_prefix(device):
    """A prefix of many rows is computed from converted keys, whose maxima go without powers."""
    g = torch.Generator(device=device).manual_seed(3)
    reqs, keys = [(4, 1700 + i) for i in range(40)], 1696
    for zeros_first in (True, False):
        q, cache, table, starts, seqs = make(g, reqs, 8, 1, 128, 16, torch.bfloat16)
        q.zero_()
        table[:, :keys // 16] = table[0, :keys // 16]
        own, shared = table[:, keys // 16:].reshape(-1), table[0, :keys // 16]
        own = own[own >= 0].long()
        zero, large = (shared.long(), own) if zeros_first else (own, shared.long())
        cache.exponents[zero, ..., 1], cache.exponents[large, ..., 1] = 127 - 80, 127 + 60
        cache.v_codes[zero] = 0
        step = chunk.ChunkStep(starts, seqs, table, 8, cache, prefixes=[(0, 40, keys)])
        assert step.args.chunk.wide > 0 and step.args.chunk.narrow > 0
        got = chunk.chunk_attention(q, cache, step, 0.1)
        check(got, q, cache, table, starts, seqs, 0, 0.1)
