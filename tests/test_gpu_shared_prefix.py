"""Attention of requests that share a prefix, over plain pages, against the formula in
64 bits with the tolerance of the chunk attention (the partials that are joined are
fp32: within its 2^-20)."""
import pytest
import torch

from oscar_amd.kernels import append, chunk
from tests.test_gpu_chunk_attention import check, make

pytestmark = pytest.mark.gpu

STEPS = [
    ([(1, 4200), (1, 4100), (1, 4099)], [(0, 3, 4099)]),
    ([(4, 3000 + i) for i in range(32)], [(0, 32, 2999)]),
    ([(1, 100), (2, 500), (0, 3), (3, 600), (1, 40), (7, 999), (5, 800), (1, 31)], [(1, 3, 500), (5, 2, 777)]),
    ([(300, 900), (1, 900), (64, 950)], [(0, 3, 900)]),
    ([(0, 64), (2, 70), (2, 64)], [(0, 3, 64)]),
    ([(1, 31), (1, 31)], [(0, 2, 31)]),
    ([(1, 40 * i + 300) for i in range(70)], [(0, 30, 300), (30, 40, 1500)]),
    ([(17, 33000), (2, 33001)], [(0, 2, 33000)]),
]


def share(table, prefixes, caches, page):
    """The groups' whole pages become their first request's, and broken ones alike."""
    for first, count, keys in prefixes:
        table[first:first + count, :keys // page] = table[first, :keys // page]
        if keys % page:
            own = table[first:first + count, keys // page].long()
            for c in caches:
                c[own, :keys % page] = c[own[0], :keys % page].clone()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_against_the_formula(device, dtype, case):
    reqs, prefixes = STEPS[case]
    g = torch.Generator(device=device).manual_seed(case)
    for hq, hk, d, page, layout in ((6, 1, 256, 128, "apart"), (8, 2, 128, 48, "heads_first"), (4, 4, 64, 16, "joint"),
                                    (7, 1, 64, 64, "apart")):
        q, caches, table, starts, seqs = make(g, reqs, hq, hk, d, page, dtype, layout, spread=2.0)
        share(table, prefixes, caches, page)
        cache = append.PagedCache(*caches)
        step = chunk.ChunkStep(starts, seqs, table, hq, cache, prefixes=prefixes)
        out = torch.full_like(q, 7.0)
        chunk.chunk_attention(q, cache, step, d ** -0.5, out=out)
        check(out, q, caches, table, starts, seqs, 0, d ** -0.5, page)
        again = chunk.chunk_attention(q, cache, step, d ** -0.5)
        assert torch.equal(out, again)


def test_the_prefix_is_read_from_the_first_request(device):
    """The other requests' table need not hold the prefix' pages."""
    g = torch.Generator(device=device).manual_seed(3)
    reqs, page = [(0, 500), (1, 600), (2, 520), (1, 512)], 16
    q, caches, table, starts, seqs = make(g, reqs, 4, 1, 128, page, torch.bfloat16)
    share(table, [(0, 4, 512)], caches, page)
    table[0] = table[1]
    cache = append.PagedCache(*caches)
    want = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 4, cache, prefixes=[(1, 3, 512)]), 0.1)
    table[2:, :512 // page] = -1
    got = chunk.chunk_attention(q, cache, chunk.ChunkStep(starts, seqs, table, 4, cache, prefixes=[(1, 3, 512)]), 0.1)
    assert torch.equal(got, want) and want.isfinite().all()


def test_unmapped_pages_and_hidden_values(device):
    """A prefix of unmapped pages is no key of anyone's; NaN in it reaches all of its
    requests and no other, NaN in a request's own keys that request."""
    g = torch.Generator(device=device).manual_seed(4)
    reqs, page = [(1, 300), (2, 256), (1, 300)], 16
    q, caches, table, starts, seqs = make(g, reqs, 4, 1, 128, page, torch.bfloat16)
    prefixes = [(0, 2, 256)]
    share(table, prefixes, caches, page)
    cache = append.PagedCache(*caches)
    step = lambda t: chunk.ChunkStep(starts, seqs, t, 4, cache, prefixes=prefixes)       # noqa: E731
    want = chunk.chunk_attention(q, cache, step(table), 0.1)
    gone = table.clone()
    gone[:2, :16] = -1
    got = chunk.chunk_attention(q, cache, step(gone), 0.1)
    keys, values = (c[table[0, 16:].long()].reshape(-1, 1, 128)[:45] for c in caches)
    s = (q[0].double() @ keys[:, 0].double().t()) * 0.1
    assert torch.allclose(got[0].double(), torch.softmax(s, -1) @ values[:, 0].double(), atol=2e-2)
    caches[1][table[0, 3].long(), 5] = float("nan")
    got = chunk.chunk_attention(q, cache, step(table), 0.1)
    assert got[:3].isnan().all() and torch.equal(got[3:], want[3:])
    caches[1][table[0, 3].long(), 5] = 0.0
    caches[1][table[0, 17].long(), 5] = float("inf")
    got = chunk.chunk_attention(q, cache, step(table), 0.1)
    assert not got[0].isfinite().any() and got[1:].isfinite().all()


def test_graph_and_streams(device):
    g = torch.Generator(device=device).manual_seed(5)
    reqs, prefixes, page = [(1, 2100 + i) for i in range(12)], [(0, 12, 2048)], 32
    q, caches, table, starts, seqs = make(g, reqs, 6, 1, 256, page, torch.bfloat16)
    share(table, prefixes, caches, page)
    cache = append.PagedCache(*caches)
    step = chunk.ChunkStep(starts, seqs, table, 6, cache, prefixes=prefixes)
    chunk.chunk_attention(q, cache, step, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = chunk.chunk_attention(q, cache, step, 0.1)
    side = torch.cuda.Stream()
    for seed in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device=device))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = chunk.chunk_attention(q, cache, step, 0.1)
        graph.replay()
        want = chunk.chunk_attention(q, cache, step, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(other, want)
        check(held, q, caches, table, starts, seqs, 0, 0.1, page)


FULL = [
    ([(0, 900), (4, 1900), (3, 1930), (900, 1900), (2, 1905), (1400, 2000), (1, 1900), (5, 2011)], [(0, 8, 1900)]),
    ([(1200, 100), (1, 100), (2, 100), (1000, 130), (1, 96)], [(0, 4, 100)]),
    ([(1, 333), (1300, 333), (1100, 400)], [(0, 3, 333)]),
]


@pytest.mark.parametrize("dtype, bits", [(torch.bfloat16, 16), (torch.float16, 16), (torch.bfloat16, 8), (torch.float16, 8)],
                         ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(FULL)))
def test_prompts_that_fill_the_gpu(device, dtype, bits, d, case):
    """They compute the prefix themselves, from the first one's pages too, the last of which may
    hold other keys in theirs; their own table rows need not hold it."""
    from tests import test_gpu_quant_attention as quant

    reqs, prefixes = FULL[case]
    hq, hk, page = 16, 4, 48
    g = torch.Generator(device=device).manual_seed(10 * case + d)
    if bits == 8:
        q, cache, table, starts, seqs = quant.make(g, reqs, hq, hk, d, page, dtype)
        caches = [cache.k_codes, cache.v_codes, cache.exponents.transpose(1, 2)]
    else:
        q, caches, table, starts, seqs = make(g, reqs, hq, hk, d, page, dtype, "joint", spread=2.0)
        cache = append.PagedCache(*caches)
    assert sum(n * 4 for n, _ in reqs if n >= 32) * hk > 256 * 128
    step = chunk.ChunkStep(starts, seqs, table, hq, cache, prefixes=prefixes)
    assert sum(p[-1] for p in prefixes) >= 100
    sizes = step.args.chunk if bits == 8 else step.args
    sharing = [n for n, _ in reqs if 0 < n < 32]
    assert sizes.wide > 0 and sizes.parts <= len(sharing) * hk
    first, count, keys = prefixes[0]
    at = next(i for i in range(first, first + count) if reqs[i][0])
    whole = keys // 32 * 32
    # what the others' rows stand for, as a table of their own
    full = table.clone()
    full[first:first + count, :whole // page] = table[at, :whole // page]
    rest = whole % page
    for i in range(first, first + count):
        table[i, :whole // page] = table[at, :whole // page] if i == at else -1
        if rest and i != at and reqs[i][0]:       # (one without tokens has no such page)
            page_of, own = full[at, whole // page].long(), full[i, whole // page].long()
            for c in caches:
                c[own, :rest] = c[page_of, :rest]
    step = chunk.ChunkStep(starts, seqs, table, hq, cache, prefixes=prefixes)
    out = torch.full_like(q, 7.0)
    chunk.chunk_attention(q, cache, step, d ** -0.5, out=out)
    if bits == 8:
        quant.check(out, q, cache, full, starts, seqs, 0, d ** -0.5)
    else:
        check(out, q, caches, full, starts, seqs, 0, d ** -0.5, page)
    # the same, whatever their own pages hold in the prefix' places
    for i in range(first, first + count):
        if rest and i != at and reqs[i][0]:       # (one without tokens has no such page)
            for c in caches:
                c[full[i, whole // page].long(), :rest] = c[full[at, 0].long(), 1:rest + 1].flip(0)
    assert torch.equal(out, chunk.chunk_attention(q, cache, step, d ** -0.5))
    assert torch.equal(out, chunk.chunk_attention(q.clone(), cache, step, d ** -0.5, out=q))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_hidden_values_of_prompts_that_fill_the_gpu(device, d, bits):
    """NaN in the prefix reaches all rows of its requests; of a request's own keys those that see
    them; pages outside the cache are no keys."""
    from tests import test_gpu_quant_attention as quant

    reqs, prefixes, page, hq, hk = [(1200, 200), (1000, 230), (60, 40)], [(0, 2, 200)], 16, 16, 4
    g = torch.Generator(device=device).manual_seed(d)
    if bits == 8:
        q, cache, table, starts, seqs = quant.make(g, reqs, hq, hk, d, page, torch.bfloat16)
        values, nan = cache.v_codes, 0x7F
    else:
        q, caches, table, starts, seqs = make(g, reqs, hq, hk, d, page, torch.bfloat16)
        cache, values, nan = append.PagedCache(*caches), caches[1], float("nan")
    table[0, 3] = -1
    table[1, :12] = -1
    step = chunk.ChunkStep(starts, seqs, table, hq, cache, prefixes=prefixes)
    clean = chunk.chunk_attention(q, cache, step, 0.1)
    assert clean.isfinite().all()
    marks = [(0, 5, 1), (0, 191, 2), (1, 300, 3), (0, 1399, 4), (1, 195, 5), (0, 50, 6)]   # request, key, feature
    touched = torch.zeros_like(clean, dtype=torch.bool)
    for r, key, feature in marks:
        if table[r, key // page] < 0:
            continue
        values[table[r, key // page].long(), key % page, 1, feature] = nan
        for i in (0, 1) if key < 192 else (r,):
            n, h = reqs[i]
            sees = h + torch.arange(n, device=device) >= key
            touched[starts[i]:starts[i + 1], 4:8, feature] |= sees[:, None]
    got = chunk.chunk_attention(q, cache, step, 0.1)
    assert torch.equal(got.isnan(), touched) and torch.equal(got[~touched], clean[~touched])
