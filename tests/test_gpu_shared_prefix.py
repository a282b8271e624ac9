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
