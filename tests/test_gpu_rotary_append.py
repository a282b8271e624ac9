"""Position rotation and the plain cache's write on the GPU, against the formula
in 64 bits.

Tolerance of a turned value y = x1 c - x2 s (the table's entries taken as they
are): three fp32 roundings of terms no larger than |x1| + |x2|, then one
rounding to the type: 2^-23 (|x1| + |x2|) + eps / 2 |y|, and half of the type's
smallest step.  Values that pass through, and caches' untouched slots, are equal
bit for bit."""
import pytest
import torch

from oscar_amd.kernels import _lib, append, rotary

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def turned(x, positions, turn, adjacent, axes, inverse=False):
    """(y, bound) in 64 bits of x [N, H, D] on the CPU; positions [axes, N]."""
    rd = turn.rotary_dim
    half = rd // 2
    x64, table = x.double().cpu(), turn.table.double().cpu()
    pos = positions.cpu().reshape(-1, x.shape[0])
    y, reach = x64.clone(), torch.zeros_like(x64)
    for j in range(half):
        row = table[pos[axes[j] if axes is not None else 0]]
        c, s = row[:, j, None], row[:, half + j, None] * (-1 if inverse else 1)
        a, b = (2 * j, 2 * j + 1) if adjacent else (j, j + half)
        y[..., a], y[..., b] = x64[..., a] * c - x64[..., b] * s, x64[..., b] * c + x64[..., a] * s
        reach[..., a] = reach[..., b] = x64[..., a].abs() + x64[..., b].abs()
    info = torch.finfo(x.dtype)
    step = info.smallest_normal * info.eps / 2
    bound = torch.where(reach > 0, 2.0 ** -23 * reach + info.eps / 2 * y.abs() + step, 0.0)
    return y, bound


def close(got, want):
    y, bound = want
    off = (got.double().cpu() - y).abs() - bound
    assert off.max().item() <= 0, f"off by {off.max().item():.3e} more than the bound"


def rows(g, n, hq, hk, d, dtype, fused):
    x = torch.randn(n, hq + 2 * hk, d, generator=g, device="cuda:0") * 3
    parts = x.to(dtype).split((hq, hk, hk), 1)
    return parts if fused else [p.contiguous() for p in parts]


# (head size, rotary_dim): 16-byte pieces and, where halves or heads are no
# multiple of them, single pairs
SHAPES = [(256, 64), (128, 128), (64, 32), (96, 48), (80, 80), (64, 24), (66, 6), (2, 2), (256, 256)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d, rd", SHAPES)
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotate(device, dtype, d, rd, adjacent):
    g = torch.Generator(device=device).manual_seed(d * rd + adjacent)
    for n, hq, hk, fused, axes in ((1, 6, 1, False, None), (5, 3, 2, True, None), (1037, 2, 1, True, None),
                                   (33, 12, 4, False, 3)):
        pair_axes = None if axes is None else [int(a) for a in torch.randint(0, 3, (rd // 2,))]
        if pair_axes is not None:
            pair_axes[0] = 2
        turn = rotary.Rotary(rotary.rotary_table(5000, rd, device=device), adjacent, pair_axes)
        q, k, _ = rows(g, n, hq, hk, d, dtype, fused)
        pos = torch.randint(0, 5000, (turn.axes, n), generator=g, device=device)
        for inverse in (False, True):
            got = rotary.rotate(q, k, pos[0] if turn.axes == 1 else pos, turn, inverse=inverse)
            close(got[0], turned(q, pos, turn, adjacent, pair_axes, inverse))
            close(got[1], turned(k, pos, turn, adjacent, pair_axes, inverse))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_in_place_equals_new_tensors(device, dtype):
    g = torch.Generator(device=device).manual_seed(3)
    for d, rd, adjacent in ((256, 64, False), (64, 64, True), (66, 6, False), (66, 6, True)):
        turn = rotary.Rotary(rotary.rotary_table(300, rd, device=device), adjacent)
        q, k, _ = rows(g, 211, 5, 2, d, dtype, True)
        pos = torch.arange(211, device=device)
        want_q, want_k = rotary.rotate(q, k, pos, turn)
        got_q, got_k = rotary.rotate(q, k, pos, turn, query_out=q, key_out=k)
        assert got_q is q and got_k is k and torch.equal(q, want_q) and torch.equal(k, want_k)


def test_gradient_is_the_inverse(device):
    """d/dx of sum(g . rotate(x)): the formula's, autograd's of the plain form in
    64 bits, and central differences of the kernel in fp32."""
    g = torch.Generator(device=device).manual_seed(4)
    turn = rotary.Rotary(rotary.rotary_table(100, 32, device=device), axes=rotary.section_axes((6, 5, 5)))
    pos = torch.randint(0, 100, (3, 7), generator=g, device=device)
    x = torch.randn(7, 2, 48, generator=g, device=device)
    w = torch.randn(7, 2, 48, generator=g, device=device)
    grad, _ = rotary.rotate(w, None, pos, turn, inverse=True)
    axes = rotary.section_axes((6, 5, 5))
    close(grad, turned(w, pos, turn, False, axes, inverse=True))
    leaf = x.double().cpu().requires_grad_()
    table = turn.table.double().cpu()
    index = torch.arange(16)
    token = pos.cpu()[torch.tensor(axes)].t()
    c, s = table[token, index][:, None], table[token, index + 16][:, None]
    a, b = leaf[..., :16], leaf[..., 16:32]
    y = torch.cat((a * c - b * s, b * c + a * s, leaf[..., 32:]), -1)
    (y * w.double().cpu()).sum().backward()
    reach = torch.ones_like(leaf) * 2.0 ** -22 * w.abs().max().item() * 2
    assert ((grad.double().cpu() - leaf.grad).abs() <= reach).all()
    # the map is linear, so a difference of step 1 has only the sums' roundings:
    # 7 * 2 * 48 terms below 4 * 4 = 16 each, in fp32 products
    for at in ((0, 0, 0), (3, 1, 17), (6, 0, 31), (2, 1, 40)):
        up, down = x.clone(), x.clone()
        up[at] += 0.5
        down[at] -= 0.5
        diff = sum(sign * (rotary.rotate(z, None, pos, turn)[0].double() * w.double()).sum().item()
                   for sign, z in ((1, up), (-1, down)))
        assert diff == pytest.approx(grad[at].item(), abs=4 * 16 * 2.0 ** -23)


def test_positions_outside_the_table_leave_rows_alone(device):
    turn = rotary.Rotary(rotary.rotary_table(10, 32, device=device), axes=[0, 1] * 8)
    pos = torch.tensor([[0, 9, 10, 3, -1, 2], [0, 9, 3, 1 << 40, 4, 9]], device=device)
    q = torch.randn(6, 3, 64, device=device).bfloat16()
    out = torch.full_like(q, 7.0)
    rotary.rotate(q, None, pos, turn, query_out=out)
    bad = torch.tensor([2, 3, 4])
    assert (out[bad] == 7.0).all()
    good = torch.tensor([0, 1, 5])
    close(out[good], turned(q[good], pos[:, good], turn, False, [0, 1] * 8))


@pytest.mark.parametrize("dtype", TYPES[:2], ids=str)
@pytest.mark.parametrize("layout", ["apart", "joint", "heads_first", "stacked"])
@pytest.mark.parametrize("n, hq, hk, d, rd, page", [(1, 6, 1, 256, 64, 128), (4, 6, 1, 256, 64, 128),
                                                   (301, 8, 8, 64, 64, 16), (77, 12, 2, 128, 96, 48),
                                                   (50, 3, 3, 72, 12, 32), (1500, 7, 1, 128, 128, 1)])
def test_append(device, dtype, layout, n, hq, hk, d, rd, page):
    g = torch.Generator(device=device).manual_seed(n + d)
    pages = n // page + 5
    if layout == "joint":
        both = torch.randn(pages, 2, page, hk, d, generator=g, device=device).to(dtype)
        caches = [both[:, 0], both[:, 1]]
    elif layout == "heads_first":
        caches = [torch.randn(pages, hk, page, d, generator=g, device=device).to(dtype).transpose(1, 2)
                  for _ in range(2)]
    elif layout == "stacked":
        caches = list(torch.randn(2, pages, page, hk, d, generator=g, device=device).to(dtype))
    else:
        caches = [torch.randn(pages, page, hk, d, generator=g, device=device).to(dtype) for _ in range(2)]
    before = [c.clone() for c in caches]
    turn = rotary.Rotary(rotary.rotary_table(4096, rd, device=device), adjacent=layout == "joint")
    q, k, v = rows(g, n + 3, hq, hk, d, dtype, layout != "apart")       # three padding rows
    pos = torch.randint(0, 4096, (n,), generator=g, device=device)
    slots = torch.randperm(pages * page, generator=g, device=device)[:n]
    if n > 4:
        slots[::7] = -1
        slots[1], slots[2], slots[3] = pages * page, (1 << 40) + 5, -(1 << 40)
    got = append.append_rotated(q, k, v, pos, turn, append.PagedCache(*caches), slots)
    assert got.shape == (n, hq, d)
    close(got, turned(q[:n], pos, turn, turn.args.adjacent, None))
    live = (slots >= 0) & (slots < pages * page)
    at = slots[live]
    keys = caches[0].reshape(-1, hk, d)[at]
    y, bound = turned(k[:n], pos, turn, turn.args.adjacent, None)
    close(keys, (y[live.cpu()], bound[live.cpu()]))
    assert torch.equal(caches[1].reshape(-1, hk, d)[at], v[:n][live])
    rest = torch.ones(pages * page, dtype=torch.bool, device=device)
    rest[at] = False
    for c, b in zip(caches, before):
        assert torch.equal(c.reshape(-1, hk, d)[rest], b.reshape(-1, hk, d)[rest])


def test_append_leaves_out_tokens_without_a_position(device):
    turn = rotary.Rotary(rotary.rotary_table(10, 64, device=device))
    cache = append.PagedCache(*(torch.zeros(2, 16, 1, 64, device=device, dtype=torch.bfloat16) for _ in range(2)))
    x = torch.ones(4, 1, 64, device=device, dtype=torch.bfloat16)
    out = torch.full_like(x, 5.0)
    append.append_rotated(x, x, x, torch.tensor([1, 10, -1, 9], device=device), turn, cache,
                          torch.tensor([3, 4, 5, 6], device=device), query_out=out)
    written = cache.v_cache.view(32, 64)[:, 0] != 0
    assert written.nonzero().flatten().tolist() == [3, 6]
    assert (cache.k_cache.view(32, 64)[4:6] == 0).all() and (out[1:3] == 5.0).all() and (out[0] != 5.0).any()


def test_append_without_query_and_without_tokens(device):
    turn = rotary.Rotary(rotary.rotary_table(10, 64, device=device))
    cache = append.PagedCache(*(torch.zeros(2, 16, 1, 64, device=device, dtype=torch.float16) for _ in range(2)))
    x = torch.ones(4, 1, 64, device=device, dtype=torch.float16)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    assert append.append_rotated(None, x, x, none, turn, cache, none) is None
    assert append.append_rotated(x, x, x, none, turn, cache, none).shape == (0, 1, 64)
    assert (cache.v_cache == 0).all()
    # int32 positions and slots, every other entry of longer tensors
    pos = torch.arange(8, device=device, dtype=torch.int32)[::2]
    append.append_rotated(None, x, x, pos, turn, cache, torch.arange(8, device=device, dtype=torch.int32)[::2])
    assert (cache.v_cache.view(32, 64)[:8:2] == 1).all() and (cache.v_cache.view(32, 64)[1:8:2] == 0).all()
    assert rotary.rotate(x[:0], None, none, turn)[0].shape == (0, 1, 64)


def test_offsets_past_32_bits(device):
    """Pages more than 2^32 bytes apart (one tensor of 6 GB of which two pages are used)."""
    base = torch.empty(3 << 30, dtype=torch.bfloat16, device=device)
    page = 16 * 64
    pages = base.numel() // page
    caches = [base.view(pages, 16, 1, 64), torch.zeros(8, 16, 1, 64, dtype=torch.bfloat16, device=device)]
    with pytest.raises(ValueError, match="share"):
        append.PagedCache(*caches)
    joint = base.view(pages // 2, 2, 16, 1, 64)
    cache = append.PagedCache(joint[:, 0], joint[:, 1])
    turn = rotary.Rotary(rotary.rotary_table(10, 64, device=device))
    x = torch.randn(2, 1, 64, device=device).bfloat16()
    slots = torch.tensor([0, pages // 2 * 16 - 1], device=device)
    joint[0], joint[-1] = 0, 0
    append.append_rotated(None, x, x, torch.tensor([0, 0], device=device), turn, cache, slots)
    assert torch.equal(joint[0, 1, 0], x[0]) and torch.equal(joint[-1, 1, 15], x[1])
    assert torch.equal(joint[-1, 0, 15], x[1])          # position 0 turns nothing


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("adjacent", [False, True])
def test_more_rows_than_the_caches_hold(device, dtype, adjacent):
    """More than 128 MB of rows take another way to memory; some of them checked."""
    g = torch.Generator(device=device).manual_seed(11)
    turn = rotary.Rotary(rotary.rotary_table(3000, 32, device=device), adjacent)
    n = (150 << 20) // (10 * 64 * dtype.itemsize)
    q, k, v = rows(g, n, 6, 2, 64, dtype, True)
    pos = torch.randint(0, 3000, (n,), generator=g, device=device)
    some = torch.cat([torch.arange(40), torch.arange(n - 40, n), torch.randint(0, n, (200,))]).to(device)
    got = rotary.rotate(q, k, pos, turn)
    close(got[0][some], turned(q[some], pos[some], turn, adjacent, None))
    close(got[1][some], turned(k[some], pos[some], turn, adjacent, None))
    if dtype == torch.float32:
        return                              # (a cache is bf16 or fp16)
    caches = [torch.zeros(-(-n // 16) + 1, 16, 2, 64, device=device, dtype=dtype) for _ in range(2)]
    slots = torch.randperm(16 * (caches[0].shape[0] - 1), generator=g, device=device)[:n]
    out = append.append_rotated(q, k, v, pos, turn, append.PagedCache(*caches), slots)
    assert torch.equal(out, got[0])
    flat = [c.view(-1, 2, 64) for c in caches]
    assert torch.equal(flat[0][slots], got[1]) and torch.equal(flat[1][slots], v)
    assert all((c[-1] == 0).all() for c in caches)


def test_streams_and_replays(device):
    g = torch.Generator(device=device).manual_seed(9)
    turn = rotary.Rotary(rotary.rotary_table(600, 64, device=device))
    caches = [torch.zeros(40, 16, 2, 64, device=device, dtype=torch.bfloat16) for _ in range(2)]
    cache = append.PagedCache(*caches)
    q, k, v = rows(g, 500, 4, 2, 64, torch.bfloat16, True)
    pos = torch.arange(500, device=device)
    slots = torch.randperm(640, generator=g, device=device)[:500]
    want = append.append_rotated(q, k, v, pos, turn, cache, slots)
    want_caches = [c.clone() for c in caches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = append.append_rotated(q, k, v, pos, turn, cache, slots)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = append.append_rotated(q, k, v, pos, turn, cache, slots)
    for _ in range(3):
        for c in caches:
            c.zero_()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(caches, want_caches))


def test_strides_of_single_tokens_and_heads_mean_nothing(device):
    """One token whose stride is past 4 GiB, one head of an odd stride."""
    g = torch.Generator(device=device).manual_seed(25)
    turn = rotary.Rotary(rotary.rotary_table(30, 32, device=device))
    for (n, h), token, head in (((1, 4), 1 << 33, 64), ((5, 1), 64, (1 << 33) + 1), ((1, 1), 1 << 34, 1 << 34)):
        x = torch.randn(n, h, 64, generator=g, device=device).half()
        pos = torch.arange(n, device=device) + 3
        want, _ = rotary.rotate(x, None, pos, turn)
        mine, out = (torch.zeros(4000, device=device).half().as_strided((n, h, 64), (token, head, 1)) for _ in range(2))
        mine.copy_(x)
        got, _ = rotary.rotate(mine, None, pos, turn, query_out=out)
        assert got is out and torch.equal(out, want)
        if h == 1:
            cache = append.PagedCache(*(torch.zeros(2, 16, 1, 64, device=device).half() for _ in range(2)))
            append.append_rotated(None, mine, mine, pos, turn, cache, torch.arange(n, device=device))
            assert torch.equal(cache.k_cache[0, :n], want) and torch.equal(cache.v_cache[0, :n], x)


def test_outputs_among_the_calls_rows(device):
    """In place in slices of one projection; an exchange is refused."""
    g = torch.Generator(device=device).manual_seed(27)
    turn = rotary.Rotary(rotary.rotary_table(30, 32, device=device))
    x = torch.randn(9, 3, 64, generator=g, device=device).half()
    pos = torch.arange(9, device=device)
    before = x.clone()
    want = rotary.rotate(x[:, :1], x[:, 1:2], pos, turn)
    for call in (lambda: rotary.rotate(x[:, :1], x[:, 1:2], pos, turn, query_out=x[:, 1:2], key_out=x[:, :1]),
                 lambda: rotary.rotate(x[:8], None, pos[:8], turn, query_out=x[1:]),
                 lambda: append.append_rotated(
                     x[:, :1], x[:, 1:2], x[:, 2:], pos, turn,
                     append.PagedCache(*(torch.zeros(1, 16, 1, 64, device=device).half() for _ in range(2))), pos,
                     query_out=x[:, 2:])):
        with pytest.raises(_lib.OscarKernelError, match="overlaps"):
            call()
    assert torch.equal(x, before)
    rotary.rotate(x[:, :1], x[:, 1:2], pos, turn, query_out=x[:, :1], key_out=x[:, 1:2])
    assert torch.equal(x[:, :1], want[0]) and torch.equal(x[:, 1:2], want[1]) and torch.equal(x[:, 2], before[:, 2])


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_flow_through_rotate(device, dtype, inverse):
    """Slices of a projection that requires a gradient: the formula's, turned the other
    way and rounded once; none for tokens that are left out, nor for the values."""
    g = torch.Generator(device=device).manual_seed(28)
    axes = rotary.section_axes((6, 5, 5))
    turn = rotary.Rotary(rotary.rotary_table(100, 32, device=device), axes=axes)
    pos = torch.randint(0, 100, (3, 9), generator=g, device=device)
    x = torch.randn(9, 5, 48, generator=g, device=device).to(dtype).requires_grad_()
    w = torch.randn(9, 4, 48, generator=g, device=device).to(dtype)
    q, k, _ = x.split((3, 1, 1), 1)
    got = rotary.rotate(q, k, pos, turn, inverse=inverse)
    plain = rotary.rotate(q.detach(), k.detach(), pos, turn, inverse=inverse)
    assert all(torch.equal(a, b) and a.requires_grad and not b.requires_grad for a, b in zip(got, plain))
    torch.autograd.backward(got, w.split((3, 1), 1))
    close(x.grad[:, :4], turned(w, pos, turn, False, axes, inverse=not inverse))
    assert (x.grad[:, 4] == 0).all()

    pos[1, 2] = 100                                                     # left out: its rows give and get nothing
    leaf = x.detach()[:, :4].clone().requires_grad_()
    out = rotary.rotate(leaf, None, pos, turn, inverse=inverse)[0]
    kept = torch.tensor([0, 1, 3, 4, 5, 6, 7, 8], device=device)
    grad, = torch.autograd.grad(out, leaf, w)
    y, bound = turned(w[kept], pos[:, kept], turn, False, axes, inverse=not inverse)
    close(grad[kept], (y, bound))
    assert (grad[2] == 0).all()


def test_gradients_of_what_requires_them(device):
    """Queries or keys alone, broadcast gradients, differences, second derivatives;
    none without grad mode or into given tensors."""
    g = torch.Generator(device=device).manual_seed(29)
    turn = rotary.Rotary(rotary.rotary_table(100, 32, device=device), adjacent=True)
    pos = torch.randint(0, 100, (7,), generator=g, device=device)
    q, k = (torch.randn(7, h, 48, generator=g, device=device) for h in (2, 1))
    ones = turned(torch.ones_like(q), pos, turn, True, None, inverse=True)
    a = q.clone().requires_grad_()
    out_q, out_k = rotary.rotate(a, k, pos, turn)
    assert out_q.requires_grad
    (out_q.sum() + out_k.sum()).backward()                               # (an expanded gradient)
    close(a.grad, ones)
    b = k.clone().requires_grad_()
    rotary.rotate(q, b, pos, turn)[1].sum().backward()
    close(b.grad, tuple(x[:, :1] for x in ones))
    c, d = q.clone().requires_grad_(), k.clone().requires_grad_()
    rotary.rotate(c, d, pos, turn)[0].sum().backward()                   # (the keys' output is not used)
    close(c.grad, ones)
    assert d.grad is None
    e = torch.randn(9, 1, 48, generator=g, device=device).requires_grad_()      # (more key rows than queries)
    rotary.rotate(q, e, pos, turn)[1].sum().backward()
    close(e.grad[:7], tuple(x[:, :1] for x in ones))
    assert (e.grad[7:] == 0).all()

    # sum(rotate(x)^4) by differences of step h, in 64 bits; |x| <= 3, so |y| <= 4.3, and
    # two outputs depend on an x.  Their third derivatives are 24 |y| <= 104 each: off by
    # h^2 / 6 * 208.  Each y is off by 2^-23 * 6 + 2^-24 * 4.3 <= 2^-20, its fourth power by
    # 4 |y|^3 2^-20 <= 2^-11.6, and four of them over 2 h by 2^-10.6 / h; the gradient, 8
    # roundings of 4 |y|^3 twice, by 2^-24 * 8 * 640 = 2^-11.6
    x = q.clamp(-3, 3).requires_grad_()
    grad, = torch.autograd.grad((rotary.rotate(x, None, pos, turn)[0] ** 4).sum(), x, create_graph=True)
    h = 2.0 ** -5
    for at in ((0, 0, 0), (3, 1, 17), (6, 0, 31), (2, 1, 40)):
        sums = []
        for sign in (1, -1):
            z = x.detach().clone()
            z[at] += sign * h
            sums.append((rotary.rotate(z, None, pos, turn)[0].double() ** 4).sum().item())
        off = h * h / 6 * 208 + 2.0 ** -10.6 / h + 2.0 ** -11
        assert (sums[0] - sums[1]) / (2 * h) == pytest.approx(grad[at].item(), abs=off)
    # d/dx of sum(w grad): 12 rotate back(y^2 rotate(w)); u is off by 8 roundings, 2^-21 of
    # the largest, and two of them make a value
    w = torch.randn(q.shape, generator=g, device=device)
    second, = torch.autograd.grad((grad * w).sum(), x)
    y = rotary.rotate(x.detach(), None, pos, turn)[0].double()
    u = (12 * y ** 2 * rotary.rotate(w, None, pos, turn)[0].double()).float()
    want, bound = turned(u, pos, turn, True, None, inverse=True)
    close(second, (want, bound + 2.0 ** -20 * u.abs().amax().item()))

    with torch.no_grad():
        assert not rotary.rotate(a, b, pos, turn)[0].requires_grad
    into = torch.empty_like(q)
    assert not rotary.rotate(a, None, pos, turn, query_out=into)[0].requires_grad


def test_a_captured_gradient(device):
    """Rotation and gradient in one graph; rows, gradient and positions change between replays."""
    g = torch.Generator(device=device).manual_seed(32)
    turn = rotary.Rotary(rotary.rotary_table(100, 64, device=device))
    x = torch.randn(33, 4, 64, generator=g, device=device).bfloat16().requires_grad_()
    w = torch.randn(33, 4, 64, generator=g, device=device).bfloat16()
    pos = torch.arange(33, device=device)
    rotary.rotate(w, None, pos, turn)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary.rotate(x, None, pos, turn)[0]
        grad, = torch.autograd.grad(out, x, w)
    for last in (32, 99, 100):                                          # (100: left out, no gradient)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=device))
            w.copy_(torch.randn(x.shape, generator=g, device=device))
            pos[32] = last
        graph.replay()
        torch.cuda.synchronize()
        want = torch.zeros_like(w)
        rotary.rotate(w, None, pos, turn, query_out=want, inverse=True)
        assert torch.equal(grad, want)
        assert torch.equal(out[:32], rotary.rotate(x.detach(), None, pos, turn)[0][:32])
        assert (grad[32] == 0).all() == (last == 100)
