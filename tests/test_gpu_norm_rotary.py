"""Normed and turned heads on the GPU, and their gradients, against the formula in
64 bits.

Tolerance of y = R(t), t = r x w, r = 1 / sqrt(mean x^2 + eps), w = weight + offset: the
sum of squares of at most 256 features is 16 additions in a lane and 6 over lanes (or
fewer), so it is off by 23 * 2^-24 of itself and r by half of that, a root and a
quotient; t adds w's own rounding and two products: 18 * 2^-24 of it in all.  The
rotation adds three roundings of terms no larger than |t1| + |t2| (a feature that does
not turn: |t|), and the type rounds once: 2^-19 (|t1| + |t2|) + eps / 2 |y| and half of
the type's smallest step.

Of dx = r (u - x^ mean(u x^)), u = R^T(g) w, x^ = r x: each factor is off by at most 24 *
2^-24 (u as y above), the mean by as much again, so 2^-18 of r (|u| + |x^| mean(|u||x^|)),
|u| taken as (|g1| + |g2|) |w|, and the roundings to the type as above.
Of dw = sum of h x^: 2^-19 of the terms' magnitudes, and the additions': at most 20 rows
of heads in a lane, 256 groups, 8 workgroups a place, 8 places and 64 threads: 356, taken
as 420 * 2^-24."""
import pytest
import torch

from oscar_amd.kernels import _lib, append, rotary

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# (head size, rotary_dim): 16-byte pieces and, where halves or heads are no multiple of
# them, single pairs
SHAPES = [(256, 64), (128, 128), (64, 32), (96, 48), (80, 80), (64, 24), (66, 6), (2, 2), (256, 256), (48, 16),
          (192, 64)]


def turn64(x, positions, turn, adjacent, axes, back=False):
    """R(p) x (or R(p)^T x) in 64 bits of x [N, H, D] on the CPU; positions [axes, N]."""
    half = turn.rotary_dim // 2
    y, table = x.clone(), turn.table.double().cpu()
    pos = positions.cpu().reshape(-1, x.shape[0])
    for j in range(half):
        row = table[pos[axes[j] if axes is not None else 0]]
        c, s = row[:, j, None], row[:, half + j, None] * (-1 if back else 1)
        a, b = (2 * j, 2 * j + 1) if adjacent else (j, j + half)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def partners(x, turn, adjacent):
    """|x1| + |x2| at every feature (|x| where it does not turn)."""
    rd = turn.rotary_dim
    size = x.abs()
    head = size[..., :rd]
    pairs = head.unflatten(-1, (rd // 2, 2)) if adjacent else head.unflatten(-1, (2, rd // 2)).transpose(-1, -2)
    both = pairs.sum(-1, keepdim=True).expand(pairs.shape)
    both = both.flatten(-2) if adjacent else both.transpose(-1, -2).flatten(-2)
    return torch.cat((both, size[..., rd:]), -1)


def rounding(y, dtype):
    info = torch.finfo(dtype)
    return info.eps / 2 * y.abs() + info.smallest_normal * info.eps / 2


def normed(x, weight, positions, turn, adjacent, axes, eps, offset):
    """(y, bound) in 64 bits."""
    x64 = x.double().cpu()
    w = weight.double().cpu() + offset
    t = x64 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps) * w
    y = turn64(t, positions, turn, adjacent, axes)
    return y, 2.0 ** -19 * partners(t, turn, adjacent) + rounding(y, x.dtype)


def gradients(x, weight, g, positions, turn, adjacent, axes, eps, offset, live=None):
    """((dx, bound), (dw, bound)) in 64 bits."""
    x64, g64, w = x.double().cpu(), g.double().cpu(), weight.double().cpu() + offset
    if live is not None:
        g64 = g64 * live.cpu()[:, None, None]
    r = 1.0 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps)
    unit = r * x64
    h, reach = turn64(g64, positions, turn, adjacent, axes, back=True), partners(g64, turn, adjacent)
    dx = r * (h * w - unit * (h * w * unit).mean(-1, keepdim=True))
    size = reach * w.abs()
    off = 2.0 ** -18 * r * (size + unit.abs() * (size * unit.abs()).mean(-1, keepdim=True))
    dw, terms = (h * unit).sum((0, 1)), (reach * unit.abs()).sum((0, 1))
    return ((dx, off + rounding(dx, x.dtype)),
            (dw, (2.0 ** -19 + 420 * 2.0 ** -24) * terms + rounding(dw, weight.dtype)))


def close(got, want):
    y, bound = want
    assert got.shape == y.shape
    off = (got.double().cpu() - y).abs() - bound
    assert off.numel() == 0 or off.max().item() <= 0, f"off by {off.max().item():.3e} more than the bound"


def rows(g, n, hq, hk, d, dtype, fused):
    x = torch.randn(n, hq + 2 * hk, d, generator=g, device="cuda:0") * 3
    parts = x.to(dtype).split((hq, hk, hk), 1)
    return parts if fused else [p.contiguous() for p in parts]


def weights(g, d, dtype, offset):
    return [(1 - offset + 0.3 * torch.randn(d, generator=g, device="cuda:0")).to(dtype) for _ in range(2)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d, rd", SHAPES)
@pytest.mark.parametrize("adjacent", [False, True])
def test_norm_rotate(device, dtype, d, rd, adjacent):
    g = torch.Generator(device=device).manual_seed(d * rd + adjacent)
    for n, hq, hk, fused, axes, eps, offset in ((1, 6, 1, False, None, 1e-6, 0.0), (5, 3, 2, True, None, 1e-5, 1.0),
                                                (1037, 2, 1, True, None, 0.0, 0.0), (33, 12, 4, False, 3, 1.0, 1.0)):
        pair_axes = None if axes is None else [int(a) for a in torch.randint(0, 3, (rd // 2,))]
        if pair_axes is not None:
            pair_axes[0] = 2
        turn = rotary.Rotary(rotary.rotary_table(5000, rd, device=device), adjacent, pair_axes)
        q, k, _ = rows(g, n, hq, hk, d, dtype, fused)
        pos = torch.randint(0, 5000, (turn.axes, n), generator=g, device=device)
        given = pos[0] if turn.axes == 1 else pos
        for wdtype in (torch.float32, torch.bfloat16):
            wq, wk = weights(g, d, wdtype, offset)
            got = rotary.norm_rotate(q, k, wq, wk, given, turn, eps, offset)
            close(got[0], normed(q, wq, pos, turn, adjacent, pair_axes, eps, offset))
            close(got[1], normed(k, wk, pos, turn, adjacent, pair_axes, eps, offset))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d, rd", SHAPES)
@pytest.mark.parametrize("adjacent", [False, True])
def test_gradients(device, dtype, d, rd, adjacent):
    g = torch.Generator(device=device).manual_seed(d + rd + adjacent)
    for n, hq, hk, fused, offset, wdtype in ((1, 6, 1, False, 0.0, torch.float32), (5, 3, 2, True, 1.0, torch.bfloat16),
                                             (1037, 2, 1, True, 0.0, torch.float16),
                                             (65, 12, 4, False, 1.0, torch.float32)):
        turn = rotary.Rotary(rotary.rotary_table(500, rd, device=device), adjacent)
        q, k, _ = (x.detach().requires_grad_() for x in rows(g, n, hq, hk, d, dtype, fused))
        wq, wk = (w.requires_grad_() for w in weights(g, d, wdtype, offset))
        pos = torch.randint(0, 500, (n,), generator=g, device=device)
        out = rotary.norm_rotate(q, k, wq, wk, pos, turn, 1e-6, offset)
        grads = [torch.randn(x.shape, generator=g, device=device).to(dtype) for x in out]
        dq, dk, dwq, dwk = torch.autograd.grad(out, (q, k, wq, wk), grads)
        for x, w, go, dx, dw in ((q, wq, grads[0], dq, dwq), (k, wk, grads[1], dk, dwk)):
            assert dx.dtype == dtype and dw.dtype == wdtype
            want = gradients(x.detach(), w.detach(), go, pos, turn, adjacent, None, 1e-6, offset)
            close(dx, want[0])
            close(dw, want[1])


def test_gradient_against_differences(device):
    """The kernel's differences are the formula's (of outputs rounded to fp32: 2^-22 of
    672 terms below 16, over the step), the formula's are its derivative's."""
    g = torch.Generator(device=device).manual_seed(4)
    axes = rotary.section_axes((6, 5, 5))
    turn = rotary.Rotary(rotary.rotary_table(100, 32, device=device), axes=axes)
    pos = torch.randint(0, 100, (3, 7), generator=g, device=device)
    x = torch.randn(7, 2, 48, generator=g, device=device)
    go = torch.randn(7, 2, 48, generator=g, device=device)
    w = weights(g, 48, torch.float32, 0.0)[0]
    (dx, _), (dw, _) = gradients(x, w, go, pos, turn, False, axes, 1e-6, 0.0)

    def both(x, w):
        y = rotary.norm_rotate(x, None, w, None, pos, turn)[0]
        return ((y.double() * go.double()).sum().item(),
                (normed(x.double(), w.double(), pos, turn, False, axes, 1e-6, 0.0)[0] * go.double().cpu()).sum().item())

    step = 2.0 ** -8                          # (exact in the inputs' fp32)
    for at in ((0, 0, 0), (3, 1, 17), (6, 0, 31), (2, 1, 40)):
        up, down = x.clone(), x.clone()
        up[at] += step
        down[at] -= step
        span = (up[at].double() - down[at].double()).item()
        (k1, f1), (k0, f0) = both(up, w), both(down, w)
        assert (k1 - k0) / span == pytest.approx((f1 - f0) / span, abs=672 * 16 * 2.0 ** -22 / span)
        # third derivatives of a unit vector's components are below 16 max|g w| / |x|^2
        assert (f1 - f0) / span == pytest.approx(dx[at].item(), abs=step ** 2 * 16 * 8)
    for at in (0, 17, 47):
        up, down = w.clone(), w.clone()
        up[at] += 0.5
        down[at] -= 0.5
        (k1, f1), (k0, f0) = both(x, up), both(x, down)
        assert f1 - f0 == pytest.approx(dw[at].item(), abs=1e-9 + 2.0 ** -20)       # (linear; up - down is rounded)
        assert k1 - k0 == pytest.approx(f1 - f0, abs=672 * 16 * 2.0 ** -22)


def test_parts_of_the_gradient(device):
    """Any of the four may be asked for alone; broadcast gradients; rows shared by heads."""
    g = torch.Generator(device=device).manual_seed(6)
    turn = rotary.Rotary(rotary.rotary_table(50, 32, device=device))
    pos = torch.arange(9, device=device)
    q, k, _ = rows(g, 9, 4, 2, 64, torch.bfloat16, True)
    wq, wk = weights(g, 64, torch.bfloat16, 0.0)
    for needed in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (2, 3)):
        leaves = [x.detach().clone() for x in (q, k, wq, wk)]
        for i in needed:
            leaves[i].requires_grad_()
        out = rotary.norm_rotate(*leaves, pos, turn)
        (out[0].sum() + out[1].sum()).backward()
        one = torch.ones(1, 1, 1, device=device, dtype=torch.bfloat16)
        for i, x in enumerate(leaves):
            if i not in needed:
                assert x.grad is None
                continue
            x, w = leaves[i % 2], leaves[2 + i % 2]
            want = gradients(x.detach(), w.detach(), one.expand(x.shape), pos, turn, False, None, 1e-6, 0.0)
            close(leaves[i].grad, want[i // 2])
    # one output without a gradient
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, wq, wk)]
    rotary.norm_rotate(*leaves, pos, turn)[1].sum().backward()
    assert leaves[0].grad is None and leaves[2].grad is None and leaves[1].grad is not None
    # one kv head's rows, broadcast over heads: its gradient is the sum of theirs
    base = torch.randn(9, 1, 64, generator=g, device=device).requires_grad_()
    go = torch.randn(9, 4, 64, generator=g, device=device)
    out, _ = rotary.norm_rotate(base.expand(9, 4, 64), None, wq.float(), None, pos, turn)
    got, = torch.autograd.grad(out, base, go)
    (dx, bound), _ = gradients(base.detach().expand(9, 4, 64), wq.float(), go, pos, turn, False, None, 1e-6, 0.0)
    assert ((got.double().cpu() - dx.sum(1, keepdim=True)).abs() <= bound.sum(1, keepdim=True)
            + 4 * 2.0 ** -24 * dx.abs().sum(1, keepdim=True)).all()
    # a second time is refused
    out, _ = rotary.norm_rotate(base, None, wq.float(), None, pos, turn)
    first, = torch.autograd.grad(out.sum(), base, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_in_place_equals_new_tensors(device, dtype):
    g = torch.Generator(device=device).manual_seed(3)
    for d, rd, adjacent in ((256, 64, False), (64, 64, True), (66, 6, False), (66, 6, True)):
        turn = rotary.Rotary(rotary.rotary_table(300, rd, device=device), adjacent)
        q, k, _ = rows(g, 211, 5, 2, d, dtype, True)
        w = weights(g, d, torch.float32, 0.0)
        pos = torch.arange(211, device=device)
        want_q, want_k = rotary.norm_rotate(q, k, *w, pos, turn)
        got_q, got_k = rotary.norm_rotate(q, k, *w, pos, turn, query_out=q, key_out=k)
        assert got_q is q and got_k is k and torch.equal(q, want_q) and torch.equal(k, want_k)


def test_positions_outside_the_table_leave_rows_alone(device):
    g = torch.Generator(device=device).manual_seed(5)
    turn = rotary.Rotary(rotary.rotary_table(10, 32, device=device), axes=[0, 1] * 8)
    pos = torch.tensor([[0, 9, 10, 3, -1, 2], [0, 9, 3, 1 << 40, 4, 9]], device=device)
    q = torch.randn(6, 3, 64, generator=g, device=device).bfloat16()
    w = weights(g, 64, torch.float32, 0.0)[0].requires_grad_()
    out = torch.full_like(q, 7.0)
    rotary.norm_rotate(q, None, w.detach(), None, pos, turn, query_out=out)
    live = torch.tensor([True, True, False, False, False, True], device=device)
    assert (out[~live] == 7.0).all()
    close(out[live], normed(q[live], w.detach(), pos[:, live], turn, False, [0, 1] * 8, 1e-6, 0.0))
    q.requires_grad_()
    out, _ = rotary.norm_rotate(q, None, w, None, pos, turn)
    go = torch.randn(6, 3, 64, generator=g, device=device).bfloat16()
    dq, dw = torch.autograd.grad(out, (q, w), go)
    want = gradients(q.detach(), w.detach(), go, pos.clamp(0, 9), turn, False, [0, 1] * 8, 1e-6, 0.0, live)
    assert (dq[~live] == 0).all()
    close(dq, want[0])
    close(dw, want[1])


def test_rows_of_zeros_and_of_large_values(device):
    turn = rotary.Rotary(rotary.rotary_table(4, 64, device=device))
    w = torch.ones(64, device=device)
    q = torch.zeros(3, 1, 64, device=device)
    q[1] = 1e18
    q[2, 0, 5] = float("nan")
    pos = torch.zeros(3, dtype=torch.int64, device=device)
    got, _ = rotary.norm_rotate(q, None, w, None, pos, turn)
    assert (got[0] == 0).all() and torch.allclose(got[1], torch.ones_like(got[1]), atol=1e-6) and got[2].isnan().all()


def test_many_tokens_add_up_in_order(device):
    """More blocks of tokens than workgroups: gradients of weights, and again the same bits."""
    g = torch.Generator(device=device).manual_seed(8)
    n = 40000
    turn = rotary.Rotary(rotary.rotary_table(n, 64, device=device))
    q = torch.randn(n, 4, 64, generator=g, device=device).requires_grad_()
    w = weights(g, 64, torch.float32, 0.0)[0].requires_grad_()
    go = torch.randn(n, 4, 64, generator=g, device=device)
    pos = torch.arange(n, device=device)
    grads = [torch.autograd.grad(rotary.norm_rotate(q, None, w, None, pos, turn)[0], (q, w), go) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    # 160000 rows on 2048 workgroups of 64 groups: blocks of 16 tokens, 64 rows each, twice at most
    (dx, bound), (dw, off) = gradients(q.detach(), w.detach(), go, pos, turn, False, None, 1e-6, 0.0)
    close(grads[0][0], (dx, bound))
    close(grads[0][1], (dw, off))


def test_no_tokens(device):
    turn = rotary.Rotary(rotary.rotary_table(4, 64, device=device))
    w = torch.ones(64, device=device, requires_grad=True)
    q = torch.zeros(0, 2, 64, device=device, requires_grad=True)
    out, _ = rotary.norm_rotate(q, None, w, None, torch.zeros(0, dtype=torch.int64, device=device), turn)
    dq, dw = torch.autograd.grad(out.sum(), (q, w))
    assert out.shape == dq.shape == (0, 2, 64) and (dw == 0).all()


def test_streams_and_graphs(device):
    """A captured forward and backward, replayed between eager calls, gives the eager results."""
    g = torch.Generator(device=device).manual_seed(9)
    turn = rotary.Rotary(rotary.rotary_table(100, 64, device=device))
    pos = torch.arange(100, device=device)
    q, k = (torch.randn(100, h, 128, generator=g, device=device).bfloat16().requires_grad_() for h in (6, 2))
    w = [x.requires_grad_() for x in weights(g, 128, torch.float32, 0.0)]
    go = [torch.randn(100, h, 128, generator=g, device=device).bfloat16() for h in (6, 2)]

    def step():
        out = rotary.norm_rotate(q, k, *w, pos, turn)
        return [x.detach() for x in (*out, *torch.autograd.grad(out, (q, k, *w), go))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step()
    torch.cuda.current_stream().wait_stream(side)
    eager = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(warm, eager))
    del warm
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        g.manual_seed(seed)
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=g, device=device))
            go[1].copy_(torch.randn(go[1].shape, generator=g, device=device))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_append_normed(device):
    """Against norm_rotate's keys at their slots; all other bytes as they were."""
    g = torch.Generator(device=device).manual_seed(10)
    for dtype, d, rd, page, n in ((torch.bfloat16, 128, 64, 16, 300), (torch.float16, 256, 256, 128, 3),
                                  (torch.bfloat16, 72, 12, 32, 50)):
        turn = rotary.Rotary(rotary.rotary_table(400, rd, device=device))
        caches = [torch.randn(n // page + 4, page, 2, d, generator=g, device=device).to(dtype) for _ in range(2)]
        before = [c.clone() for c in caches]
        q, k, v = rows(g, n, 6, 2, d, dtype, True)
        w = weights(g, d, torch.float32, 1.0)
        slots = torch.randperm(caches[0].shape[0] * page, generator=g, device=device)[:n]
        slots[1] = -1
        pos = torch.randint(0, 400, (n,), generator=g, device=device)
        pos[2] = 400
        want_q, want_k = rotary.norm_rotate(q, k, *w, pos, turn, offset=1.0)
        cache = append.PagedCache(*caches)
        got = append.append_normed(q, k, v, pos, turn, cache, slots, *w, offset=1.0)
        live = (pos < 400)
        assert torch.equal(got[live], want_q[live])
        live &= slots >= 0
        for c, b, x in zip(caches, before, (want_k, v)):
            b.view(-1, 2, d)[slots[live]] = x[live]
            assert torch.equal(c, b)


def test_refusals(device):
    turn = rotary.Rotary(rotary.rotary_table(8, 64, device=device))
    q = torch.zeros(5, 4, 64, device=device)
    w = torch.ones(64, device=device)
    pos = torch.zeros(5, dtype=torch.int64, device=device)
    x = torch.zeros(5, 8, 64, device=device)
    with pytest.raises(_lib.OscarKernelError, match="overlaps"):
        rotary.norm_rotate(x[:, :4], None, w, None, pos, turn, query_out=x[:, 2:6])
    with pytest.raises(ValueError, match="device"):
        rotary.norm_rotate(q, None, w.cpu(), None, pos, turn)


def test_positions_of_any_kind(device):
    """int32 and strided positions, rows of a padded batch behind them."""
    g = torch.Generator(device=device).manual_seed(8)
    turn = rotary.Rotary(rotary.rotary_table(500, 32).to(device))
    wq, wk = weights(g, 64, torch.float32, 0.0)
    q, k = (torch.randn(20, h, 64, generator=g, device=device).bfloat16() for h in (3, 2))
    positions = torch.randint(0, 500, (17,), generator=g, device=device)
    want = rotary.norm_rotate(q[:17], k[:17], wq, wk, positions, turn)
    wide = torch.zeros(17, 3, dtype=torch.int64, device=device)
    wide[:, 1] = positions
    for p in (positions.int(), wide[:, 1], wide.int()[:, 1]):
        for x, y in zip(rotary.norm_rotate(q[:17], k[:17], wq, wk, p, turn), want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d, rd", [(256, 64), (128, 128), (192, 64)])
def test_rows_off_16_bytes(device, dtype, d, rd):
    """Heads whose rows begin at single values: the outputs, the gradient, the writes."""
    g = torch.Generator(device=device).manual_seed(d)
    turn = rotary.Rotary(rotary.rotary_table(500, rd, device=device))
    n = 37
    fused = torch.randn(n, 5 * d + 3, generator=g, device=device).to(dtype)[:, 1:1 + 5 * d].unflatten(1, (5, d))
    q, k, v = fused[:, :3], fused[:, 3:4], fused[:, 4:]
    wq, wk = weights(g, d, torch.float32, 0.0)
    pos = torch.randint(0, 500, (n,), generator=g, device=device)
    out = torch.empty(n, 4 * d + 1, dtype=dtype, device=device)[:, 1:].unflatten(1, (4, d))
    got = rotary.norm_rotate(q, k, wq, wk, pos, turn, query_out=out[:, :3], key_out=out[:, 3:])
    for x, y, w in zip(got, (q, k), (wq, wk)):
        close(x, normed(y, w, pos[None], turn, False, None, 1e-6, 0.0))
    leaf = fused.detach().requires_grad_()
    wq.requires_grad_()
    grad = torch.randn(n, 3 * d + 1, generator=g, device=device).to(dtype)[:, 1:].unflatten(1, (3, d))
    dx, dw = torch.autograd.grad(rotary.norm_rotate(leaf[:, :3], None, wq, None, pos, turn)[0], (leaf, wq), grad)
    want = gradients(q.detach(), wq.detach(), grad, pos, turn, False, None, 1e-6, 0.0)
    close(dx[:, :3], want[0])
    close(dw, want[1])
    assert dx[:, 3:].eq(0).all()
    if dtype == torch.float32:
        return
    slots = torch.randperm(64, generator=g, device=device)[:n]
    caches = [append.quant_cache(4, 16, 1, d, dtype, device) for _ in range(2)]
    for cache, rows_of in zip(caches, (lambda x: x, lambda x: x.contiguous())):
        append.append_quantized(None, rows_of(k), rows_of(v), pos, turn, cache, slots)
    for x in ("k_codes", "v_codes", "exponents"):       # (no norm: the same sums whatever the lanes)
        assert torch.equal(getattr(caches[0], x), getattr(caches[1], x))
