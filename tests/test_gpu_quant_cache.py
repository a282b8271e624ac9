"""The 8-bit paged cache's write and its reading, against the definition in 64 bits.

A row's power of two e is the smallest with max|y| <= 448 2^e; a value rounds to the
nearest e4m3 number times 2^e, ties to even.  Values rows and keys that do not turn are
known exactly, so their codes and powers are.  A turned (and normed) key is known within
its fp32 error, 2^-23 (2^-19 normed) of |x1| + |x2|: its stored value is the rounding of
some number in that interval, so it lies between the roundings of the interval's ends,
with the power of the interval's smallest or largest row maximum."""
import pytest
import torch

from oscar_amd.kernels import append, rotary
from tests.test_gpu_norm_rotary import normed, partners, turn64, weights

pytestmark = pytest.mark.gpu
RANGE = {torch.bfloat16: (-80, 100), torch.float16: (-15, 8)}


def power(top, dtype):
    """The exponent of a row maximum (64 bits)."""
    low, high = RANGE[dtype]
    mantissa, e = torch.frexp(top)
    return torch.where(top == 0, low, torch.where(mantissa > 0.875, e - 8, e - 9).clamp(low, high))


def pow2(e):
    return torch.ldexp(torch.ones((), dtype=torch.float64), e)


def rounded(y, e, dtype):
    """y (64 bits) as codes at power e stand for it; what is not finite is NaN."""
    t = y / pow2(e)
    step = pow2(torch.frexp(t.nan_to_num(0.0, 0.0, 0.0)).exponent.clamp(min=-5) - 4)
    most = torch.where(e == RANGE[dtype][1], 240.0, 448.0)
    q = torch.minimum(torch.maximum(torch.round(t / step) * step, -most), most) * pow2(e)
    return torch.where(y.isfinite(), q, float("nan"))


def stored(x, dtype):
    """(values, exponents) of rows that are known exactly."""
    y = x.double().cpu()
    e = power(torch.where(y.isfinite(), y.abs(), 0.0).amax(-1, keepdim=True), dtype)
    return rounded(y, e, dtype), e[..., 0]


def make(g, n, hq, hk, d, dtype, fused, scale=3.0):
    x = torch.randn(n, hq + 2 * hk, d, generator=g, device="cuda:0") * scale
    x[..., ::17] *= 20
    x *= 2.0 ** torch.randint(-6, 3, (n, hq + 2 * hk, 1), generator=g, device="cuda:0")
    parts = x.to(dtype).split((hq, hk, hk), 1)
    return parts if fused else [p.contiguous() for p in parts]


def blank(g, layout, pages, page, hk, d, device):
    if layout == "joint":
        both = torch.randint(0, 256, (pages, 2, page, hk, d), generator=g, device=device, dtype=torch.uint8)
        codes = [both[:, 0], both[:, 1]]
    elif layout == "heads_first":
        codes = [torch.randint(0, 256, (pages, hk, page, d), generator=g, device=device, dtype=torch.uint8)
                 .transpose(1, 2) for _ in range(2)]
    else:
        codes = [torch.randint(0, 256, (pages, page, hk, d), generator=g, device=device, dtype=torch.uint8)
                 for _ in range(2)]
    exponents = torch.randint(0, 256, (pages, hk, page, 2), generator=g, device=device, dtype=torch.uint8)
    return codes, exponents


def values(codes, exponents, i):
    """All slots [slots, Hk, D] of a cache by definition, 64 bits on the CPU."""
    c = codes[i].cpu().contiguous().view(torch.float8_e4m3fn).double()
    return (c * pow2(exponents[..., i].cpu().int().transpose(1, 2)[..., None] - 127)).flatten(0, 1)


SIZES = [(1, 6, 1, 256, 64, 128), (4, 6, 1, 256, 64, 128), (301, 8, 8, 64, 64, 16), (77, 12, 2, 128, 96, 48),
         (50, 3, 3, 80, 24, 32), (1500, 7, 1, 128, 128, 1), (33, 4, 2, 48, 16, 16)]


@pytest.mark.parametrize("dtype", list(RANGE), ids=str)
@pytest.mark.parametrize("layout", ["apart", "joint", "heads_first"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("n, hq, hk, d, rd, page", SIZES)
def test_write(device, dtype, layout, norm, n, hq, hk, d, rd, page):
    g = torch.Generator(device=device).manual_seed(n + d + norm)
    pages = n // page + 5
    codes, exponents = blank(g, layout, pages, page, hk, d, device)
    before = [x.clone() for x in (*codes, exponents)]
    cache = append.QuantCache(*codes, exponents, dtype)
    adjacent = n % 2 == 0
    turn = rotary.Rotary(rotary.rotary_table(4000, rd, device=device), adjacent)
    q, k, v = make(g, n, hq, hk, d, dtype, layout == "apart")
    slots = torch.randperm(pages * page, generator=g, device=device)[:n]
    pos = torch.randint(0, 4000, (n,), generator=g, device=device)
    if n > 4:
        slots[0], slots[1], pos[2] = -1, pages * page, 4000
    w = weights(g, d, torch.float32, 1.0) if norm else (None, None)
    got = append.append_quantized(q, k, v, pos, turn, cache, slots, *w, offset=1.0 if norm else 0.0)
    live = (pos < 4000)
    safe = torch.where(live, pos, 0)
    if norm:
        want, bound = normed(q, w[0], safe, turn, adjacent, None, 1e-6, 1.0)
        key, off = normed(k, w[1], safe, turn, adjacent, None, 1e-6, 1.0)
        off -= torch.finfo(dtype).eps / 2 * key.abs()       # (keys are not rounded to the type on the way)
    else:
        want = turn64(q.double().cpu(), safe, turn, adjacent, None)
        bound = (2.0 ** -23 * partners(q.double().cpu(), turn, adjacent) + torch.finfo(dtype).eps / 2 * want.abs()
                 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)
        key = turn64(k.double().cpu(), safe, turn, adjacent, None)
        off = 2.0 ** -23 * partners(k.double().cpu(), turn, adjacent)
        off[..., rd:] = 0
    alive = live.cpu()
    assert ((got.double().cpu() - want).abs()[alive] <= bound[alive]).all()
    written = (live & (slots >= 0) & (slots < pages * page)).cpu()
    at = slots.cpu()[written]
    # values: exactly
    value, e = stored(v, dtype)
    assert torch.equal(values(codes, exponents, 1)[at], value[written])
    held = exponents.cpu().transpose(1, 2).flatten(0, 1).int() - 127
    assert torch.equal(held[at][..., 1], e[written].int())
    # keys: between the roundings of what fp32 may have made of them, at either's power
    key, off = key[written], off[written]
    low = power((key.abs() - off).clamp(min=0).amax(-1, keepdim=True), dtype)
    high = power((key.abs() + off).amax(-1, keepdim=True), dtype)
    mine = held[at][..., :1]
    assert ((mine == low) | (mine == high)).all()
    stands = values(codes, exponents, 0)[at]
    assert (stands >= rounded(key - off, mine, dtype)).all() and (stands <= rounded(key + off, mine, dtype)).all()
    # every other byte as it was
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[at] = False
    for x, y in zip(codes, before):
        assert torch.equal(x.reshape(-1, hk, d)[rest.to(device)], y.reshape(-1, hk, d)[rest.to(device)])
    assert torch.equal(exponents.transpose(1, 2).reshape(-1, hk, 2)[rest.to(device)],
                       before[2].transpose(1, 2).reshape(-1, hk, 2)[rest.to(device)])


@pytest.mark.parametrize("dtype", list(RANGE), ids=str)
def test_codes_of_every_value(device, dtype):
    """Value rows are known: every finite number of the type, in rows whose maximum is
    each of several, ties among them; zeros, infinities and NaN."""
    every = torch.arange(-(1 << 15), 1 << 15, device=device).to(torch.int16).view(dtype)
    every = every[torch.randperm(1 << 16, generator=torch.Generator(device=device).manual_seed(1), device=device)]
    rows = [every.view(-1, 64)]
    for top in (1.0, 1.75, 1.7578125, 448.0, 449.0, 3.0e-5, 60000.0, 240.0 * 256, 65504.0):
        x = every.view(-1, 64).clone()
        x = torch.where(x.float().abs() <= top, x, (x.float().sign() * top).to(dtype))
        x[:, 0] = top
        rows.append(x)
    x = torch.randn(64, 64, generator=torch.Generator(device=device).manual_seed(2), device=device).to(dtype)
    x[1] = 0
    x[2, 5], x[3, 7], x[4, 9] = float("inf"), float("nan"), -float("inf")
    x[5] = float("nan")
    rows.append(x)
    v = torch.cat(rows)[:, None]
    n = v.shape[0]
    cache = append.quant_cache(-(-n // 16), 16, 1, 64, dtype, device)
    turn = rotary.Rotary(rotary.rotary_table(1, 64, device=device))
    slots = torch.arange(n, device=device)
    append.append_quantized(None, v, v, torch.zeros_like(slots), turn, cache, slots)
    want, e = stored(v, dtype)
    k, got = append.read_back(cache, slots)
    assert got.dtype == dtype
    assert torch.equal(got.double().cpu().nan_to_num(nan=1e300), want.nan_to_num(nan=1e300))
    held = cache.exponents.cpu().transpose(1, 2).flatten(0, 1).int() - 127
    assert torch.equal(held[:n, :, 1], e.int())
    fp32 = append.read_back(cache, slots, dtype=torch.float32)[1]
    assert torch.equal(fp32.double().cpu().nan_to_num(nan=1e300), want.nan_to_num(nan=1e300))


@pytest.mark.parametrize("dtype", list(RANGE), ids=str)
@pytest.mark.parametrize("layout", ["apart", "joint", "heads_first"])
@pytest.mark.parametrize("hk, d, page", [(1, 256, 128), (8, 64, 16), (2, 128, 48), (3, 80, 1), (1, 16, 7)])
def test_read_back(device, dtype, layout, hk, d, page):
    g = torch.Generator(device=device).manual_seed(d)
    codes, exponents = blank(g, layout, 9, page, hk, d, device)
    low, high = RANGE[dtype]
    for c in codes:                          # (240 2^high is the largest a write leaves)
        c.copy_(torch.where((c & 0x7F) > 0x77, 0x55, c))
    exponents.copy_(torch.randint(low + 127, high + 128, exponents.shape, generator=g, device=device))
    cache = append.QuantCache(codes[0].view(torch.float8_e4m3fn), codes[1].view(torch.float8_e4m3fn), exponents, dtype)
    for n in (0, 1, 5, 700):
        slots = torch.randint(-2, 9 * page + 2, (n,), generator=g, device=device)
        live = ((slots >= 0) & (slots < 9 * page)).cpu()
        for kind in (None, torch.float32):
            got = append.read_back(cache, slots, dtype=kind)
            for i in range(2):
                want = values(codes, exponents, i)[torch.where(live, slots.cpu(), 0)]
                want = torch.where(live[:, None, None], want, 0.0)
                assert torch.equal(got[i].double().cpu(), want)
    out = torch.full((4, 5, 2, hk, d), 7.0, dtype=dtype, device=device)
    pair = append.read_back(cache, slots[:4], key_out=out[:, 1, 0], value_out=out[:, 3, 1])
    assert torch.equal(pair[0], append.read_back(cache, slots[:4])[0])
    assert torch.equal(out[:, 3, 1], append.read_back(cache, slots[:4].int())[1])
    out[:, 1, 0], out[:, 3, 1] = 7.0, 7.0
    assert (out == 7.0).all()


def test_slots_past_32_bits(device):
    """A cache of 2^31 slots and more (its codes 34 GB), near its end."""
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("needs 90 GB of GPU memory")
    pages, page, d = (1 << 27) + 3, 16, 16
    codes = torch.empty(2, pages, page, 1, d, dtype=torch.uint8, device=device)
    exponents = torch.empty(pages, 1, page, 2, dtype=torch.uint8, device=device)
    cache = append.QuantCache(codes[0], codes[1], exponents, torch.bfloat16)
    slots = torch.tensor([(1 << 31) + 40, 5, (1 << 31) - 1, 1 << 31], device=device)
    x = torch.randn(4, 1, d, device=device).bfloat16()
    turn = rotary.Rotary(rotary.rotary_table(1, 16, device=device))
    append.append_quantized(None, x, -x, torch.zeros(4, dtype=torch.int64, device=device), turn, cache, slots)
    k, v = append.read_back(cache, slots)
    want, _ = stored(x, torch.bfloat16)
    assert torch.equal(k.double().cpu(), want) and torch.equal(v.double().cpu(), -want)


def test_streams_and_graphs(device):
    g = torch.Generator(device=device).manual_seed(3)
    turn = rotary.Rotary(rotary.rotary_table(100, 64, device=device))
    cache = append.quant_cache(4, 16, 2, 64, torch.bfloat16, device)
    q, k, v = make(g, 20, 4, 2, 64, torch.bfloat16, False)
    w = weights(g, 64, torch.float32, 0.0)
    pos, slots = torch.arange(20, device=device), torch.arange(20, device=device) + 7

    def step():
        turned = append.append_quantized(q, k, v, pos, turn, cache, slots, *w)
        return [turned, *append.read_back(cache, slots)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        g.manual_seed(seed)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=device))
        cache.exponents.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
