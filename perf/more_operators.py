"""Normed and turned heads, the 8-bit paged cache, and attention that shares a prefix: what is timed of them.

Five operators of the layers around the INT2 path.  ``norm`` gives query and key
heads their norm and their positions in one pass, for training with its
gradient.  ``store`` does that on the way of a step's keys and values into an
8-bit paged cache, and takes them back as later steps will read them.  ``read``
takes whole histories back.  ``attend`` is the causal attention of a step's new
tokens over such a cache.  ``shared`` is that attention, over a 16-bit or an
8-bit cache, for requests that begin with the same keys.  A step is written as
text, one `new@history` entry per request; groups that share a prefix as
`first:count:keys`.

The 8-bit cache: a value is code * 2^(exponent - 127), codes e4m3 [pages, page,
kv heads, head_dim], exponents one byte for each token and head of K and of V
[pages, kv heads, page, 2].  A row's exponent is the smallest with which its
largest magnitude is at most 448 times the power, within [-15, 8] for fp16 rows and
[-80, 100] for bf16 ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EXPONENTS = {"bf16": (-80, 100), "fp16": (-15, 8)}
EPS = 1e-6
POSITIONS = 32768
OUTLIERS = (7, 39, 55)                # key channels of 8 times the others' scale
MOST_FLOPS = 6.8e11                   # of a drawn step: the largest listed one's
MOST_BYTES = 2.7e8                    # of a drawn step's cached keys and values
MOST_VALUES = 30843 * 40 * 128        # of a drawn norm: the largest listed one's features

# One rank's share of the deployment that the framework's own configurations
# describe: 6 query heads on one K/V head of 256 features, 128-token pages.
DEPLOYED = {"type": "bf16", "heads": 6, "kv_heads": 1, "head_dim": 256, "page": 128}

# Histories of 32 concurrent requests, spread over [2048, 16384].
CONCURRENT = (4171, 13250, 9002, 2311, 15777, 6640, 11893, 3527, 14608, 8215, 5099, 12346, 2998, 16201, 7433, 10560,
              4822, 9671, 13999, 3210, 6011, 15102, 8888, 2555, 11047, 7019, 12877, 5450, 10013, 14250, 3777, 9333)


def _rows(name, kind, tokens, **options):
    turn = {"rotary_dim": 64, "adjacent": False, "axes": "", "fused": True, "normed": True, "weight": "bf16",
            "offset": 1.0, "gradient": False, "skipped": 0.0}
    return {"name": name, "kind": kind, "tokens": tokens, **DEPLOYED, **turn, **options}


def _step(name, kind, requests, **options):
    return {"name": name, "kind": kind, "requests": requests, **DEPLOYED, "bits": 8, "window": 0, "prefixes": "",
            **options}


def listed():
    every = ",".join(f"4@{h}" for h in CONCURRENT)
    return [
        # One token of one user.
        _rows("norm 1", "norm", 1),
        # A prompt of text and images: three position axes in turn, query and
        # key as slices of one fused projection.
        _rows("norm image prompt 9256", "norm", 9256, axes="interleaved"),
        # Training: a batch's forward and the gradients of heads and weights.
        _rows("norm training 30843", "norm", 30843, heads=32, kv_heads=8, head_dim=128, rotary_dim=128, fused=False,
              weight="fp32", offset=0.0, gradient=True),
        # The draft layer's write of one MTP step.
        _rows("store 4", "store", 4),
        # A bulk write of prompts with padding slots, in scattered slots, heads
        # without norms, and the rows that the layer's first attention takes back.
        _rows("store 65536", "store", 65536, normed=False, axes="blocks", skipped=0.0625),
        # One user's history, taken back to be read at 16 bits by the layer's long prompt.
        _step("read 24579", "read", "0@24579"),
        # The histories of a busy server, several heads, small pages.
        _step("read 32 of 2-16K", "read", every.replace("4@", "0@"), kv_heads=8, heads=32, head_dim=128, page=16,
              type="fp16"),
        # One user, a short chat: the smallest step there is.
        _step("decode 1x1 1K", "attend", "1@1024"),
        # A busy server: 32 users verifying four MTP tokens each.
        _step("mtp 32x4 2-16K", "attend", every),
        # Chunked prefill: one prompt's chunk beside seven users' MTP steps.
        _step("mixed chunk + 7x4", "attend", "4@5000,4@2711,4096@8192,4@900,4@16000,4@333,4@7777,4@12001", type="fp16",
              heads=32, kv_heads=8, head_dim=128, page=64),
        # Eight users of one system prompt, a token each.
        _step("shared 8x1 over 4K", "shared", ",".join(f"1@{4100 + 77 * i}" for i in range(8)), heads=32, kv_heads=8,
              head_dim=128, page=16, bits=16, prefixes="0:8:4096"),
        # 32 users of one long document verifying four MTP tokens each.
        _step("shared 32x4 over 24579", "shared", ",".join(f"4@{24579 + h // 16}" for h in CONCURRENT),
              prefixes="0:32:24579"),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads = rng.choice(((6, 1), (6, 1), (12, 2), (32, 8), (16, 4), (8, 8), (7, 1), (24, 8), (16, 1)))
    options = {"heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice((64, 128, 128, 256, 256)),
               "page": rng.choice((16, 32, 64, 128, 128, 48)), "type": rng.choice(("bf16", "bf16", "fp16"))}
    d = options["head_dim"]
    kind = rng.choice(("norm", "norm", "store", "store", "read", "attend", "attend", "attend", "shared", "shared"))
    if kind in ("norm", "store"):
        options["rotary_dim"] = d // rng.choice((1, 1, 2, 4))
        options["axes"] = rng.choice(("", "", "blocks", "interleaved"))
        options["adjacent"] = rng.random() < 0.3
        options["fused"] = rng.random() < 0.5
        options["offset"] = rng.choice((0.0, 1.0))
        options["weight"] = rng.choice((options["type"], "fp32"))
        options["normed"] = kind == "norm" or rng.random() < 0.7
        options["skipped"] = rng.choice((0.0, 0.0625)) if kind == "store" else 0.0
        if kind == "norm":
            options["gradient"] = rng.random() < 0.5
            if rng.random() < 0.2:
                options["type"] = "fp32"
                options["weight"] = "fp32"
        most = min(65536, MOST_VALUES // (d * (heads + 2 * kv_heads)))
        if options["type"] == "fp32":
            most //= 2
        case = _rows("", kind, _log(rng, 1, most), **options)
        del case["name"]
        return case

    if kind == "shared":
        options["bits"] = rng.choice((8, 16))
    token = 2 * kv_heads * d * options.get("bits", 8) // 8

    def histories(count, lo):
        most = max(lo + 1, min(32768, int(MOST_BYTES / (count * token))))
        return [_log(rng, lo, most) for _ in range(count)]

    if kind == "read":
        requests = [(0, h) for h in histories(_log(rng, 1, 32), 1)]
    elif kind == "shared":
        new, requests, groups = rng.choice((1, 1, 2, 4, 4, 0)), [], []
        for _ in range(rng.choice((1, 1, 2))):
            count = _log(rng, 2, 48)
            prefix = _log(rng, 32, min(32768, int(8 * MOST_BYTES / (count * token))))
            groups.append((len(requests), count, prefix))
            requests += [(new or rng.randint(1, 64), prefix + _log(rng, 1, 2048) - 1) for _ in range(count)]
        if rng.random() < 0.3:        # users of none
            requests += [(new or 1, h) for h in histories(rng.randint(1, 8), 16)]
        options["prefixes"] = ",".join("%d:%d:%d" % g for g in groups)
    else:
        shape = rng.choice(("decode", "decode", "prefill", "mixed"))
        if shape == "decode":
            new = rng.choice((1, 1, 2, 4, 4, 8, 0))
            requests = [(new or rng.randint(1, 16), h) for h in histories(_log(rng, 1, 64), 1)]
        else:
            requests = [(_log(rng, 17, 9256), 0 if rng.random() < 0.4 else h) for h in histories(rng.randint(1, 3), 16)]
            if shape == "mixed":
                requests += [(rng.choice((1, 2, 4)), h) for h in histories(rng.randint(1, 16), 16)]
                rng.shuffle(requests)
        options["window"] = rng.choice((0, 0, 0, _log(rng, 1, 8192)))
    flops = 4 * d * heads * sum(_visible(n, h, options.get("window", 0)) for n, h in requests)
    if flops > MOST_FLOPS:
        requests = [(max(1, int(n * MOST_FLOPS / flops)), h) for n, h in requests]
    case = _step("", kind, ",".join(f"{n}@{h}" for n, h in requests), **options)
    del case["name"]
    return case


# ------------------------------------------------------------------ sizes
def _requests(case):
    return [tuple(int(x) for x in r.split("@")) for r in case["requests"].split(",")]


def _prefixes(case):
    return [tuple(int(x) for x in g.split(":")) for g in case["prefixes"].split(",") if g]


def _visible(new, history, window):
    """Keys that a request's new tokens see, summed over the tokens."""
    if not window:
        return new * history + new * (new + 1) // 2
    growing = max(0, min(new, window - history))        # tokens that see less than the window
    return growing * history + growing * (growing + 1) // 2 + (new - growing) * window


def work(case):
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    size = TYPES[case["type"]].itemsize
    if case["kind"] in ("norm", "store"):
        n, rd = case["tokens"], case["rotary_dim"]
        rows = n * (hq + hk) * d * size
        nbytes = 2 * rows + n * 8 * (3 if case["axes"] else 1) + min(n, POSITIONS) * rd * 4
        if case["gradient"]:          # g and x read, dx written
            nbytes += 3 * rows
        if case["kind"] == "store":   # keys to codes, values read and to codes, both taken back
            nbytes += n * hk * (-d * size + d + 1 + d * size + d + 1) + n * hk * 2 * (d + 1 + d * size) + n * 16
        return {"bytes": nbytes, "flops": (3 * rd + (6 * d if case["normed"] else 0)) * n * (hq + hk)
                + (16 * n * (hq + hk) * d if case["gradient"] else 0)}
    reqs = _requests(case)
    if case["kind"] == "read":
        n = sum(h for _, h in reqs)
        return {"bytes": n * (8 + 2 * hk * (d + 1 + d * size)), "flops": 2 * n * hk * d}
    seen = [n + h if not case["window"] else min(n + h, n + case["window"] - 1) for n, h in reqs]
    keys = sum(seen)
    for first, count, prefix in _prefixes(case):
        keys -= (count - 1) * prefix
    row = d + 1 if case["bits"] == 8 else d * size
    return {"bytes": size * d * 2 * hq * sum(n for n, _ in reqs) + 2 * hk * row * keys,
            "flops": 4 * d * hq * sum(_visible(n, h, case["window"]) for n, h in reqs)}


# ------------------------------------------------------------------ inputs
def _table(length, rotary_dim):
    """Cosines, then sines, of position * 1e6^(-2j / rotary_dim), fp32 [length, rotary_dim]."""
    turn = 1e6 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(length, dtype=torch.float64)[:, None] * turn
    return torch.cat((angle.cos(), angle.sin()), -1).float().to(DEVICE)


def _pair_axes(case):
    """The position axis each feature pair turns by: time, height and width in
    blocks, or in turn (height and width each a third of the pairs)."""
    pairs = case["rotary_dim"] // 2
    third = pairs // 3
    if not case["axes"]:
        return None
    if case["axes"] == "blocks":
        return [0] * (pairs - 2 * third) + [1] * third + [2] * third
    return [j % 3 if j < 3 * third else 0 for j in range(pairs)]


def _positions(case, host):
    """int64 [tokens], or [3, tokens] of text and images in turn: an image's
    tokens share their time and lie on a grid of height and width."""
    n = case["tokens"]
    if not case["axes"]:
        return np.arange(n, dtype=np.int64) % POSITIONS
    parts, at, left = [], 0, n
    while left > 0:
        text = min(left, int(host.randint(1, 300)))
        parts.append(np.tile(np.arange(at, at + text), (3, 1)))
        at, left = at + text, left - text
        high, wide = int(host.randint(4, 49)), int(host.randint(4, 49))
        grid = np.stack((np.full(high * wide, at), at + np.repeat(np.arange(high), wide),
                         at + np.tile(np.arange(wide), high)))[:, :left]
        parts.append(grid)
        at, left = at + max(high, wide), left - grid.shape[1]
        at %= POSITIONS - 400         # (a batch of several prompts)
    return np.concatenate(parts, 1).astype(np.int64)


def _row_inputs(case, g, host):
    """Query, key and value [tokens, heads, head_dim], slices of one projection or each its own
    tensor; positions; weights of the norms; for a gradient the outputs'; slots."""
    n, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    dtype, weight = TYPES[case["type"]], TYPES[case["weight"]]
    x = torch.randn(n, hq + 2 * hk, d, generator=g, device=DEVICE)
    x[:, hq:hq + hk, list(OUTLIERS)] *= 8.0
    parts = x.to(dtype).split((hq, hk, hk), 1)
    w = dict(zip("qkv", parts if case["fused"] else [p.contiguous() for p in parts]))
    w["positions"] = torch.from_numpy(_positions(case, host)).to(DEVICE)
    w["table"] = _table(POSITIONS, case["rotary_dim"])
    for name in ("wq", "wk"):
        w[name] = (1.0 - case["offset"] + 0.2 * torch.randn(d, generator=g, device=DEVICE)).to(weight)
    if case["gradient"]:
        w["gq"] = torch.randn(n, hq, d, generator=g, device=DEVICE).to(dtype)
        w["gk"] = torch.randn(n, hk, d, generator=g, device=DEVICE).to(dtype)
    if case["kind"] == "store":
        pages = n // case["page"] + 8
        slots = host.permutation(pages * case["page"])[:n].astype(np.int64)
        slots[host.permutation(n)[:int(n * case["skipped"])]] = -1
        w["slots"] = torch.from_numpy(slots).to(DEVICE)
        w["cache"] = _blank(case, pages)
    return w


def _blank(case, pages):
    """An 8-bit cache of zeros: codes of K and of V, exponents."""
    shape = (pages, case["page"], case["kv_heads"], case["head_dim"])
    codes = [torch.zeros(shape, dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn) for _ in range(2)]
    return [*codes, torch.zeros(pages, shape[2], shape[1], 2, dtype=torch.uint8, device=DEVICE)]


def _step_inputs(case, g, host):
    """Shuffled pages (a prefix' whole ones shared by its requests) of random keys and values,
    the block table, queries, starts and lengths."""
    reqs, page, hq, hk, d = _requests(case), case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    need = [max(1, -(-(n + h) // page)) for n, h in reqs]
    given = [0] * len(reqs)           # pages of the group's first request
    for first, count, prefix in _prefixes(case):
        given[first + 1:first + count] = [prefix // page] * (count - 1)
    pages = sum(need) - sum(given) + 3
    order = host.permutation(pages)
    table = np.zeros((len(reqs), max(need)), dtype=np.int32)
    at = 0
    for row, whole, had in zip(table, need, given):
        row[had:whole] = order[at:at + whole - had]
        at += whole - had
    for first, count, prefix in _prefixes(case):
        table[first:first + count, :prefix // page] = table[first, :prefix // page]
    w = {"table": torch.from_numpy(table).to(DEVICE)}
    dtype = TYPES[case["type"]]
    shape = (pages, page, hk, d)
    if case["bits"] == 8:
        w["cache"] = _blank(case, pages)
    else:
        w["cache"] = [torch.zeros(shape, dtype=dtype, device=DEVICE) for _ in range(2)]
    for i, outliers in enumerate((OUTLIERS, ())):
        for a in range(0, pages, 4096 // page):
            x = torch.randn(w["cache"][i][a:a + 4096 // page].shape, generator=g, device=DEVICE)
            x[..., list(outliers)] *= 8.0
            if case["bits"] == 8:
                codes, exponents = _quantise(x, case["type"])
                w["cache"][i].view(torch.uint8)[a:a + 4096 // page] = codes.view(torch.uint8)
                w["cache"][2][a:a + 4096 // page, ..., i] = exponents.transpose(1, 2)
            else:
                w["cache"][i][a:a + 4096 // page] = x.to(dtype)
    # a prefix' last, broken page: each request has its own, of the same keys
    for first, count, prefix in _prefixes(case):
        if prefix % page:
            own, whole = w["table"][first:first + count, prefix // page].long(), prefix % page
            for x in w["cache"][:2]:
                x = x.view(torch.uint8) if case["bits"] == 8 else x
                x[own, :whole] = x[own[0], :whole]
            if case["bits"] == 8:
                w["cache"][2][own, :, :whole] = w["cache"][2][own[0], :, :whole]
    w["q"] = torch.randn(sum(n for n, _ in reqs), hq, d, generator=g, device=DEVICE).to(dtype)
    w["starts"] = np.cumsum([0] + [n for n, _ in reqs]).tolist()
    w["seqs"] = [n + h for n, h in reqs]
    if case["kind"] == "read":        # every key's slot, request by request
        w["slots"] = torch.from_numpy(np.concatenate(
            [row[np.arange(s) // page].astype(np.int64) * page + np.arange(s) % page
             for row, s in zip(table, w["seqs"])])).to(DEVICE)
    return w


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    return (_row_inputs if case["kind"] in ("norm", "store") else _step_inputs)(case, g, host)


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        from oscar_amd.kernels import append, chunk, rotary

        if case["kind"] in ("norm", "store"):         # a model's rotation
            state["turn"] = rotary.Rotary(state["table"], adjacent=case["adjacent"], axes=_pair_axes(case))
        if case.get("gradient"):
            for name in ("q", "k", "wq", "wk"):
                state[name].requires_grad_()
        if "cache" in state:                          # a layer's cache
            cache = state["cache"]
            state["pages"] = (append.QuantCache(*cache, TYPES[case["type"]]) if len(cache) == 3
                              else append.PagedCache(*cache))
        if case["kind"] in ("attend", "shared"):      # a step's request layout, the same for all its layers
            state["step"] = chunk.ChunkStep(state["starts"], state["seqs"], state["table"], case["heads"],
                                            state["pages"], window=case["window"], prefixes=_prefixes(case))
    elif "axes" in case and case["axes"]:
        state["pair_axes"] = torch.tensor(_pair_axes(case), device=DEVICE)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the framework
def _run_own(state):
    from oscar_amd.kernels import append, chunk, rotary

    case = state["case"]
    if case["kind"] == "norm":
        heads = state["q"], state["k"], state["wq"], state["wk"]
        out = rotary.norm_rotate(*heads, state["positions"], state["turn"], eps=EPS, offset=case["offset"])
        if not case["gradient"]:
            return out
        grads = torch.autograd.grad(out, heads, (state["gq"], state["gk"]))
        return [x.detach() for x in (*out, *grads)]
    if case["kind"] == "store":
        weights = (state["wq"], state["wk"]) if case["normed"] else (None, None)
        query = append.append_quantized(state["q"], state["k"], state["v"], state["positions"], state["turn"],
                                        state["pages"], state["slots"], *weights, eps=EPS, offset=case["offset"])
        return [query, *append.read_back(state["pages"], state["slots"])]
    if case["kind"] == "read":
        return append.read_back(state["pages"], state["slots"])
    return chunk.chunk_attention(state["q"], state["pages"], state["step"], case["head_dim"] ** -0.5)


# ------------------------------------------------------------------ plain torch, fp32
def _run_plain(state):
    case = state["case"]
    if case["kind"] == "read":
        return _plain_read(state)
    if case["kind"] in ("attend", "shared"):
        return _plain_attention(state)
    positions, table, half = state["positions"], state["table"], case["rotary_dim"] // 2
    if positions.ndim == 1:
        rows = table[positions]
        cos, sin = rows[:, None, :half], rows[:, None, half:]
    else:                             # every axis' row, then each pair's own
        pick = state["pair_axes"][None, :, None].expand(positions.shape[1], half, 1)
        rows = table[positions.t().contiguous()]                            # [N, axes, rotary_dim]
        cos = rows[..., :half].transpose(1, 2).gather(2, pick).transpose(1, 2)
        sin = rows[..., half:].transpose(1, 2).gather(2, pick).transpose(1, 2)
    normed = [_plain_norm(state[x], state["w" + x], case) for x in "qk"]
    turned = [_plain_rotate(y, cos, sin, case["adjacent"]) for y, _, _ in normed]
    dtype = TYPES[case["type"]]
    if case["kind"] == "norm":
        out = [y.to(dtype) for y in turned]
        if not case["gradient"]:
            return out
        back = [_plain_gradient(_plain_rotate(state["g" + x].float(), cos, -sin, case["adjacent"]), state["w" + x],
                                unit, r, case) for x, (_, unit, r) in zip("qk", normed)]
        return [*out, *(dx for dx, _ in back), *(dw for _, dw in back)]
    slots, page = state["slots"], case["page"]
    live = slots >= 0
    at, codes_k, codes_v, scales = slots[live], *(x.view(torch.uint8) for x in state["cache"])
    for i, (codes, x) in enumerate(((codes_k, turned[1]), (codes_v, state["v"].float()))):
        c, e = _quantise(x[live], case["type"])
        codes[at // page, at % page] = c.view(torch.uint8)
        scales[at // page, :, at % page, i] = e
    return [turned[0].to(dtype), *_plain_read(state)]


def _plain_norm(x, weight, case):
    """(the normed heads, x / rms, 1 / rms); the heads themselves where there is no norm."""
    y = x.float()
    if not case["normed"]:
        return y, None, None
    r = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return y * r * (weight.float() + case["offset"]), y * r, r


def _plain_rotate(y, cos, sin, adjacent):
    half = cos.shape[-1]
    if adjacent:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _plain_gradient(h, weight, unit, r, case):
    """Gradients of heads and of their weights from h, the outputs' turned back."""
    u = h * (weight.float() + case["offset"])
    dx = r * (u - unit * (u * unit).mean(-1, keepdim=True))
    return dx.to(TYPES[case["type"]]), (h * unit).sum((0, 1)).to(weight.dtype)


def _quantise(x, kind):
    """(e4m3 codes, biased exponents) of fp32 rows [..., D]."""
    low, high = EXPONENTS[kind]
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))        # in [0.5, 1)
    e = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)           # 448 = 0.875 * 2^9
    e = torch.where(mantissa == 0, low, e).clamp(low, high)
    scaled = x * _power(-e)
    most = torch.where(e == high, 240.0, 448.0)     # (the next code would pass the type's largest)
    return torch.minimum(torch.maximum(scaled, -most), most).to(torch.float8_e4m3fn), (e[..., 0] + 127).to(torch.uint8)


def _power(e):
    """2^e as it stands in fp32's bits (a power function's last place would move values off a border)."""
    return ((e + 127).int() << 23).view(torch.float32)


def _plain_values(codes, exponents):
    """fp32 rows [..., D] of uint8 codes and exponents [...]."""
    return codes.view(torch.float8_e4m3fn).float() * _power(exponents[..., None].int() - 127)


def _plain_read(state):
    slots, page = state["slots"], state["case"]["page"]
    at = slots.clamp(min=0)
    out = []
    for i in range(2):
        codes = state["cache"][i].view(torch.uint8)[at // page, at % page]
        x = _plain_values(codes, state["cache"][2][at // page, :, at % page, i])
        out.append(torch.where((slots >= 0)[:, None, None], x, 0.0).to(TYPES[state["case"]["type"]]))
    return out


def _plain_attention(state):
    case, q = state["case"], state["q"]
    hq, hk, d, page, window = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "window"))
    group = hq // hk
    out = torch.empty_like(q)
    for i, (a, b, seq) in enumerate(zip(state["starts"], state["starts"][1:], state["seqs"])):
        low = max(0, seq - (b - a) - window + 1) if window else 0
        at = torch.arange(low, seq, device=q.device)
        pages = state["table"][i, at // page].long()
        if case["bits"] == 8:
            keys, values = (_plain_values(state["cache"][n].view(torch.uint8)[pages, at % page],
                                          state["cache"][2][pages, :, at % page, n]) for n in range(2))
        else:
            keys, values = (x[pages, at % page].float() for x in state["cache"])
        keys, values = keys.permute(1, 2, 0).contiguous(), values.transpose(0, 1).contiguous()
        step = max(1, (1 << 28) // (hq * (seq - low)))
        for t in range(a, b, step):   # (a long prompt's scores in parts)
            u = min(b, t + step)
            last = torch.arange(seq - b + t, seq - b + u, device=q.device).repeat_interleave(group)
            rows = q[t:u].float().view(u - t, hk, group, d).transpose(0, 1).reshape(hk, -1, d)
            s = torch.bmm(rows, keys) * d ** -0.5
            hidden = at[None, :] > last[:, None]
            if window:
                hidden = hidden | (at[None, :] <= last[:, None] - window)
            s = s.masked_fill(hidden, -math.inf)
            p = (s - s.amax(-1, keepdim=True)).exp()
            o = torch.bmm(p, values) / p.sum(-1, keepdim=True)
            out[t:u] = o.view(hk, u - t, group, d).transpose(0, 1).reshape(u - t, hq, d).to(q.dtype)
    return out


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    w = _inputs(case, seed)
    if case["kind"] == "read":
        return [_exact_rows(w["cache"][i], w["cache"][2][..., i], w["slots"]) for i in range(2)]
    if case["kind"] in ("attend", "shared"):
        return _exact_attention(case, w)
    pairs = case["rotary_dim"] // 2
    axes = _pair_axes(case) or [0] * pairs
    positions = w["positions"].view(-1, case["tokens"])
    index = torch.arange(pairs, device=DEVICE)
    token = positions[torch.tensor(axes, device=DEVICE)].t()                # [N, pairs]
    wave = torch.complex(w["table"][token, index].double(), w["table"][token, index + pairs].double())[:, None]
    first, second = (2 * index, 2 * index + 1) if case["adjacent"] else (index, index + pairs)

    def turn(x, wave):
        y = x.clone()
        z = torch.complex(y[..., first], y[..., second]) * wave
        y[..., first], y[..., second] = z.real, z.imag
        return y

    turned, dx, dw = [], [], []
    for name in "qk":
        x, weight = w[name].double(), w["w" + name].double() + case["offset"]
        if not case["normed"]:
            turned.append(turn(x, wave))
            continue
        size = torch.sqrt(torch.sum(x * x, -1, keepdim=True) / case["head_dim"] + EPS)
        turned.append(turn(x / size * weight, wave))
        if case["gradient"]:
            back = turn(w["g" + name].double(), wave.conj())
            dw.append(torch.sum(back * x / size, (0, 1)))
            inner = torch.sum(back * weight * x, -1, keepdim=True) / case["head_dim"]
            dx.append(back * weight / size - x * inner / size ** 3)
    if case["kind"] == "norm":
        return [*turned, *dx, *dw]
    out = [turned[0]]
    for x in (turned[1], w["v"].double()):
        y = _exact_rounding(x, *EXPONENTS[case["type"]])
        out.append(torch.where((w["slots"] < 0)[:, None, None], 0.0, y))
    return out


def _exact_power(e):
    """2^e in 64 bits, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rounding(x, low, high):
    """What an 8-bit row stands for: multiples of a step that goes with each value's size."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0)).clamp(low, high)                # (or one off, next to a border)
    e = torch.where(top > 448.0 * _exact_power(e), e + 1, torch.where(top <= 448.0 * _exact_power(e - 1), e - 1, e))
    e = e.clamp(low, high)
    step = _exact_power(torch.frexp(x * _exact_power(-e)).exponent.clamp(min=-5) - 4)
    most = torch.where(e == high, 240.0, 448.0)
    return torch.clamp(torch.round(x * _exact_power(-e) / step) * step, -most, most) * _exact_power(e)


def _exact_rows(codes, exponents, slots):
    """[N, kv heads, D] from the codes' bits: sign, four of exponent, three of mantissa."""
    bits = codes.view(torch.uint8).flatten(0, 1)[slots].to(torch.int64)
    power, low = (bits >> 3) & 15, (bits & 7).double()
    size = torch.where(power == 0, low / 8.0 * 2.0 ** -6, (1.0 + low / 8.0) * _exact_power(power - 7))
    e = exponents.transpose(1, 2).flatten(0, 1)[slots].to(torch.int64) - 127
    return torch.where(bits >= 128, -size, size) * _exact_power(e)[..., None]


def _exact_attention(case, w):
    hq, hk, page, window = case["heads"], case["kv_heads"], case["page"], case["window"]
    scale = case["head_dim"] ** -0.5
    out = []
    for (new, history), row in zip(_requests(case), w["table"]):
        slot = torch.arange(new + history, device=DEVICE)
        slot = row[slot // page].long() * page + slot % page
        if case["bits"] == 8:
            keys, values = (_exact_rows(w["cache"][i], w["cache"][2][..., i], slot) for i in range(2))
        else:
            keys, values = (c.flatten(0, 1)[slot].double() for c in w["cache"])
        keys, values = keys.transpose(0, 1).contiguous(), values.transpose(0, 1).contiguous()
        query = w["q"][len(out):len(out) + new].double().unflatten(1, (hk, hq // hk)).transpose(0, 1).contiguous()
        got = torch.empty_like(query)                                       # [kv_heads, new, group, head_dim]
        part = max(1, (1 << 26) // ((hq // hk) * (new + history)))
        for t in range(0, new, part):
            low = max(0, history + t + 1 - window) if window else 0
            high = min(new + history, history + t + part)
            ahead = torch.arange(low, high, device=DEVICE) - torch.arange(history + t, high, device=DEVICE)[:, None]
            seen = (ahead <= 0) if not window else (ahead <= 0) & (ahead > -window)
            for h in range(hk):
                score = (query[h, t:t + part].flatten(0, 1) @ keys[h, low:high].t()).unflatten(0, (-1, hq // hk))
                score = torch.where(seen[:, None], scale * score, -math.inf)
                got[h, t:t + part] = (torch.softmax(score, -1).flatten(0, 1) @ values[h, low:high]).unflatten(
                    0, (-1, hq // hk))
        out.extend(got.transpose(0, 1).flatten(1, 2))
    return torch.stack(out)
