"""The position rotation, the plain paged cache's write and the attention over it: what is timed of them.

Three operators a serving engine calls on the layers around the INT2 path.
``rotate`` turns query and key heads by their tokens' positions, on one axis or
on several (time, height, width of image and video prompts), forward and
inverse.  ``append`` does that on the way of a step's keys and values into a
plain (bf16 or fp16) paged cache.  ``chunk`` is the causal attention of a step's
new tokens over such a cache.  A step is written as text, one `new@history`
entry per request: "4@24579" is one request with 4 new tokens over 24579 cached
ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
OUTLIERS = (7, 39, 55)                # key channels of 8 times the others' scale
MOST_FLOPS = 1.14e12                  # of a drawn step: the largest listed one's
MOST_BYTES = 270e6                    # of a drawn step's cached keys and values
MOST_VALUES = 30843 * 40 * 128        # of a drawn rotation or write: the largest listed one's features

# One rank's share of the deployment that the framework's own configurations
# describe: 6 query heads on one K/V head of 256 features, 128-token pages.
DEPLOYED = {"type": "bf16", "heads": 6, "kv_heads": 1, "head_dim": 256, "page": 128, "joint": False, "fused": False}

# Histories of 32 concurrent requests, spread over [2048, 16384].
CONCURRENT = (4171, 13250, 9002, 2311, 15777, 6640, 11893, 3527, 14608, 8215, 5099, 12346, 2998, 16201, 7433, 10560,
              4822, 9671, 13999, 3210, 6011, 15102, 8888, 2555, 11047, 7019, 12877, 5450, 10013, 14250, 3777, 9333)


def _rotation(name, kind, tokens, **options):
    turn = {"rotary_dim": 64, "adjacent": False, "axes": "", "inverse": False, "skipped": 0.0}
    return {"name": name, "kind": kind, "tokens": tokens, **DEPLOYED, **turn, **options}


def _step(name, requests, **options):
    return {"name": name, "kind": "chunk", "requests": requests, **DEPLOYED, "window": 0, **options}


def listed():
    return [
        # One token of one user, a quarter of its head's features turned.
        _rotation("rotate 1", "rotate", 1),
        # A prompt of text and images: three position axes in turn, query and
        # key as slices of one fused projection.
        _rotation("rotate image prompt 9256", "rotate", 9256, axes="interleaved", fused=True),
        # Training: the gradient of a batch's queries and keys, whole heads.
        _rotation("rotate gradient 30843", "rotate", 30843, type="fp16", heads=32, kv_heads=8, head_dim=128,
                  rotary_dim=128, adjacent=True, inverse=True),
        # The draft layer's write of one MTP step.
        _rotation("append 4", "append", 4, fused=True),
        # A new prompt, whole heads turned, its keys and values in pages that hold both.
        _rotation("append prompt 3001", "append", 3001, heads=32, kv_heads=8, head_dim=128, rotary_dim=128, page=16,
                  joint=True, fused=True),
        # A bulk write of image tokens with padding slots, in scattered slots.
        _rotation("append 65536", "append", 65536, axes="blocks", skipped=0.0625),
        # One user, a short chat: the smallest step there is.
        _step("decode 1x1 1K", "1@1024"),
        # A busy server: 32 users verifying four MTP tokens each.
        _step("mtp 32x4 2-16K", ",".join(f"4@{h}" for h in CONCURRENT)),
        # Long-context decoding of a few users.
        _step("decode 8x1 32K", ",".join(["1@32768"] * 8)),
        # A long prompt's last chunk over its cached part.
        _step("prefill 9256 over 15K", "9256@15360"),
        # Chunked prefill: one prompt's chunk beside seven users' MTP steps.
        _step("mixed chunk + 7x4", "4@5000,4@2711,1024@4096,4@900,4@16000,4@333,4@7777,4@12001", type="fp16", heads=32,
              kv_heads=8, head_dim=128, page=64),
        # Two prompts in a sliding-window layer of small heads.
        _step("window prompts 6000 + 1501", "6000@0,1501@4500", heads=16, kv_heads=4, head_dim=64, page=32, joint=True,
              fused=True, window=1024),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads = rng.choice(((6, 1), (6, 1), (12, 2), (32, 8), (16, 4), (8, 8), (7, 1), (24, 8), (16, 1)))
    options = {"heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice((64, 128, 128, 256, 256)),
               "page": rng.choice((16, 32, 64, 128, 128, 48)), "type": rng.choice(("bf16", "bf16", "fp16")),
               "joint": rng.random() < 0.3, "fused": rng.random() < 0.5}
    kind = rng.choice(("rotate", "rotate", "append", "append", "chunk", "chunk", "chunk", "chunk", "chunk"))
    if kind != "chunk":
        if kind == "rotate" and rng.random() < 0.25:
            options["type"] = "fp32"
        options["rotary_dim"] = options["head_dim"] // rng.choice((1, 1, 2, 4))
        options["axes"] = rng.choice(("", "", "blocks", "interleaved"))
        options["adjacent"] = rng.random() < 0.3
        options["inverse"] = kind == "rotate" and rng.random() < 0.3
        options["skipped"] = rng.choice((0.0, 0.0625)) if kind == "append" else 0.0
        most = min(65536, MOST_VALUES // (options["head_dim"] * (heads + 2 * kv_heads)))
        if options["type"] == "fp32":
            most //= 2
        case = _rotation("", kind, _log(rng, 1, most), **options)
        del case["name"]
        return case

    d = options["head_dim"]
    token = 4 * kv_heads * d          # bytes of a cached token

    def histories(count, lo):
        most = max(lo + 1, min(32768, int(MOST_BYTES / (count * token))))
        return [_log(rng, lo, most) for _ in range(count)]

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
    flops = 4 * d * heads * sum(_visible(n, h, options["window"]) for n, h in requests)
    if flops > MOST_FLOPS:
        requests = [(max(1, int(n * MOST_FLOPS / flops)), h) for n, h in requests]
    case = _step("", ",".join(f"{n}@{h}" for n, h in requests), **options)
    del case["name"]
    return case


# ------------------------------------------------------------------ sizes
def _requests(case):
    return [tuple(int(x) for x in r.split("@")) for r in case["requests"].split(",")]


def _visible(new, history, window):
    """Keys that a request's new tokens see, summed over the tokens."""
    if not window:
        return new * history + new * (new + 1) // 2
    growing = max(0, min(new, window - history))        # tokens that see less than the window
    return growing * history + growing * (growing + 1) // 2 + (new - growing) * window


def work(case):
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    size = TYPES[case["type"]].itemsize
    if case["kind"] == "chunk":
        reqs = _requests(case)
        seen = [n + h if not case["window"] else min(n + h, n + case["window"] - 1) for n, h in reqs]
        return {"bytes": size * d * (2 * hq * sum(n for n, _ in reqs) + 2 * hk * sum(seen)),
                "flops": 4 * d * hq * sum(_visible(n, h, case["window"]) for n, h in reqs)}
    n, rd = case["tokens"], case["rotary_dim"]
    axes = 3 if case["axes"] else 1
    nbytes = n * (2 * (hq + hk) * d * size + 8 * axes)
    if case["kind"] == "append":
        written = n - int(n * case["skipped"])
        nbytes += n * (hk * d * size + 8) + written * hk * d * size - (n - written) * hk * d * size
    nbytes += min(n, 32768) * rd * 4
    return {"bytes": nbytes, "flops": 3 * n * (hq + hk) * rd}


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
        return np.arange(n, dtype=np.int64) % 32768
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
        at %= 32768 - 400             # (a batch of several prompts)
    return np.concatenate(parts, 1).astype(np.int64)


def _heads(case, g, n):
    """Query, key and value [n, heads, head_dim]: slices of one projection, or each its own tensor."""
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    x = torch.randn(n, hq + 2 * hk, d, generator=g, device=DEVICE)
    x[:, hq:hq + hk, list(OUTLIERS)] *= 8.0
    x = x.to(TYPES[case["type"]])
    parts = x.split((hq, hk, hk), 1)
    return parts if case["fused"] else [p.contiguous() for p in parts]


def _caches(case, pages):
    """K and V pages [pages, page, kv_heads, head_dim]: two tensors, or views of one whose pages hold both."""
    shape = (case["page"], case["kv_heads"], case["head_dim"])
    if case["joint"]:
        both = torch.zeros(pages, 2, *shape, dtype=TYPES[case["type"]], device=DEVICE)
        return [both[:, 0], both[:, 1]]
    return [torch.zeros(pages, *shape, dtype=TYPES[case["type"]], device=DEVICE) for _ in range(2)]


def _inputs(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    w = {}
    if case["kind"] != "chunk":
        n = case["tokens"]
        w["q"], w["k"], w["v"] = _heads(case, g, n)
        w["positions"] = torch.from_numpy(_positions(case, host)).to(DEVICE)
        w["table"] = _table(32768, case["rotary_dim"])
        if case["kind"] == "append":
            pages = n // case["page"] + 8
            slots = host.permutation(pages * case["page"])[:n].astype(np.int64)
            slots[host.permutation(n)[:int(n * case["skipped"])]] = -1
            w["slots"] = torch.from_numpy(slots).to(DEVICE)
            w["caches"] = _caches(case, pages)
        return w
    reqs = _requests(case)
    page = case["page"]
    need = [-(-(n + h) // page) for n, h in reqs]
    pages = sum(need) + 3
    order = host.permutation(pages)
    table = np.zeros((len(reqs), max(need)), dtype=np.int32)
    for row, first, count in zip(table, np.cumsum([0] + need), need):
        row[:count] = order[first:first + count]
    w["table"] = torch.from_numpy(table).to(DEVICE)
    w["caches"] = _caches(case, pages)
    for cache, outliers in zip(w["caches"], (OUTLIERS, ())):
        for a in range(0, pages, 256):
            x = torch.randn(cache[a:a + 256].shape, generator=g, device=DEVICE)
            x[..., list(outliers)] *= 8.0
            cache[a:a + 256] = x.to(cache.dtype)
    w["q"] = _heads(case, g, sum(n for n, _ in reqs))[0]
    w["starts"] = np.cumsum([0] + [n for n, _ in reqs]).tolist()
    w["seqs"] = [n + h for n, h in reqs]
    return w


def prepare(case, seed):
    w = _inputs(case, seed)
    state = {"case": case, **w}
    if own:
        from oscar_amd.kernels import append, chunk, rotary

        if case["kind"] != "chunk":   # a model's rotation, a layer's cache
            state["turn"] = rotary.Rotary(w["table"], adjacent=case["adjacent"], axes=_pair_axes(case))
        if case["kind"] != "rotate":
            state["cache"] = append.PagedCache(*w["caches"])
        if case["kind"] == "chunk":   # a step's request layout, the same for all its layers
            state["step"] = chunk.ChunkStep(w["starts"], w["seqs"], w["table"], case["heads"], state["cache"],
                                            window=case["window"])
    elif case["kind"] != "chunk" and case["axes"]:
        state["pair_axes"] = torch.tensor(_pair_axes(case), device=DEVICE)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the framework
def _run_own(state):
    from oscar_amd.kernels import append, chunk, rotary

    case = state["case"]
    if case["kind"] == "rotate":
        return rotary.rotate(state["q"], state["k"], state["positions"], state["turn"], inverse=case["inverse"])
    if case["kind"] == "append":
        query = append.append_rotated(state["q"], state["k"], state["v"], state["positions"], state["turn"],
                                      state["cache"], state["slots"])
        return [query, *state["caches"]]
    return chunk.chunk_attention(state["q"], state["cache"], state["step"], case["head_dim"] ** -0.5)


# ------------------------------------------------------------------ plain torch, fp32
def _run_plain(state):
    case = state["case"]
    if case["kind"] == "chunk":
        return _plain_chunk(state)
    positions, table, half = state["positions"], state["table"], case["rotary_dim"] // 2
    if positions.ndim == 1:
        rows = table[positions]
        cos, sin = rows[:, None, :half], rows[:, None, half:]
    else:                             # every axis' row, then each pair's own
        pick = state["pair_axes"][None, :, None].expand(positions.shape[1], half, 1)
        rows = table[positions.t().contiguous()]                            # [N, axes, rotary_dim]
        cos = rows[..., :half].transpose(1, 2).gather(2, pick).transpose(1, 2)
        sin = rows[..., half:].transpose(1, 2).gather(2, pick).transpose(1, 2)
    if case["inverse"]:
        sin = -sin
    turned = [_plain_rotate(x, cos, sin, case["adjacent"]) for x in (state["q"], state["k"])]
    if case["kind"] == "rotate":
        return turned
    slots = state["slots"]
    live = slots >= 0
    at = slots[live]
    for cache, x in zip(state["caches"], (turned[1], state["v"])):
        cache[at // case["page"], at % case["page"]] = x[live]
    return [turned[0], *state["caches"]]


def _plain_rotate(x, cos, sin, adjacent):
    half = cos.shape[-1]
    y = x.float()
    if adjacent:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)


def _plain_chunk(state):
    case, q = state["case"], state["q"]
    hq, hk, d, page, window = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "window"))
    group = hq // hk
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for i, (a, b, seq) in enumerate(zip(state["starts"], state["starts"][1:], state["seqs"])):
        pages = state["table"][i, :-(-seq // page)].long()
        keys, values = (c[pages].reshape(-1, hk, d)[:seq].float() for c in state["caches"])
        step = max(1, (1 << 28) // (group * seq))
        for t in range(a, b, step):
            u = min(b, t + step)
            last = torch.arange(seq - b + t, seq - b + u, device=q.device)
            first = max(0, seq - b + t - window + 1) if window else 0
            end = seq - b + u
            at = torch.arange(first, end, device=q.device)
            hidden = at[None, :] > last[:, None]
            if window:
                hidden = hidden | (at[None, :] <= last[:, None] - window)
            hidden = hidden.repeat_interleave(group, 0)
            for h in range(hk):
                rows = q[t:u, h * group:(h + 1) * group].float().reshape(-1, d)
                s = (rows @ keys[first:end, h].t()) * d ** -0.5
                s = s.masked_fill(hidden, -math.inf)
                p = (s - s.amax(-1, keepdim=True)).exp()
                o = (p @ values[first:end, h]) / p.sum(-1, keepdim=True)
                out[t:u, h * group:(h + 1) * group] = o.view(u - t, group, d).to(q.dtype)
    return out


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    w = _inputs(case, seed)
    if case["kind"] == "chunk":
        return _exact_chunk(case, w)
    pairs = case["rotary_dim"] // 2
    axes = _pair_axes(case) or [0] * pairs
    positions = w["positions"].view(-1, case["tokens"])
    index = torch.arange(pairs, device=DEVICE)
    token = positions[torch.tensor(axes, device=DEVICE)].t()                # [N, pairs]
    wave = torch.complex(w["table"][token, index].double(), w["table"][token, index + pairs].double())
    if case["inverse"]:
        wave = wave.conj()
    first, second = (2 * index, 2 * index + 1) if case["adjacent"] else (index, index + pairs)
    turned = []
    for x in (w["q"], w["k"]):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * wave[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        turned.append(y)
    if case["kind"] == "rotate":
        return turned
    out = [turned[0]]
    for cache, x in zip(w["caches"], (turned[1], w["v"].double())):
        rows = cache.double().flatten(0, 1)
        rows = torch.cat((rows, torch.zeros_like(rows[:1])))                # skipped tokens end in the last row
        rows[torch.where(w["slots"] < 0, rows.shape[0] - 1, w["slots"])] = x
        out.append(rows[:-1].view(cache.shape))
    return out


def _exact_chunk(case, w):
    hq, hk, page, window = case["heads"], case["kv_heads"], case["page"], case["window"]
    scale = case["head_dim"] ** -0.5
    out = []
    for (new, history), row in zip(_requests(case), w["table"]):
        slot = torch.arange(new + history, device=DEVICE)
        slot = row[slot // page].long() * page + slot % page
        keys, values = (c.flatten(0, 1)[slot].double().transpose(0, 1).contiguous() for c in w["caches"])
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
