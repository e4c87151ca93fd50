"""Positions and a 4-bit key/value cache for token blocks: what their operators cost.

Operators that run one after another in a block over latent or text tokens:

* ``rope``: each head's queries and keys normed (root mean square) and rotated by
  positions of one axis (a sequence) or several (depth, height, width) in one pass;
* ``append``: keys and values rounded to 4 bits as they are written into a paged
  cache (integers -8 .. 7 with one scale for each 16 channels of a token), and what
  was written read back;
* ``read``: cached tokens, in 4 or in 8 bits, read back as rows;
* ``attention``: attention over the 4-bit cache.

``run`` computes them in elementary operations in 32 bits (angles in 64), or, with
``own`` set, by this package's entry points.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
BASE = 10000.0
GROUP = 16  # channels per scale of the 4-bit cache
TOP = 198  # largest scale byte: 1.75 * 2^9
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed() -> list[dict]:
    return [
        # one generated token for each of 32 sequences: nothing but latency
        {"name": "rope-token", "op": "rope", "batch": 32, "tokens": 1, "heads": 16, "kv_heads": 4, "dim": 128,
         "rotate": "128", "interleaved": False, "start": 4000, "dtype": "bfloat16"},
        # the 16x20x20 level's voxels as tokens, positions along depth, height and width
        {"name": "rope-level1", "op": "rope", "batch": 1, "tokens": 6400, "heads": 4, "kv_heads": 4, "dim": 64,
         "rotate": "16+24+24", "interleaved": True, "start": 0, "dtype": "float16"},
        # prompts of a wide model, behind long contexts: a ragged count of tokens, far positions
        {"name": "rope-prompt", "op": "rope", "batch": 4, "tokens": 4097, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotate": "128", "interleaved": False, "start": 131072, "dtype": "bfloat16"},
        # one token of each of 32 sequences, written behind what their pages hold
        {"name": "append-token", "op": "append", "batch": 32, "tokens": 1, "start": 2047, "kv_heads": 4, "dim": 128,
         "page": 64, "dtype": "bfloat16"},
        # prompts' keys and values
        {"name": "append-prompt", "op": "append", "batch": 4, "tokens": 4097, "start": 1000, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bfloat16"},
        # the 77 tokens of a text context, bound in 8 bits for 4 items, as rows again
        {"name": "read-context", "op": "read", "bits": 8, "batch": 4, "length": 77, "kv_heads": 4, "dim": 64,
         "page": 64, "dtype": "float16"},
        # whole sequences of all lengths up to 16384, from 4 bits
        {"name": "read-long", "op": "read", "bits": 4, "batch": 8, "length": 16384, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bfloat16"},
        # one token after a very long sequence: all SMs share one cache
        {"name": "attend-long", "op": "attention", "batch": 1, "queries": 1, "length": 262144, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "causal": True, "dtype": "bfloat16"},
        # one token for each of 32 sequences of all lengths up to 16384, in small pages
        {"name": "attend-batch", "op": "attention", "batch": 32, "queries": 1, "length": 16384, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 32, "causal": True, "dtype": "bfloat16"},
        # the 16x20x20 level's tokens over another volume's and the text context's, bound once
        {"name": "attend-level1", "op": "attention", "batch": 1, "queries": 6400, "length": 6477, "kv_heads": 4,
         "group": 1, "dim": 64, "page": 64, "causal": False, "dtype": "float16"},
        # a prompt's next 1024 tokens over the cache they were just written to
        {"name": "attend-prompt", "op": "attention", "batch": 2, "queries": 1024, "length": 16384, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "causal": True, "dtype": "bfloat16"},
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["rope", "append", "read", "attention", "attention"])
    dtype, dim, page = rng.choice(["float16", "bfloat16"]), rng.choice([32, 64, 128]), rng.choice([16, 32, 64, 128])
    heads = rng.choice([1, 2, 3, 4, 8])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 128])
        group = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 32)
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, max(2, 4 * 4097 * 40 * 128 // (batch * heads * (group + 1) * dim)))
        part = max(16, dim // 32 * 16)
        rotate = rng.choice([f"{dim}", f"{part}", f"{part // 2}+{part // 2}", f"{dim - part}+{part // 2}+{part // 2}"])
        return {"op": op, "batch": batch, "tokens": min(tokens, 51200), "heads": heads * group, "kv_heads": heads,
                "dim": dim, "rotate": rotate, "interleaved": rng.random() < 0.5,
                "start": _log(rng, 1, 1 << 20), "dtype": dtype}
    if op == "append":
        batch = _log(rng, 1, 48)
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, max(2, 4 * 4097 // batch))
        return {"op": op, "batch": batch, "tokens": tokens, "start": rng.randrange(0, 2048), "kv_heads": heads,
                "dim": dim, "page": page, "dtype": dtype}
    if op == "read":
        batch = _log(rng, 1, 32)
        return {"op": op, "bits": rng.choice([4, 4, 8]), "batch": batch, "length": _log(rng, 1, 8 * 16384 // batch),
                "kv_heads": heads, "dim": dim, "page": page, "dtype": dtype}
    batch, group = _log(rng, 1, 48), min(rng.choice([1, 2, 4, 8]), 32 // heads)
    length = _log(rng, 1, min(262144, 32 * 16384 * 8 // (batch * heads)))
    queries = 1 if rng.random() < 0.4 else _log(
        rng, 2, max(2, min(8192, 2 * 32 * 1024 * 16384 // (batch * heads * group * length))))
    return {"op": op, "batch": batch, "queries": queries, "length": length, "kv_heads": heads, "group": group,
            "dim": dim, "page": page, "causal": rng.random() < 0.5, "dtype": dtype}


# --------------------------------------------------------------------- inputs


def _sizes(case: dict, *names: str) -> tuple[int, ...]:
    return tuple(int(case[n]) for n in names)


def _rotated(case: dict) -> list[int]:
    """Channels that turn with each axis' positions."""
    return [int(n) for n in str(case["rotate"]).split("+")]


def _lengths(case: dict) -> list[int]:
    """Tokens in each item's cache: all lengths up to the case's, the last item's in full; an idle
    slot (no token at all) among four or more items that only read."""
    b, top = _sizes(case, "batch", "length")
    lengths = [max(1, top * (i + 1) // b) for i in range(b)]
    if b >= 4:
        lengths[b // 2] = 0
    return lengths


def _starts(case: dict) -> list[int]:
    """Where each item's new tokens go: the case's start in the last item, less before it."""
    b, top = _sizes(case, "batch", "start")
    return [top - (b - 1 - i) * (top // b) for i in range(b)]


def _visible(case: dict) -> int:
    """(query, key) pairs of one head that the mask leaves, over the whole batch."""
    total, m = 0, int(case["queries"])
    for n in _lengths(case):
        if not case["causal"]:
            total += m * n
        else:  # query i sees the keys up to n - m + i
            first = max(0, m - n)  # the first query that sees a key
            seen = m - first
            total += seen * (n - m + first + 1) + seen * (seen - 1) // 2
    return total


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rotary(case: dict) -> dict:
    """Each turning pair's frequency and axis, and the plan that a program keeps of them: turns per
    position, as a fraction of 2^64."""
    frequency, axis = [], []
    for a, d in enumerate(_rotated(case)):
        frequency += [BASE ** (-2 * i / d) for i in range(d // 2)]
        axis += [a] * (d // 2)
    turns = [int(f / (2 * math.pi) * 2 ** 64) for f in frequency]
    return {"frequency": torch.tensor(frequency, dtype=torch.float64, device="cuda"),
            "turns": torch.tensor([t - (1 << 64) * (t >> 63) for t in turns], dtype=torch.int64, device="cuda"),
            "axis": torch.tensor(axis, dtype=torch.int32, device="cuda")}


def _positions(case: dict) -> torch.Tensor:
    """Behind what a sequence holds, or, along several axes, a volume's voxels in order."""
    batch, tokens = _sizes(case, "batch", "tokens")
    axes = len(_rotated(case))
    at = torch.arange(tokens, device="cuda")
    if axes == 1:
        per = (torch.tensor(_starts(case), device="cuda")[:, None] + at)[..., None]
    else:
        side = max(1, round(tokens ** (1 / axes)))
        parts = []
        for _ in range(axes - 1):
            parts.append(at % side)
            at = at // side
        per = torch.stack([*parts, at][::-1], -1).expand(batch, -1, -1)
    return per.to(torch.int32).contiguous()


def _table(case: dict, g: torch.Generator, tokens: int) -> torch.Tensor:
    batch, page = _sizes(case, "batch", "page")
    width = -(-tokens // page)
    return torch.randperm(batch * width, generator=g, device="cuda").to(torch.int32).view(batch, width)


def _cache4(case: dict, g: torch.Generator, pages: int) -> dict:
    """Codes and scales as rounding normal values of about unit size leaves them."""
    heads, page, dim = _sizes(case, "kv_heads", "page", "dim")
    s: dict = {}
    for n in ("k", "v"):
        codes = (_normal(g, pages * heads * page, dim).mul_(3.2).round_().clamp_(-8, 7) + 8).to(torch.uint8)
        s[n] = (codes[:, ::2] | (codes[:, 1::2] << 4)).view(pages, heads, page, dim // 2)
        s[n + "_scale"] = torch.randint(96, 112, (pages, heads, dim // GROUP, page), generator=g, device="cuda",
                                        dtype=torch.uint8)
    return s


def _cache8(case: dict, g: torch.Generator, pages: int) -> dict:
    heads, page, dim = _sizes(case, "kv_heads", "page", "dim")
    s: dict = {}
    for n in ("k", "v"):
        s[n] = _normal(g, pages, heads, page, dim).mul_(60.0).clamp_(-448.0, 448.0).to(E4M3)
        s[n + "_scale"] = torch.randint(118, 121, (pages, heads), generator=g, device="cuda", dtype=torch.uint8).view(E8M0)
    return s


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    s: dict = {"case": case}
    batch = int(case["batch"])
    if case["op"] == "rope":
        tokens, heads, kv_heads, dim = _sizes(case, "tokens", "heads", "kv_heads", "dim")
        # one projection's queries, keys and values; a few channels run larger, as projections have them
        gain = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.03, 8.0, 1.0).repeat(heads + 2 * kv_heads)
        qkv = (_normal(g, batch, tokens, (heads + 2 * kv_heads) * dim) * gain).to(dtype)
        s |= _rotary(case) | {"q": qkv[..., :heads * dim], "k": qkv[..., heads * dim:(heads + kv_heads) * dim],
                              "positions": _positions(case), "q_gamma": 1 + 0.1 * _normal(g, dim),
                              "k_gamma": 1 + 0.1 * _normal(g, dim)}
        return s
    if case["op"] == "append":
        tokens, heads, dim = _sizes(case, "tokens", "kv_heads", "dim")
        starts = _starts(case)
        s["table"] = _table(case, g, max(starts) + tokens)
        s |= _cache4(case, g, s["table"].numel())
        kv = _normal(g, batch, tokens, 2 * heads * dim).to(dtype)
        s |= {"k_new": kv[..., :heads * dim], "v_new": kv[..., heads * dim:],
              "start": torch.tensor(starts, dtype=torch.int32, device="cuda")}
        s["lengths"] = s["start"] + tokens
        return s
    lengths = _lengths(case)
    s["table"] = _table(case, g, max(lengths))
    s |= (_cache8 if case.get("bits") == 8 else _cache4)(case, g, s["table"].numel())
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if case["op"] == "attention":
        queries, heads, group, dim = _sizes(case, "queries", "kv_heads", "group", "dim")
        s["q"] = _normal(g, batch, queries, heads * group * dim).to(dtype)
    return s


# ----------------------------------------------------------------- plain forms


def _turned(x: torch.Tensor, gamma: torch.Tensor, s: dict) -> torch.Tensor:
    dim = int(s["case"]["dim"])
    y = x.float().unflatten(-1, (-1, dim))
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * gamma
    angle = s["positions"].double()[..., s["axis"].long()] * s["frequency"]
    cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
    pairs = s["frequency"].numel()
    turn, rest = y[..., :2 * pairs], y[..., 2 * pairs:]
    if s["case"]["interleaved"]:
        a, b = turn[..., ::2], turn[..., 1::2]
        turn = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turn[..., :pairs], turn[..., pairs:]
        turn = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turn, rest), -1).flatten(-2).to(x.dtype)


def _rope(s: dict) -> dict:
    return {"q": _turned(s["q"], s["q_gamma"], s), "k": _turned(s["k"], s["k_gamma"], s)}


def _scale_values(device: torch.device) -> torch.Tensor:
    """What the 256 scale bytes stand for: five bits of exponent and three of mantissa, a float16's upper ones."""
    return (torch.arange(256, device=device, dtype=torch.int16) << 7).view(torch.float16).float()


def _write(codes: torch.Tensor, scales: torch.Tensor, new: torch.Tensor, page: torch.Tensor, slot: torch.Tensor) -> None:
    """The least scale s with max|x| <= 7.5 s for each 16 channels, and x / s to the nearest integer of -8 .. 7."""
    heads, half = codes.shape[1], codes.shape[3]
    x = new.float().unflatten(-1, (heads, -1, GROUP))
    values = _scale_values(new.device)
    byte = torch.searchsorted(7.5 * values[:TOP + 1], x.abs().amax(-1)).clamp(max=TOP)
    by = values[byte]
    n = torch.round(x / torch.where(by == 0, torch.ones_like(by), by)[..., None]).clamp(-8, 7) + 8
    n = n.to(torch.uint8).unflatten(-1, (-1, 2))
    codes[page, :, slot] = (n[..., 0] | (n[..., 1] << 4)).flatten(-2).view(*page.shape, heads, half)
    scales[page, :, :, slot] = byte.to(torch.uint8)


def _from4(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """(..., dim) values of (..., dim / 2) code bytes and (..., dim / 16) scale bytes."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return (n.unflatten(-1, (-1, GROUP)) * _scale_values(codes.device)[scales.int()][..., None]).flatten(-2)


def _places(s: dict, at: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Page and slot of (batch, n) positions."""
    page = int(s["case"]["page"])
    return s["table"].long().gather(1, (at // page).clamp(max=s["table"].shape[1] - 1)), at % page


def _append(s: dict) -> dict:
    tokens = s["k_new"].shape[1]
    at = s["start"].long()[:, None] + torch.arange(tokens, device=s["start"].device)
    page, slot = _places(s, at)
    _write(s["k"], s["k_scale"], s["k_new"], page, slot)
    _write(s["v"], s["v_scale"], s["v_new"], page, slot)
    return {n: _from4(s[n][page, :, slot], s[n + "_scale"][page, :, :, slot]).flatten(-2).to(s["k_new"].dtype)
            for n in ("k", "v")}


def _read(s: dict) -> dict:
    case = s["case"]
    at = torch.arange(int(case["length"]), device=s["table"].device).expand(int(case["batch"]), -1)
    page, slot = _places(s, at)
    held = (at < s["lengths"].long()[:, None])[..., None]

    def rows(n: str) -> torch.Tensor:
        if case["bits"] == 4:
            x = _from4(s[n][page, :, slot], s[n + "_scale"][page, :, :, slot])
        else:
            x = s[n].view(torch.uint8)[page, :, slot].view(E4M3).float() * s[n + "_scale"].float()[page][..., None]
        x = x.flatten(-2)
        return torch.where(held, x, torch.zeros_like(x)).to(getattr(torch, case["dtype"]))

    return {"k": rows("k"), "v": rows("v")}


def _attention(s: dict) -> torch.Tensor:
    case, table = s["case"], s["table"].long()
    heads, group, dim, m, page = _sizes(case, "kv_heads", "group", "dim", "queries", "page")
    batch, keys = table.shape[0], table.shape[1] * page

    def rows(n: str) -> torch.Tensor:
        x = _from4(s[n][table], s[n + "_scale"][table].transpose(-1, -2))  # (batch, width, heads, page, dim)
        return x.transpose(1, 2).reshape(batch, heads, 1, keys, dim)

    q = s["q"].float().view(batch, m, heads, group, dim).permute(0, 2, 3, 1, 4)
    scores = q @ rows("k").transpose(-1, -2) * dim ** -0.5  # (batch, heads, group, m, keys)
    n = s["lengths"].long()[:, None, None]
    key = torch.arange(keys, device=table.device)
    seen = key < n
    if case["causal"]:
        seen = seen & (key <= n - m + torch.arange(m, device=table.device)[:, None])
    seen = seen.expand(batch, m, keys)[:, None, None]
    scores = scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))))
    total = p.sum(-1, keepdim=True)
    out = p @ rows("v") / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, m, -1).to(s["q"].dtype)


# ------------------------------------------------------------------------ runs


def _run_own(s: dict):
    from lesiondiffusion_mlx_b200 import kv_cache, rotary

    case = s["case"]
    if case["op"] == "rope":
        plan = rotary.Rotary(s["turns"], s["axis"], len(_rotated(case)), bool(case["interleaved"]))
        q, k = rotary.qk_norm_rope(s["q"], s["k"], head_dim=int(case["dim"]), q_gamma=s["q_gamma"],
                                   k_gamma=s["k_gamma"], eps=EPS, rotary=plan, positions=s["positions"])
        return {"q": q, "k": k}
    held = kv_cache.KvCacheFp8 if case.get("bits") == 8 else kv_cache.KvCacheInt4
    cache = held(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["op"] == "attention":
        return kv_cache.kv_attention(s["q"], cache, s["table"], s["lengths"], scale=int(case["dim"]) ** -0.5,
                                     causal=bool(case["causal"]))
    if case["op"] == "append":
        kv_cache.kv_append(cache, s["k_new"], s["v_new"], s["table"], s["start"])
        k, v = kv_cache.kv_read(cache, s["table"], s["lengths"], tokens=int(case["tokens"]), start=s["start"],
                                dtype=s["k_new"].dtype)
    else:
        k, v = kv_cache.kv_read(cache, s["table"], s["lengths"], tokens=int(case["length"]),
                                dtype=getattr(torch, case["dtype"]))
    return {"k": k, "v": v}


def run(s: dict):
    if own:
        return _run_own(s)
    return {"rope": _rope, "append": _append, "read": _read, "attention": _attention}[s["case"]["op"]](s)


def work(case: dict) -> dict:
    """Each input read once, each output written once; for the cache, the tokens that the call concerns."""
    batch, dim, kv_heads = _sizes(case, "batch", "dim", "kv_heads")
    per = dim // 2 + dim // GROUP  # bytes of a token and head in 4 bits
    if case["op"] == "rope":
        rows = batch * int(case["tokens"])
        values = rows * (int(case["heads"]) + kv_heads) * dim
        # square, sum, two factors, and two products and a sum for each turned value
        return {"bytes": 4 * values + 4 * rows * len(_rotated(case)), "flops": 7 * values}
    if case["op"] == "append":
        rows = 2 * batch * int(case["tokens"]) * kv_heads
        # 16 bits in, the cache's bytes out and in again, 16 bits out; maximum, quotient, rounding and its product
        return {"bytes": rows * (4 * dim + 2 * per), "flops": 4 * rows * dim}
    if case["op"] == "read":
        held = 2 * sum(_lengths(case)) * kv_heads
        rows = 2 * batch * int(case["length"]) * kv_heads
        return {"bytes": held * (per if case["bits"] == 4 else dim) + rows * 2 * dim, "flops": held * dim}
    queries, group = _sizes(case, "queries", "group")
    q = batch * queries * kv_heads * group * dim
    return {"bytes": 2 * sum(_lengths(case)) * kv_heads * per + 2 * 2 * q,
            "flops": 4 * _visible(case) * kv_heads * group * dim}


# --------------------------------------------------------- in 64 bits, from the definitions


def _exact_turned(x: torch.Tensor, gamma: torch.Tensor, s: dict) -> torch.Tensor:
    """Each pair as a complex number: unit-size rows times gamma, times e^(i position frequency)."""
    case = s["case"]
    dim, pairs = int(case["dim"]), s["frequency"].numel()
    y = x.to(torch.float64).reshape(*x.shape[:2], -1, dim)
    y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / dim + EPS) * gamma.to(torch.float64)
    first = torch.arange(pairs, device=x.device)
    low, high = (2 * first, 2 * first + 1) if case["interleaved"] else (first, first + pairs)
    angle = torch.stack([s["positions"][..., int(a)].double() * f for a, f in zip(s["axis"].tolist(), s["frequency"])], -1)
    z = torch.complex(y[..., low], y[..., high]) * torch.polar(torch.ones_like(angle), angle)[:, :, None]
    y[..., low], y[..., high] = z.real, z.imag
    return y.reshape(x.shape)


def _exact_rounded(new: torch.Tensor) -> torch.Tensor:
    """Groups of 16 channels to integer multiples of their scale, which has four significant bits."""
    x = new.to(torch.float64).reshape(*new.shape[:-1], -1, GROUP)
    least = x.abs().amax(-1, keepdim=True) / 7.5
    unit = torch.exp2(torch.floor(torch.log2(least.clamp(min=2.0 ** -14))) - 3)
    scale = (torch.ceil(least / unit) * unit).clamp(max=1.75 * 2 ** 9)
    times = torch.where(scale > 0, x / scale.clamp(min=2.0 ** -17), 0.0)
    return (torch.round(times).clamp(-8, 7) * scale).reshape(new.shape)


def _exact_tokens(s: dict, n: str, b: int, length: int) -> torch.Tensor:
    """(heads, length, dim) values of item b's first tokens."""
    pages = s["table"][b].long()
    codes, scales = s[n][pages], s[n + "_scale"][pages]
    if codes.dtype == E4M3:
        x = codes.to(torch.float64) * torch.exp2(scales.view(torch.uint8).to(torch.float64) - 127)[..., None, None]
    else:
        scales = scales.transpose(2, 3).long()
        mantissa, exponent = scales % 8, scales // 8
        by = torch.where(exponent == 0, mantissa * 2.0 ** -17, (8 + mantissa) * torch.exp2(exponent.double() - 18))
        x = torch.empty((*codes.shape[:3], 2 * codes.shape[3]), dtype=torch.float64, device=codes.device)
        x[..., 0::2], x[..., 1::2] = codes % 16, torch.div(codes, 16, rounding_mode="floor")
        x = (x - 8) * by.repeat_interleave(GROUP, -1)
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return {"q": _exact_turned(s["q"], s["q_gamma"], s), "k": _exact_turned(s["k"], s["k_gamma"], s)}
    if case["op"] == "append":
        return {"k": _exact_rounded(s["k_new"]), "v": _exact_rounded(s["v_new"])}
    heads, dim, batch = _sizes(case, "kv_heads", "dim", "batch")
    if case["op"] == "read":
        out = {}
        for n in ("k", "v"):
            out[n] = torch.zeros((batch, int(case["length"]), heads, dim), dtype=torch.float64, device="cuda")
            for b, length in enumerate(_lengths(case)):
                out[n][b, :length] = _exact_tokens(s, n, b, length).transpose(0, 1)
            out[n] = out[n].flatten(-2)
        return out
    m, group = _sizes(case, "queries", "group")
    out = torch.zeros((batch, m, heads, group, dim), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        k, v = (_exact_tokens(s, x, b, n) for x in ("k", "v"))
        q = s["q"][b].double().view(m, heads, group, dim)
        step = max(1, 40_000_000 // (heads * group * n))
        for low in range(0, m, step):
            high = min(m, low + step)
            scores = torch.einsum("mhgd,hnd->mhgn", q[low:high], k) / math.sqrt(dim)
            if case["causal"]:
                last = torch.arange(low, high, device="cuda") + (n - m)
                hidden = torch.arange(n, device="cuda")[None, :] > last[:, None]
                scores.masked_fill_(hidden[:, None, None, :], float("-inf"))
            p = torch.nan_to_num(torch.softmax(scores, -1), nan=0.0)  # a row without keys: zeros
            out[b, low:high] = torch.einsum("mhgn,hnd->mhgd", p, v)
    return out.view(batch, m, -1)
