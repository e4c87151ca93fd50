"""The 8-bit serving path of a token transformer: what its operators cost.

Three operators that run one after another in a block over latent tokens whose
weights and whose key/value cache are held in 8 bits:

* ``norm``: the residual's addition, the root-mean-square norm, and its result
  as e4m3 codes with one power-of-two scale for each row and 128 channels;
* ``matmul``: those codes times a weight of e4m3 codes with one scale for each
  128 x 128 block, with bias, residual and GELU;
* ``append`` / ``attention``: a paged key/value cache of e4m3 codes with one
  scale for each page of tokens and head, its writing, and attention over it.

``run`` computes them in elementary operations in 32 bits, or, with ``own``
set, by this package's entry points.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
BLOCK = 128  # channels per scale of the rows, channels and rows per scale of a weight
FINFO_MAX = 448.0  # the largest e4m3 value
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def listed() -> list[dict]:
    return [
        # a single token of a served sequence: nothing but latency
        {"name": "norm-token", "op": "norm", "rows": 1, "channels": 2048, "dtype": "bfloat16"},
        # the tokens of the UNet's 16x20x20 level (256 channels) before a dense layer
        {"name": "norm-level1", "op": "norm", "rows": 6400, "channels": 256, "dtype": "float16"},
        # the level-0 volume's 51200 tokens (one more: a ragged last tile) of a wide model
        {"name": "norm-wide", "op": "norm", "rows": 51201, "channels": 1000, "dtype": "bfloat16"},
        # a single token through a wide feed-forward layer: the weight is read once, bytes count
        {"name": "matmul-token", "op": "matmul", "rows": 1, "k": 2048, "n": 8192, "dtype": "bfloat16", "bias": False,
         "residual": False, "gelu": False},
        # the 16x20x20 level's feed-forward expansion with GELU
        {"name": "matmul-level1", "op": "matmul", "rows": 6400, "k": 256, "n": 1024, "dtype": "float16", "bias": True,
         "residual": False, "gelu": True},
        # a long batch of tokens through a wide projection that adds the residual
        {"name": "matmul-wide", "op": "matmul", "rows": 8190, "k": 4096, "n": 4096, "dtype": "bfloat16", "bias": False,
         "residual": True, "gelu": False},
        # one generated token for each of 32 sequences of up to 2048 tokens
        {"name": "append-token", "op": "append", "batch": 32, "new": 1, "length": 2048, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bfloat16"},
        # a prompt's keys and values, written behind what the cache already holds
        {"name": "append-prompt", "op": "append", "batch": 4, "new": 2049, "length": 4100, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bfloat16"},
        # one token after a very long sequence: all SMs share one cache
        {"name": "attend-long", "op": "attention", "batch": 1, "queries": 1, "length": 131072, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "causal": True, "dtype": "bfloat16"},
        # one token for each of 48 sequences of all lengths up to 8192
        {"name": "attend-batch", "op": "attention", "batch": 48, "queries": 1, "length": 8192, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "causal": True, "dtype": "bfloat16"},
        # the 16x20x20 level's tokens over the 77-token text context, projected once and read every step
        {"name": "attend-context", "op": "attention", "batch": 1, "queries": 6400, "length": 77, "kv_heads": 4,
         "group": 1, "dim": 64, "page": 64, "causal": False, "dtype": "float16"},
        # a prompt's 2048 tokens over the cache they were just written to
        {"name": "attend-prompt", "op": "attention", "batch": 4, "queries": 2048, "length": 8000, "kv_heads": 8,
         "group": 4, "dim": 128, "page": 64, "causal": True, "dtype": "bfloat16"},
    ]


def _log(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["norm", "matmul", "append", "attention"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "norm":
        channels = _log(rng, 32, 8192)
        channels = channels if rng.random() < 0.3 else max(8, channels // 8 * 8)
        rows = _log(rng, 1, min(51201, 51_000_000 // channels))
        case = {"op": op, "rows": rows, "channels": channels, "dtype": dtype}
    elif op == "matmul":
        k, n = _log(rng, 64, 8192), _log(rng, 16, 8192)
        k, n = (k, n) if rng.random() < 0.3 else (max(16, k // 16 * 16), max(16, n // 16 * 16))
        rows = _log(rng, 1, min(16384, 8190 * 4096 * 4096 // (k * n)))
        case = {"op": op, "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5, "gelu": rng.random() < 0.3}
    elif op == "append":
        batch, heads = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        new = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8196 // batch))
        case = {"op": op, "batch": batch, "new": new, "length": new + rng.randrange(0, 2048), "kv_heads": heads,
                "dim": rng.choice([32, 64, 128]), "page": rng.choice([16, 32, 64, 128]), "dtype": dtype}
    else:
        batch, heads, group = _log(rng, 1, 48), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        group = min(group, 32 // heads)
        length = _log(rng, 1, min(131072, 48 * 8192 * 8 // (batch * heads)))
        queries = 1 if rng.random() < 0.4 else _log(
            rng, 2, max(2, min(8192, 4 * 32 * 2048 * 8000 // (batch * heads * group * length))))
        case = {"op": op, "batch": batch, "queries": queries, "length": length, "kv_heads": heads, "group": group,
                "dim": rng.choice([32, 64, 128]), "page": rng.choice([16, 32, 64, 128]),
                "causal": rng.random() < 0.5, "dtype": dtype}
    return draw(rng) if 3072 in case.values() else case


# --------------------------------------------------------------------- inputs


def _lengths(case: dict) -> list[int]:
    """Tokens in each item's cache: all lengths up to the case's, the last item's in full; an idle
    slot (no token at all) among four or more items that only read."""
    b, top = int(case["batch"]), int(case["length"])
    least = int(case["new"]) if case["op"] == "append" else 1
    lengths = [max(least, top * (i + 1) // b) for i in range(b)]
    if b >= 4 and case["op"] == "attention":
        lengths[b // 2] = 0
    return lengths


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


def _exponents(amax: torch.Tensor) -> torch.Tensor:
    """The least e with amax <= 448 * 2^e (0 for amax = 0): the scale is 2^e."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)
    return torch.where(amax == 0, torch.zeros_like(e), e)


def _to_e8m0(e: torch.Tensor) -> torch.Tensor:
    return (e + 127).to(torch.uint8).view(E8M0)


def _power(e: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return torch.exp2(e.to(dtype))


def _finite_amax(y: torch.Tensor, dim) -> torch.Tensor:
    return torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y)).amax(dim)


def _row_blocks(y: torch.Tensor) -> torch.Tensor:
    rows, k = y.shape
    blocks = -(-k // BLOCK)
    return torch.nn.functional.pad(y, (0, blocks * BLOCK - k)).view(rows, blocks, BLOCK)


def _quantize_rows(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes (rows, k) and e8m0 scales (rows, ceil(k / 128)) of 32-bit rows."""
    rows, k = y.shape
    blocks = _row_blocks(y)
    e = _exponents(_finite_amax(blocks, -1)).clamp(-127, 127)
    codes = (blocks * _power(-e)[..., None]).to(E4M3)
    return codes.view(rows, -1)[:, :k], _to_e8m0(e)


def _padded(t: torch.Tensor, unit: int) -> torch.Tensor:
    """The same rows with a row stride that is a multiple of ``unit`` elements."""
    rows, k = t.shape
    wide = torch.zeros((rows, -(-k // unit) * unit), dtype=torch.uint8, device=t.device)
    wide[:, :k] = t.contiguous().view(torch.uint8)
    return wide.view(t.dtype)[:, :k]


def _quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    blocks = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    e = _exponents(blocks.abs().amax((1, 3)))
    codes = (blocks * _power(-e)[:, None, :, None]).to(E4M3)
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k], _to_e8m0(e)


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _activations(g: torch.Generator, rows: int, k: int) -> torch.Tensor:
    """Unit normal rows in which a few channels run an order of magnitude larger, as residual streams have them."""
    gain = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return _normal(g, rows, k) * gain


def _cache(case: dict, g: torch.Generator) -> dict:
    """A paged cache that holds the items' tokens in pages of a shuffled order, and the table of them."""
    batch, heads, dim, page = (int(case[n]) for n in ("batch", "kv_heads", "dim", "page"))
    lengths = _lengths(case)
    width = max(1, -(-max(lengths) // page))
    pages = batch * width
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).view(batch, width)
    exponents = torch.randint(-9, -6, (2, pages, heads), generator=g, device="cuda")
    bits = _normal(g, 2 * pages * heads * page, dim).mul_(60.0).clamp_(-FINFO_MAX, FINFO_MAX).to(E4M3)
    codes = bits.view(2, pages, heads, page, dim)
    return {"k": codes[0], "v": codes[1], "k_scale": _to_e8m0(exponents[0]), "v_scale": _to_e8m0(exponents[1]),
            "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    s: dict = {"case": case}
    if case["op"] == "norm":
        rows, c = int(case["rows"]), int(case["channels"])
        s |= {"x": _activations(g, rows, c).to(dtype), "residual": (2.0 * _activations(g, rows, c)).to(dtype),
              "gamma": 1 + 0.1 * _normal(g, c)}
    elif case["op"] == "matmul":
        rows, k, n = int(case["rows"]), int(case["k"]), int(case["n"])
        codes, scales = _quantize_rows(_activations(g, rows, k))
        w_codes, w_scales = _quantize_weight(_normal(g, n, k) * k ** -0.5)
        s |= {"codes": _padded(codes, 16), "scales": _padded(scales, 4), "w_codes": _padded(w_codes, 16),
              "w_scales": w_scales, "bias": 0.1 * _normal(g, n) if case["bias"] else None,
              "residual": _normal(g, rows, n).to(dtype) if case["residual"] else None}
    else:
        s |= _cache(case, g)
        batch, width = int(case["batch"]), int(case["kv_heads"]) * int(case["dim"])
        if case["op"] == "append":
            new = int(case["new"])
            s |= {"k_new": _normal(g, batch, new, width).to(dtype), "v_new": _normal(g, batch, new, width).to(dtype),
                  "start": s["lengths"] - new}
        else:
            s["q"] = _normal(g, batch, int(case["queries"]), width * int(case["group"])).to(dtype)
    return s


# ----------------------------------------------------------------- plain forms


def _norm(s: dict) -> dict:
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["gamma"]
    codes, scales = _quantize_rows(y)
    return {"h": h.to(s["x"].dtype), "codes": codes, "scales": scales}


def _gelu(y: torch.Tensor) -> torch.Tensor:
    return 0.5 * y * (1 + torch.erf(y * 2 ** -0.5))


def _matmul(s: dict) -> torch.Tensor:
    case = s["case"]
    k, n = int(case["k"]), int(case["n"])
    a = s["codes"].float() * s["scales"].float().repeat_interleave(BLOCK, 1)[:, :k]
    scale = s["w_scales"].float().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = a @ (s["w_codes"].float() * scale).T
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return (_gelu(y) if case["gelu"] else y).to(getattr(torch, case["dtype"]))


def _append_one(s: dict, codes: torch.Tensor, scales: torch.Tensor, new: torch.Tensor) -> None:
    """Write the new tokens behind the old ones of the pages they touch: a page's scale grows where
    the new values need it, and what the page held is rounded again to the larger scale."""
    case = s["case"]
    heads, dim, page = (int(case[n]) for n in ("kv_heads", "dim", "page"))
    batch, count = new.shape[:2]
    touched = -(-(count + page - 1) // page)  # pages that a run of `count` tokens can touch
    slot = s["start"].long()[:, None] // page + torch.arange(touched, device=new.device)
    at = slot[:, :, None] * page + torch.arange(page, device=new.device) - s["start"].long()[:, None, None]
    fresh, old = (at >= 0) & (at < count), at < 0  # (batch, touched, page)
    there = fresh.any(-1)  # the pages that receive a token
    index = s["table"].long().gather(1, slot.clamp(max=s["table"].shape[1] - 1))
    picked = at.clamp(0, count - 1).reshape(batch, -1, 1).expand(-1, -1, heads * dim)
    values = new.float().gather(1, picked).view(batch, touched, page, heads, dim).transpose(2, 3)
    values = torch.where(fresh[:, :, None, :, None], values, torch.zeros_like(values))
    e = _exponents(_finite_amax(values, (-2, -1))).clamp(-96, 96)  # (batch, touched, heads)
    e_old = scales[index].view(torch.uint8).int() - 127
    e = torch.where(old.any(-1)[..., None], torch.maximum(e, e_old), e)
    kept = codes[index].float() * _power(e_old - e)[..., None, None]
    out = (values * _power(-e)[..., None, None]).to(E4M3).float()
    out = torch.where(fresh[:, :, None, :, None], out, kept)
    out = torch.where((fresh | old)[:, :, None, :, None], out, codes[index].float())
    codes[index[there]] = out[there].to(E4M3)
    scales.view(torch.uint8)[index[there]] = (e[there] + 127).to(torch.uint8)


def _append(s: dict) -> dict:
    _append_one(s, s["k"], s["k_scale"], s["k_new"])
    _append_one(s, s["v"], s["v_scale"], s["v_new"])
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attention(s: dict) -> torch.Tensor:
    case, table = s["case"], s["table"].long()
    heads, group, dim, m = (int(case[n]) for n in ("kv_heads", "group", "dim", "queries"))
    batch, width = table.shape
    keys = width * int(case["page"])

    def rows(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
        x = codes[table].float() * scales[table].float()[..., None, None]  # (batch, width, heads, page, dim)
        return x.transpose(1, 2).reshape(batch, heads, 1, keys, dim)

    q = s["q"].float().view(batch, m, heads, group, dim).permute(0, 2, 3, 1, 4)
    scores = q @ rows(s["k"], s["k_scale"]).transpose(-1, -2) * dim ** -0.5  # (batch, heads, group, m, keys)
    n = s["lengths"].long()[:, None, None]
    key = torch.arange(keys, device=table.device)
    seen = key < n
    if case["causal"]:
        seen = seen & (key <= n - m + torch.arange(m, device=table.device)[:, None])
    seen = seen.expand(batch, m, keys)[:, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = p @ rows(s["v"], s["v_scale"]) / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, m, -1).to(s["q"].dtype)


# ------------------------------------------------------------------------ runs


def _run_own(s: dict):
    from lesiondiffusion_mlx_b200 import _lib, fp8, kv_cache

    case = s["case"]
    if case["op"] == "norm":
        q, h = fp8.rms_norm_fp8(s["x"], s["gamma"], residual=s["residual"], eps=EPS)
        return {"h": h, "codes": q.codes, "scales": q.scales}
    if case["op"] == "matmul":
        return fp8.matmul_fp8(fp8.Fp8Rows(s["codes"], s["scales"]), fp8.Fp8Weight(s["w_codes"], s["w_scales"]),
                              s["bias"], residual=s["residual"],
                              act=_lib.LDB_ACT_GELU if case["gelu"] else _lib.LDB_ACT_NONE,
                              out_dtype=getattr(torch, case["dtype"]))
    cache = kv_cache.KvCacheFp8(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["op"] == "append":
        kv_cache.kv_append(cache, s["k_new"], s["v_new"], s["table"], s["start"])
        return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return kv_cache.kv_attention(s["q"], cache, s["table"], s["lengths"], scale=int(case["dim"]) ** -0.5,
                                 causal=bool(case["causal"]))


def run(s: dict):
    if own:
        return _run_own(s)
    return {"norm": _norm, "matmul": _matmul, "append": _append, "attention": _attention}[s["case"]["op"]](s)


def work(case: dict) -> dict:
    """Each input read once, each output written once; for the cache, the tokens that the call concerns."""
    if case["op"] == "norm":
        rows, c = int(case["rows"]), int(case["channels"])
        # x, residual and h in 16 bits, the codes in 8, a scale for each 128; square, sum, two products, scale and round
        return {"bytes": rows * (7 * c + -(-c // BLOCK)) + 4 * c, "flops": 6 * rows * c}
    if case["op"] == "matmul":
        rows, k, n = int(case["rows"]), int(case["k"]), int(case["n"])
        scales = -(-k // BLOCK) * (rows + -(-n // BLOCK))
        return {"bytes": k * (rows + n) + scales + 2 * rows * n * (2 if case["residual"] else 1)
                + (4 * n if case["bias"] else 0), "flops": 2 * rows * k * n}
    heads, dim, batch = int(case["kv_heads"]), int(case["dim"]), int(case["batch"])
    if case["op"] == "append":
        # 16 bits in, 8 bits out, for keys and values; compare for the maximum, scale and round
        tokens = batch * int(case["new"])
        return {"bytes": 2 * tokens * heads * dim * 3, "flops": 2 * 3 * tokens * heads * dim}
    q = batch * int(case["queries"]) * heads * int(case["group"]) * dim
    # without a causal mask, or for as many keys as any query sees, every cached token is read once
    return {"bytes": 2 * sum(_lengths(case)) * heads * dim + 2 * 2 * q,
            "flops": 4 * _visible(case) * heads * int(case["group"]) * dim}


# --------------------------------------------------------- in 64 bits, from the definitions


def _value(codes: torch.Tensor, scale_bits: torch.Tensor) -> torch.Tensor:
    """code * 2^(bits - 127) in 64 bits; ``scale_bits`` is broadcast against the codes."""
    return codes.to(torch.float64) * torch.exp2(scale_bits.to(torch.float64) - 127)


def _least_exponent(amax: float) -> int:
    """The least e in [-96, 96] with amax <= 448 * 2^e (0 for amax = 0)."""
    return 0 if amax == 0 else max(-96, min(96, math.ceil(math.log2(amax / FINFO_MAX))))


def _exact_append(s: dict, codes: torch.Tensor, scales: torch.Tensor, new: torch.Tensor) -> tuple:
    """Page by page: what the run returns, as 64-bit values."""
    page, (batch, count) = int(s["case"]["page"]), new.shape[:2]
    out, bits = codes.to(torch.float64), scales.view(torch.uint8).to(torch.float64)
    new = new.to(torch.float64).view(batch, count, codes.shape[1], -1).transpose(1, 2)
    for b in range(batch):
        start = int(s["start"][b])
        for slot in range(start // page, (start + count - 1) // page + 1):
            at = int(s["table"][b, slot])
            low, high = max(start, slot * page), min(start + count, slot * page + page)
            part = new[b, :, low - start:high - start]
            held = low - slot * page
            amax = part.abs().amax((1, 2)).tolist()
            e = torch.tensor([_least_exponent(a) for a in amax], dtype=torch.float64, device=new.device)
            if held:
                was = bits[at] - 127
                e = torch.maximum(e, was)
                out[at, :, :held] = (out[at, :, :held] * torch.exp2(was - e)[:, None, None]).to(E4M3).double()
            out[at, :, held:high - slot * page] = (part * torch.exp2(-e)[:, None, None]).to(E4M3).double()
            bits[at] = e + 127
    return out, torch.exp2(bits - 127)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "norm":
        # the codes and scales round what lies next to them apart: no 64-bit value stands for either
        return {"h": s["x"].double() + s["residual"].double(), "codes": None, "scales": None}
    if case["op"] == "matmul":
        k, n = int(case["k"]), int(case["n"])
        kb = torch.arange(k, device="cuda") // BLOCK
        nb = torch.arange(n, device="cuda") // BLOCK
        a = _value(s["codes"], s["scales"].view(torch.uint8)[:, kb])
        y = torch.matmul(a, _value(s["w_codes"], s["w_scales"].view(torch.uint8)[nb][:, kb]).t())
        y = y + (0 if s["bias"] is None else s["bias"].double())
        y = y + (0 if s["residual"] is None else s["residual"].double())
        return y * torch.special.ndtr(y) if case["gelu"] else y
    if case["op"] == "append":
        if int(case["batch"]) * int(case["new"]) > 60_000:
            return None
        k, k_scale = _exact_append(s, s["k"], s["k_scale"], s["k_new"])
        v, v_scale = _exact_append(s, s["v"], s["v_scale"], s["v_new"])
        return {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}
    heads, group, dim, m = (int(case[n]) for n in ("kv_heads", "group", "dim", "queries"))
    out = torch.zeros((int(case["batch"]), m, heads, group, dim), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = s["table"][b].long()
        k, v = (_value(s[x][pages], s[x + "_scale"].view(torch.uint8)[pages][..., None, None]).transpose(0, 1)
                .reshape(heads, -1, dim)[:, :n] for x in ("k", "v"))
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
    return out.view(int(case["batch"]), m, -1)
