"""The paged 8-bit key/value cache in 64 bits, token by token, from its definition."""

from __future__ import annotations

import torch

from .fp8 import exponent, to_e4m3


def append(codes: torch.Tensor, e: torch.Tensor, new: torch.Tensor, table: torch.Tensor, start: list[int],
           counts: list[int]) -> None:
    """Write ``new`` (B, L, heads, dim) into code values (pages, heads, page, dim) and exponents (pages, heads)."""
    heads, page = codes.shape[1], codes.shape[2]
    for b, (first, count) in enumerate(zip(start, counts)):
        for slot in range(first // page, (first + count - 1) // page + 1 if count else 0):
            low, high = max(first, slot * page), min(first + count, (slot + 1) * page)
            at, held = int(table[b, slot]), low - slot * page
            for h in range(heads):
                x = new[b, low - first : high - first, h].double()
                amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).max()
                need = int(exponent(amax).clamp(-96, 96))
                if held:
                    old = int(e[at, h])
                    need = old if amax == 0 else max(need, old)
                    codes[at, h, :held] = to_e4m3(codes[at, h, :held] * 2.0 ** (old - need))
                codes[at, h, held : high - slot * page] = to_e4m3(x * 2.0 ** -need)
                e[at, h] = need


def attention(q: torch.Tensor, k: torch.Tensor, k_e: torch.Tensor, v: torch.Tensor, v_e: torch.Tensor,
              table: torch.Tensor, lengths: list[int], group: int, scale: float, causal: bool) -> dict:
    """Output (B, L, heads * group, dim), and what its error bound is made of: the weighted value
    magnitudes, the largest score magnitude sum, and the largest weighted scale."""
    heads, page, dim = k.shape[1:]
    batch, m = q.shape[:2]
    q = q.double().view(batch, m, heads, group, dim)
    out, size, score, peak = (torch.zeros(batch, m, heads, group, d, dtype=torch.float64) for d in (dim, dim, 1, 1))
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        at = table[b, : -(-n // page)].long()

        def rows(codes, e):
            x = codes[at] * torch.exp2(e[at].double())[..., None, None]
            return x.transpose(0, 1).reshape(heads, -1, dim)[:, :n]

        ks, vs = rows(k, k_e), rows(v, v_e)
        ve = torch.exp2(v_e[at].double()).T.repeat_interleave(page, 1)[:, :n]
        for h in range(heads):
            for i in range(m):
                seen = min(n, n - m + i + 1) if causal else n
                if seen <= 0:
                    continue
                s = q[b, i, h] @ ks[h, :seen].T * scale
                p = torch.softmax(s, -1)
                out[b, i, h] = p @ vs[h, :seen]
                size[b, i, h] = p @ vs[h, :seen].abs()
                score[b, i, h] = (q[b, i, h].abs() @ ks[h, :seen].abs().T * scale).amax(-1, keepdim=True)
                peak[b, i, h] = (p * ve[h, :seen]).amax(-1, keepdim=True) * seen
    shape = (batch, m, heads * group, -1)
    return {"out": out.view(shape), "size": size.view(shape), "score": score.view(shape), "peak": peak.view(shape)}
