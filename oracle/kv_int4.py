"""The paged 4-bit key/value cache in 64 bits, token by token, from its definition."""

from __future__ import annotations

import torch

GROUP = 16
SCALES = [m * 2.0 ** -17 for m in range(8)] + [(8 + m) * 2.0 ** (e - 18) for e in range(1, 25) for m in range(8)][:191]
NAN = 255  # scale byte of a group that holds a value that is not finite


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """(pages, heads, page, dim) of code bytes (.., page, dim / 2) and scale bytes (.., dim / 16, page)."""
    table = torch.full((256,), float("nan"), dtype=torch.float64)
    table[: len(SCALES)] = torch.tensor(SCALES, dtype=torch.float64)
    x = torch.stack((codes % 16, codes // 16), -1).flatten(-2).double() - 8
    return x * table[scales.long()].transpose(-1, -2).repeat_interleave(GROUP, -1)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """Codes (16,) and the scale byte of one group of channels."""
    x = x.double()
    if not torch.isfinite(x).all():
        return torch.full((GROUP,), 8, dtype=torch.uint8), NAN
    top = float(x.abs().max())
    byte = next((i for i, s in enumerate(SCALES) if top <= 7.5 * s), len(SCALES) - 1)
    if byte == 0:
        return torch.full((GROUP,), 8, dtype=torch.uint8), 0
    return (torch.round(x / SCALES[byte]).clamp(-8, 7) + 8).to(torch.uint8), byte


def append(codes: torch.Tensor, scales: torch.Tensor, new: torch.Tensor, table: torch.Tensor, start: list[int],
           counts: list[int]) -> None:
    """Write ``new`` (B, L, heads, dim) into code and scale bytes."""
    heads, page = codes.shape[1], codes.shape[2]
    for b, (first, count) in enumerate(zip(start, counts)):
        for i in range(count):
            at, slot = int(table[b, (first + i) // page]), (first + i) % page
            for h in range(heads):
                for n in range(scales.shape[2]):
                    c, byte = quantize(new[b, i, h, GROUP * n: GROUP * (n + 1)])
                    codes[at, h, slot, 8 * n: 8 * (n + 1)] = c[::2] | (c[1::2] << 4)
                    scales[at, h, n, slot] = byte


def rows(x: torch.Tensor, table: torch.Tensor, b: int, n: int) -> torch.Tensor:
    """(heads, n, dim): item b's first tokens of a cache's values (pages, heads, page, dim)."""
    at = table[b, : -(-n // x.shape[2])].long()
    return x[at].transpose(0, 1).flatten(1, 2)[:, :n]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: list[int], group: int,
              scale: float, causal: bool) -> dict:
    """Output (B, L, heads * group, dim) over the cache's values ``k`` and ``v``, and what its error bound is made
    of: the weighted value magnitudes, the largest score magnitude sum, and the largest value times the tokens."""
    heads, dim = k.shape[1], k.shape[3]
    batch, m = q.shape[:2]
    q = q.double().view(batch, m, heads, group, dim)
    out, size, score, peak = (torch.zeros(batch, m, heads, group, d, dtype=torch.float64) for d in (dim, dim, 1, 1))
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        ks, vs = rows(k, table, b, n), rows(v, table, b, n)
        for i in range(m):
            seen = min(n, n - m + i + 1) if causal else n
            if seen <= 0:
                continue
            kk, vv = ks[:, :seen].transpose(1, 2), vs[:, :seen]
            p = torch.softmax(q[b, i] @ kk * scale, -1)  # (heads, group, seen)
            out[b, i], size[b, i] = p @ vv, p @ vv.abs()
            score[b, i] = (q[b, i].abs() @ kk.abs() * abs(scale)).amax(-1, keepdim=True)
            peak[b, i] = vv.abs().amax((1, 2))[:, None, None] * seen
    shape = (batch, m, heads * group, -1)
    return {"out": out.view(shape), "size": size.view(shape), "score": score.view(shape), "peak": peak.view(shape)}
