"""A token block on the 8-bit operators: pre-norm attention over an 8-bit cache and a GELU feed-forward.

One block of a token transformer with root-mean-square norms, its dense weights
and its keys and values held in 8 bits (the denoiser's own blocks have layer norms
with a bias and run in f16):

    rows, h = rms_norm_fp8(x, norm1)                  # codes for the projections, h the residual stream
    q = matmul_fp8(rows, to_q);  a = kv_attention(q, cache, ...)
    o = matmul_fp8(quantize_rows(a), to_out)
    rows, h = rms_norm_fp8(o, norm2, residual=h)      # adds the attention's output on the way
    y = matmul_fp8(quantize_rows(matmul_fp8(rows, ff1, gelu)), ff2, residual=h)

``bind`` projects a context into a cache once, ``read`` attends to it at every
step (cross-attention); ``extend`` writes the tokens' own keys and values behind
those of earlier calls and attends causally (a prompt, then token by token).

Run as a command it times both on random weights:
``python -m lesiondiffusion_mlx_b200.fp8_block``.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .fp8 import Fp8Weight, matmul_fp8, pack_weight_fp8, quantize_rows, rms_norm_fp8
from .kv_cache import KvCacheFp8, kv_append, kv_attention

WEIGHTS = ("norm1", "norm2", "to_q", "to_k", "to_v", "to_out", "ff1", "ff2")


@dataclass
class KvState:
    """A cache, the pages of each item and how many of their tokens are written."""

    cache: KvCacheFp8
    table: torch.Tensor
    lengths: torch.Tensor
    room: int     # tokens an item's pages hold
    written: int  # most tokens written to any item, as far as the host knows

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        tokens = int(k.shape[1])
        if self.written + tokens > self.room:
            raise ValueError(f"the cache holds {self.room} tokens per item, {self.written} + {tokens} do not fit")
        kv_append(self.cache, k, v, self.table, self.lengths)
        self.lengths += tokens
        self.written += tokens


class Fp8TokenBlock:
    """Norm, attention and feed-forward with weights packed to 8 bits at construction.

    ``weights`` holds ``norm1``, ``norm2`` ``(C,)``, ``to_q`` ``(heads * d, C)``,
    ``to_k`` / ``to_v`` ``(kv_heads * d, C_context)``, ``to_out`` ``(C, heads *
    d)``, ``ff1`` ``(F, C)``, ``ff2`` ``(C, F)`` and optionally ``ff1.bias`` /
    ``ff2.bias``; activations are float16 or bfloat16 ``(B, L, C)``."""

    def __init__(self, weights: dict[str, torch.Tensor], *, heads: int, kv_heads: int, eps: float = 1e-6,
                 device: torch.device | str = "cuda"):
        missing = [n for n in WEIGHTS if n not in weights]
        if missing:
            raise ValueError(f"weights are missing {missing}")
        width = int(weights["to_q"].shape[0])
        if heads % kv_heads or width % heads or int(weights["to_k"].shape[0]) != width // heads * kv_heads:
            raise ValueError(f"{heads} heads over {kv_heads} do not fit to_q {tuple(weights['to_q'].shape)} and "
                             f"to_k {tuple(weights['to_k'].shape)}")
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, width // heads, eps
        self.device = torch.device(device)

        def vector(name: str) -> torch.Tensor | None:
            w = weights.get(name)
            return None if w is None else w.to(self.device, torch.float32).contiguous()

        def packed(*names: str) -> Fp8Weight:
            return pack_weight_fp8(torch.cat([weights[n] for n in names]).to(self.device))

        self.norm1, self.norm2 = vector("norm1"), vector("norm2")
        self.bias1, self.bias2 = vector("ff1.bias"), vector("ff2.bias")
        self.to_q, self.to_kv, self.to_out = packed("to_q"), packed("to_k", "to_v"), packed("to_out")
        self.ff1, self.ff2 = packed("ff1"), packed("ff2")

    def new_state(self, batch: int, tokens: int, *, page: int = 64) -> KvState:
        """Room for ``tokens`` tokens of each of ``batch`` items, none written."""
        per = -(-tokens // page)
        table = torch.arange(batch * per, dtype=torch.int32, device=self.device).view(batch, per)
        cache = KvCacheFp8.empty(batch * per, self.kv_heads, self.head_dim, page=page, device=self.device)
        return KvState(cache, table, torch.zeros(batch, dtype=torch.int32, device=self.device), per * page, 0)

    def _keys_values(self, rows, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
        kv = matmul_fp8(rows, self.to_kv, out_dtype=dtype)
        width = self.kv_heads * self.head_dim
        return kv[..., :width], kv[..., width:]

    def bind(self, context: torch.Tensor, *, page: int = 64) -> KvState:
        """The keys and values of a ``(B, L, C_context)`` context, projected and written once."""
        state = self.new_state(int(context.shape[0]), int(context.shape[1]), page=page)
        state.append(*self._keys_values(quantize_rows(context), context.dtype))
        return state

    def _rest(self, rows, h: torch.Tensor, state: KvState, causal: bool) -> torch.Tensor:
        q = matmul_fp8(rows, self.to_q, out_dtype=h.dtype)
        a = kv_attention(q, state.cache, state.table, state.lengths, scale=self.head_dim ** -0.5, causal=causal)
        o = matmul_fp8(quantize_rows(a), self.to_out, out_dtype=h.dtype)
        rows, h = rms_norm_fp8(o, self.norm2, residual=h, eps=self.eps)
        f = matmul_fp8(rows, self.ff1, self.bias1, act=_lib.LDB_ACT_GELU, out_dtype=h.dtype)
        return matmul_fp8(quantize_rows(f), self.ff2, self.bias2, residual=h, out_dtype=h.dtype)

    def _check(self, x: torch.Tensor, state: KvState) -> None:
        """Refused here, before anything is written to the state."""
        if x.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"activations must be float16 or bfloat16, got {x.dtype}")
        if x.ndim != 3 or x.shape[0] != state.lengths.shape[0]:
            raise ValueError(f"activations must be ({state.lengths.shape[0]}, L, C), got {tuple(x.shape)}")

    def read(self, x: torch.Tensor, state: KvState) -> torch.Tensor:
        """The block with attention over every token of ``state`` (cross-attention to a bound context)."""
        self._check(x, state)
        rows, h = rms_norm_fp8(x, self.norm1, eps=self.eps)
        return self._rest(rows, h, state, False)

    def extend(self, x: torch.Tensor, state: KvState) -> torch.Tensor:
        """The block with causal self-attention: ``x``'s keys and values are written behind the state's tokens."""
        self._check(x, state)
        rows, h = rms_norm_fp8(x, self.norm1, eps=self.eps)
        state.append(*self._keys_values(rows, x.dtype))
        return self._rest(rows, h, state, True)


def random_weights(channels: int, context: int, heads: int, kv_heads: int, head_dim: int, hidden: int, *,
                   seed: int = 0) -> dict[str, torch.Tensor]:
    """Float32 weights of a block, unit-variance through every layer."""
    g = torch.Generator().manual_seed(seed)

    def dense(n: int, k: int) -> torch.Tensor:
        return torch.randn(n, k, generator=g) * k ** -0.5

    norm1, norm2 = (1 + 0.1 * torch.randn(channels, generator=g) for _ in range(2))
    return {"norm1": norm1, "norm2": norm2, "to_q": dense(heads * head_dim, channels),
            "to_k": dense(kv_heads * head_dim, context), "to_v": dense(kv_heads * head_dim, context),
            "to_out": dense(channels, heads * head_dim), "ff1": dense(hidden, channels), "ff2": dense(channels, hidden),
            "ff1.bias": 0.02 * torch.randn(hidden, generator=g), "ff2.bias": 0.02 * torch.randn(channels, generator=g)}


def main() -> None:
    def timed(name: str, call, reps: int = 50) -> None:
        for _ in range(5):
            call()
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        start.record()
        for _ in range(reps):
            call()
        end.record()
        torch.cuda.synchronize()
        print(f"{name}: {1000 * start.elapsed_time(end) / reps:.1f} us")

    # the 16x20x20 level's tokens over the 77 x 768 text context
    cross = Fp8TokenBlock(random_weights(256, 768, 4, 4, 64, 1024), heads=4, kv_heads=4)
    context = cross.bind(torch.randn(1, 77, 768, device="cuda", dtype=torch.float16))
    x = torch.randn(1, 6400, 256, device="cuda", dtype=torch.float16)
    timed("6400 tokens x 256 channels over 77 context tokens", lambda: cross.read(x, context))

    # one token of 16 sequences behind 2048 earlier ones each
    block = Fp8TokenBlock(random_weights(2048, 2048, 16, 4, 128, 8192), heads=16, kv_heads=4)
    state = block.new_state(16, 2048 + 64)
    block.extend(torch.randn(16, 2048, 2048, device="cuda", dtype=torch.bfloat16), state)
    token = torch.randn(16, 1, 2048, device="cuda", dtype=torch.bfloat16)
    timed("one token of 16 sequences behind 2048", lambda: block.extend(token, state))


if __name__ == "__main__":
    main()
