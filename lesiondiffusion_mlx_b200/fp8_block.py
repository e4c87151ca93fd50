"""A token block on the 8-bit operators: pre-norm attention over an 8-bit cache and a GELU feed-forward.

One block of a token transformer with root-mean-square norms, its dense weights
and its keys and values held in 8 bits (the denoiser's own blocks have layer norms
with a bias and run in f16):

    rows, h = rms_norm_fp8(x, norm1)                  # codes for the projections, h the residual stream
    q, k = qk_norm_rope(matmul_fp8(rows, to_q), ...)  # where the block norms its heads or tokens have positions
    a = kv_attention(q, cache, ...)
    o = matmul_fp8(quantize_rows(a), to_out)
    rows, h = rms_norm_fp8(o, norm2, residual=h)      # adds the attention's output on the way
    y = matmul_fp8(quantize_rows(matmul_fp8(rows, ff1, gelu)), ff2, residual=h)

``bind`` projects a context into a cache once, ``read`` attends to it at every
step (cross-attention); ``extend`` writes the tokens' own keys and values behind
those of earlier calls and attends causally (a prompt, then token by token).
Caches hold 8 bits or 4, and positions run along one axis (a sequence: ``extend`` counts
them by itself) or several (a volume's tokens).

Run as a command it times both on random weights:
``python -m lesiondiffusion_mlx_b200.fp8_block``.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .fp8 import Fp8Weight, matmul_fp8, pack_weight_fp8, quantize_rows, rms_norm_fp8
from .kv_cache import KvCache, KvCacheFp8, KvCacheInt4, kv_append, kv_attention
from .rotary import Rotary, grid_positions, qk_norm_rope

WEIGHTS = ("norm1", "norm2", "to_q", "to_k", "to_v", "to_out", "ff1", "ff2")


@dataclass
class KvState:
    """A cache, the pages of each item and how many of their tokens are written."""

    cache: KvCache
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
    ``ff2.bias`` and the norms of each head's queries and keys, ``q_norm`` and ``k_norm``
    ``(d,)``; activations are float16 or bfloat16 ``(B, L, C)``.  With a
    ``rotary`` plan queries and keys turn by their tokens' positions where a call has them."""

    def __init__(self, weights: dict[str, torch.Tensor], *, heads: int, kv_heads: int, eps: float = 1e-6,
                 rotary: Rotary | None = None, device: torch.device | str = "cuda"):
        missing = [n for n in WEIGHTS if n not in weights]
        if missing:
            raise ValueError(f"weights are missing {missing}")
        width = int(weights["to_q"].shape[0])
        if heads % kv_heads or width % heads or int(weights["to_k"].shape[0]) != width // heads * kv_heads:
            raise ValueError(f"{heads} heads over {kv_heads} do not fit to_q {tuple(weights['to_q'].shape)} and "
                             f"to_k {tuple(weights['to_k'].shape)}")
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, width // heads, eps
        self.device = torch.device(device)
        self.rotary = rotary
        if ("q_norm" in weights) != ("k_norm" in weights):
            raise ValueError("q_norm and k_norm come together")

        def vector(name: str) -> torch.Tensor | None:
            w = weights.get(name)
            return None if w is None else w.to(self.device, torch.float32).contiguous()

        def packed(*names: str) -> Fp8Weight:
            return pack_weight_fp8(torch.cat([weights[n] for n in names]).to(self.device))

        self.norm1, self.norm2 = vector("norm1"), vector("norm2")
        self.bias1, self.bias2 = vector("ff1.bias"), vector("ff2.bias")
        self.q_norm, self.k_norm = vector("q_norm"), vector("k_norm")
        self.to_q, self.to_kv, self.to_out = packed("to_q"), packed("to_k", "to_v"), packed("to_out")
        self.ff1, self.ff2 = packed("ff1"), packed("ff2")

    def new_state(self, batch: int, tokens: int, *, page: int = 64, bits: int = 8) -> KvState:
        """Room for ``tokens`` tokens of each of ``batch`` items in 8 or 4 bits, none written."""
        if bits not in (4, 8):
            raise ValueError(f"caches hold 4 or 8 bits, got {bits}")
        per = -(-tokens // page)
        table = torch.arange(batch * per, dtype=torch.int32, device=self.device).view(batch, per)
        kind = KvCacheInt4 if bits == 4 else KvCacheFp8
        cache = kind.empty(batch * per, self.kv_heads, self.head_dim, page=page, device=self.device)
        return KvState(cache, table, torch.zeros(batch, dtype=torch.int32, device=self.device), per * page, 0)

    def _keys_values(self, rows, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
        kv = matmul_fp8(rows, self.to_kv, out_dtype=dtype)
        width = self.kv_heads * self.head_dim
        return kv[..., :width], kv[..., width:]

    def _queries(self, rows, dtype: torch.dtype) -> torch.Tensor:
        return matmul_fp8(rows, self.to_q, out_dtype=dtype)

    def _turned(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None, *,
                q_norm: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor | None]:
        """Heads normed where the block has norms for them, and turned where there are positions."""
        if positions is not None and self.rotary is None:
            raise ValueError("positions without a rotary plan")
        if q_norm is None and positions is None:
            return q, k
        return qk_norm_rope(q, k, head_dim=self.head_dim, q_gamma=q_norm, k_gamma=self.k_norm, eps=self.eps,
                            norm=q_norm is not None, rotary=None if positions is None else self.rotary,
                            positions=positions)

    def bind(self, context: torch.Tensor, *, positions: torch.Tensor | None = None, page: int = 64,
             bits: int = 8) -> KvState:
        """The keys and values of a ``(B, L, C_context)`` context, projected and written once."""
        state = self.new_state(int(context.shape[0]), int(context.shape[1]), page=page, bits=bits)
        k, v = self._keys_values(quantize_rows(context), context.dtype)
        state.append(self._turned(k, None, positions, q_norm=self.k_norm)[0], v)
        return state

    def _rest(self, q: torch.Tensor, h: torch.Tensor, state: KvState, causal: bool) -> torch.Tensor:
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

    def read(self, x: torch.Tensor, state: KvState, *, positions: torch.Tensor | None = None) -> torch.Tensor:
        """The block with attention over every token of ``state`` (cross-attention to a bound context)."""
        self._check(x, state)
        rows, h = rms_norm_fp8(x, self.norm1, eps=self.eps)
        q, _ = self._turned(self._queries(rows, h.dtype), None, positions, q_norm=self.q_norm)
        return self._rest(q, h, state, False)

    def extend(self, x: torch.Tensor, state: KvState, *, positions: torch.Tensor | None = None) -> torch.Tensor:
        """The block with causal self-attention: ``x``'s keys and values are written behind the state's tokens.

        Positions along one axis count on from the state's tokens where none are given."""
        self._check(x, state)
        if positions is None and self.rotary is not None:
            if self.rotary.axes != 1:
                raise ValueError(f"positions along {self.rotary.axes} axes have to be given")
            positions = state.lengths[:, None]
            if x.shape[1] != 1:
                positions = positions + torch.arange(x.shape[1], dtype=torch.int32, device=x.device)
        rows, h = rms_norm_fp8(x, self.norm1, eps=self.eps)
        k, v = self._keys_values(rows, x.dtype)
        q, k = self._turned(self._queries(rows, h.dtype), k, positions, q_norm=self.q_norm)
        state.append(k, v)
        return self._rest(q, h, state, True)


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

    # the same with normed heads and positions, over a 4-bit cache
    weights = random_weights(2048, 2048, 16, 4, 128, 8192) | {"q_norm": torch.ones(128), "k_norm": torch.ones(128)}
    block = Fp8TokenBlock(weights, heads=16, kv_heads=4, rotary=Rotary.build((128,)))
    state = block.new_state(16, 2048 + 64, bits=4)
    block.extend(torch.randn(16, 2048, 2048, device="cuda", dtype=torch.bfloat16), state)
    timed("with normed heads and positions, in 4 bits", lambda: block.extend(token, state))

    # The 16x20x20 level's tokens over their own, bound in 4 bits with their places in the volume.  (Over a context this
    # short a cache saves memory, not time: the f16 attention over the same tokens takes 88 us of the GPU, this one 117.)
    volume = Fp8TokenBlock(random_weights(256, 256, 4, 4, 64, 1024), heads=4, kv_heads=4,
                           rotary=Rotary.build((16, 24, 24)))
    at = grid_positions(16, 20, 20)
    bound = volume.bind(x, positions=at, bits=4)
    timed("6400 tokens over 6400 of a volume, in 4 bits", lambda: volume.read(x, bound, positions=at))


if __name__ == "__main__":
    main()
