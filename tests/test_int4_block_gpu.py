"""The token block with normed heads, positions and a 4-bit cache against its formula in 64 bits.

The oracle rounds to 8 and to 4 bits where the block does.  A rounding to float16 (2^-11 relative)
before one to 4 bits moves one code in some 400 by a step, a 7th of its group's largest:
2^-6 of the keys and of the values in the mean square, beside the 2^-6.5 of each of the four 8-bit
inputs: within 2^-4.5 of the output together."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, fp8_block, kv_cache
from lesiondiffusion_mlx_b200.rotary import Rotary, grid_positions
from oracle import fp8 as dense
from oracle import kv_int4 as cache_oracle
from oracle import rotary as rotary_oracle
from tests.test_fp8_block_gpu import OracleBlock

pytestmark = pytest.mark.gpu


def close(got, want):
    err = (got.cpu().double() - want).norm() / want.norm()
    assert err <= 2.0 ** -4.5, float(err)


def frequencies(dims):
    pairs = [(10000.0 ** (-2 * i / d), a) for a, d in enumerate(dims) for i in range(d // 2)]
    return [f for f, _ in pairs], [a for _, a in pairs]


class Int4OracleBlock(OracleBlock):
    def __init__(self, w, heads, kv_heads, dims, interleaved):
        super().__init__(w, heads, kv_heads)
        self.turns, self.interleaved = frequencies(dims), interleaved

    def turned(self, x, gamma, positions):
        flat = x.flatten(2) if x.ndim == 4 else x
        y = rotary_oracle.qk_norm_rope(flat, self.dim, gamma, 1e-6, gamma is not None, *self.turns, self.interleaved,
                                       positions)["out"]
        return y.view(x.shape)

    def write(self, state, rows, positions, at):
        k, v = self.keys_values(rows)
        k = self.turned(k, self.w.get("k_norm"), positions)
        batch, tokens = rows.shape[:2]
        for i, new in ((0, k), (1, v)):
            cache_oracle.append(state[i], state[i + 2], new, state[4], [at] * batch, [tokens] * batch)

    def rest(self, n, h, state, lengths, positions, causal):
        q = self.turned(self.dense(n, "to_q"), self.w.get("q_norm"), positions)
        k, v, ks, vs, table = state
        a = cache_oracle.attention(q, cache_oracle.values(k, ks), cache_oracle.values(v, vs), table, lengths,
                                   self.heads // self.kv_heads, self.dim ** -0.5, causal)["out"].flatten(2)
        h, n = dense.rms_norm(self.dense(a, "to_out"), self.w["norm2"], h, 1e-6)
        f = self.dense(n, "ff1", self.w["ff1.bias"], gelu=True)
        return self.dense(f, "ff2", self.w["ff2.bias"], residual=h)


def empty_state(batch, per, kv_heads, dim, page):
    codes = [torch.full((batch * per, kv_heads, page, dim // 2), 0x88, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.zeros(batch * per, kv_heads, dim // 16, page, dtype=torch.uint8) for _ in range(2)]
    return [*codes, *scales, torch.arange(batch * per, dtype=torch.int32).view(batch, per)]


def test_extend_prompt_then_tokens(cuda_device):
    """A prompt, then token by token: positions count on by themselves."""
    heads, kv_heads, dim, page = 4, 2, 32, 16
    w = fp8_block.random_weights(96, 96, heads, kv_heads, dim, 384, seed=5)
    g = torch.Generator().manual_seed(6)
    w |= {n: 1 + 0.2 * torch.randn(dim, generator=g) for n in ("q_norm", "k_norm")}
    block = fp8_block.Fp8TokenBlock(w, heads=heads, kv_heads=kv_heads, rotary=Rotary.build((dim,), device=cuda_device))
    ref = Int4OracleBlock(w, heads, kv_heads, (dim,), False)
    state = block.new_state(2, 40, page=page, bits=4)
    assert isinstance(state.cache, kv_cache.KvCacheInt4)
    want = empty_state(2, 3, kv_heads, dim, page)
    x = torch.randn(2, 30, 96, generator=g).to(torch.float16)
    at = 0
    for tokens in (21, 1, 1, 7):
        part = x[:, at: at + tokens]
        got = block.extend(part.to(cuda_device), state)
        positions = (at + torch.arange(tokens, dtype=torch.int32)).expand(2, -1)[..., None]
        h, n = dense.rms_norm(part, w["norm1"], None, 1e-6)
        ref.write(want, n, positions, at)
        at += tokens
        close(got, ref.rest(n, h, want, [at, at], positions, True))
    assert state.lengths.tolist() == [30, 30] and _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("interleaved", [False, True])
def test_read_over_a_volume_with_its_places(cuda_device, interleaved):
    """A volume's tokens over another's, bound in 4 bits: positions along three axes, no norms of heads."""
    dims, shape = (16, 24, 24), (3, 5, 6)
    w = fp8_block.random_weights(128, 200, 4, 4, 64, 512, seed=3)
    plan = Rotary.build(dims, interleaved=interleaved, device=cuda_device)
    block = fp8_block.Fp8TokenBlock(w, heads=4, kv_heads=4, rotary=plan)
    ref = Int4OracleBlock(w, 4, 4, dims, interleaved)
    g = torch.Generator().manual_seed(4)
    context, x = torch.randn(2, 90, 200, generator=g).to(torch.float16), torch.randn(2, 90, 128, generator=g).to(torch.float16)
    at = grid_positions(*shape, device=cuda_device)
    state = block.bind(context.to(cuda_device), positions=at, bits=4)
    want, places = empty_state(2, 2, 4, 64, 64), at.cpu().expand(2, -1, -1)
    ref.write(want, context, places, 0)
    h, n = dense.rms_norm(x, w["norm1"], None, 1e-6)
    got = block.read(x.to(cuda_device), state, positions=at)
    close(got, ref.rest(n, h, want, [90, 90], places, False))
    assert torch.equal(block.read(x.to(cuda_device), state, positions=at), got)
    assert _lib.device_status(reset=True) == 0


def test_refusals_write_nothing(cuda_device):
    w = fp8_block.random_weights(64, 64, 2, 2, 32, 128)
    with pytest.raises(ValueError, match="come together"):
        fp8_block.Fp8TokenBlock(w | {"q_norm": torch.ones(32)}, heads=2, kv_heads=2)
    block = fp8_block.Fp8TokenBlock(w, heads=2, kv_heads=2)
    with pytest.raises(ValueError, match="4 or 8"):
        block.new_state(1, 10, bits=2)
    x = torch.randn(1, 4, 64, device=cuda_device, dtype=torch.float16)
    at = torch.zeros(1, 4, 2, dtype=torch.int32, device=cuda_device)
    for plan, positions, text in ((None, at, "without a rotary plan"), (Rotary.build((16, 16)), None, "2 axes"),
                                  (Rotary.build((16, 16)), at[:, :3], "positions must be")):
        block = fp8_block.Fp8TokenBlock(w, heads=2, kv_heads=2, rotary=plan)
        state = block.new_state(1, 10, page=16, bits=4)
        for t in state.cache:
            t.fill_(3)
        with pytest.raises(ValueError, match=text):
            block.extend(x, state, positions=positions)
        assert all((t == 3).all() for t in state.cache) and state.written == 0 and state.lengths.tolist() == [0]
