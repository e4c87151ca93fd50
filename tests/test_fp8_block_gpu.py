"""The 8-bit token block against its formula in 64 bits.

The oracle rounds to 8 bits where the block does.  Between two roundings to 8
bits the block rounds to 16 (2^-11 relative), which moves one code in 2^7 by a
step of 2^-3 at most: 2^-6.5 of a layer's input in the mean square, so the block's four
quantized inputs stay within 2^-5 of the output together."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, fp8_block
from oracle import fp8 as oracle
from oracle import kv_cache as kv_oracle

pytestmark = pytest.mark.gpu


class OracleBlock:
    def __init__(self, w, heads, kv_heads):
        self.w, self.heads, self.kv_heads = w, heads, kv_heads
        self.dim = w["to_q"].shape[0] // heads
        names = {"to_q": ("to_q",), "to_kv": ("to_k", "to_v"), "to_out": ("to_out",), "ff1": ("ff1",), "ff2": ("ff2",)}
        self.p = {n: oracle.dequantize_weight(*oracle.quantize_weight(torch.cat([w[k] for k in keys])))
                  for n, keys in names.items()}

    def dense(self, x, name, bias=None, residual=None, gelu=False):
        lead = x.shape[:-1]
        a = oracle.dequantize_rows(*oracle.quantize_rows(x.reshape(-1, x.shape[-1])))
        r = None if residual is None else residual.reshape(-1, residual.shape[-1])
        return oracle.matmul(a, self.p[name], bias, r, gelu)[0].view(*lead, -1)

    def keys_values(self, rows):
        kv = self.dense(rows, "to_kv").view(*rows.shape[:2], 2, self.kv_heads, self.dim)
        return kv[:, :, 0], kv[:, :, 1]

    def rest(self, n, h, state, causal):
        q = self.dense(n, "to_q")
        k, k_e, v, v_e, table, lengths = state
        a = kv_oracle.attention(q, k, k_e, v, v_e, table, lengths, self.heads // self.kv_heads, self.dim ** -0.5,
                                causal)["out"].flatten(2)
        h, n = oracle.rms_norm(self.dense(a, "to_out"), self.w["norm2"], h, 1e-6)
        f = self.dense(n, "ff1", self.w["ff1.bias"], gelu=True)
        return self.dense(f, "ff2", self.w["ff2.bias"], residual=h)


def close(got, want):
    err = (got.cpu().double() - want).norm() / want.norm()
    assert err <= 2.0 ** -5, float(err)


def empty_state(batch, per, kv_heads, dim, page):
    codes = [torch.zeros(batch * per, kv_heads, page, dim, dtype=torch.float64) for _ in range(2)]
    e = [torch.zeros(batch * per, kv_heads, dtype=torch.int64) for _ in range(2)]
    return codes, e, torch.arange(batch * per, dtype=torch.int32).view(batch, per)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_read_over_a_bound_context(cuda_device, dtype):
    w = fp8_block.random_weights(128, 200, 4, 4, 64, 512, seed=3)
    block, ref = fp8_block.Fp8TokenBlock(w, heads=4, kv_heads=4), OracleBlock(w, 4, 4)
    g = torch.Generator().manual_seed(4)
    context, x = torch.randn(2, 77, 200, generator=g).to(dtype), torch.randn(2, 90, 128, generator=g).to(dtype)
    state = block.bind(context.to(cuda_device))
    codes, e, table = empty_state(2, 2, 4, 64, 64)
    for c, s, new in zip(codes, e, ref.keys_values(context)):
        kv_oracle.append(c, s, new, table, [0, 0], [77, 77])
    h, n = oracle.rms_norm(x, w["norm1"], None, 1e-6)
    want = ref.rest(n, h, (codes[0], e[0], codes[1], e[1], table, [77, 77]), False)
    first = block.read(x.to(cuda_device), state)
    close(first, want)
    assert torch.equal(block.read(x.to(cuda_device), state), first)  # reading changes nothing
    assert _lib.device_status(reset=True) == 0


def test_extend_prompt_then_tokens(cuda_device):
    heads, kv_heads, dim, page = 4, 2, 32, 16
    w = fp8_block.random_weights(96, 96, heads, kv_heads, dim, 384, seed=5)
    block, ref = fp8_block.Fp8TokenBlock(w, heads=heads, kv_heads=kv_heads), OracleBlock(w, heads, kv_heads)
    state = block.new_state(2, 40, page=page)
    codes, e, table = empty_state(2, 3, kv_heads, dim, page)
    x = torch.randn(2, 30, 96, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    at = 0
    for tokens in (21, 1, 1, 7):
        part = x[:, at : at + tokens]
        got = block.extend(part.to(cuda_device), state)
        h, n = oracle.rms_norm(part, w["norm1"], None, 1e-6)
        for c, s, new in zip(codes, e, ref.keys_values(n)):
            kv_oracle.append(c, s, new, table, [at, at], [tokens, tokens])
        at += tokens
        close(got, ref.rest(n, h, (codes[0], e[0], codes[1], e[1], table, [at, at]), True))
    assert state.lengths.tolist() == [30, 30] and state.written == 30
    with pytest.raises(ValueError, match="do not fit"):
        block.extend(torch.zeros(2, 19, 96, device=cuda_device, dtype=torch.bfloat16), state)
    assert _lib.device_status(reset=True) == 0


def test_step_in_a_graph(cuda_device):
    """A denoise step's cross-attention block captured once and replayed on new tokens."""
    w = fp8_block.random_weights(128, 64, 2, 2, 64, 256, seed=7)
    block = fp8_block.Fp8TokenBlock(w, heads=2, kv_heads=2)
    state = block.bind(torch.randn(1, 20, 64, device=cuda_device, dtype=torch.float16))
    x = torch.randn(1, 200, 128, device=cuda_device, dtype=torch.float16)
    block.read(x, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block.read(x, state)
    x.copy_(torch.randn_like(x))
    graph.replay()
    assert torch.equal(out, block.read(x, state))


def test_refusals(cuda_device):
    w = fp8_block.random_weights(64, 64, 2, 2, 32, 128)
    with pytest.raises(ValueError, match="missing"):
        fp8_block.Fp8TokenBlock({k: v for k, v in w.items() if k != "ff2"}, heads=2, kv_heads=2)
    with pytest.raises(ValueError, match="heads"):
        fp8_block.Fp8TokenBlock(w, heads=3, kv_heads=1)
