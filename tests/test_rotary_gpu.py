"""Normed and rotated queries and keys against their definition in 64 bits.

Per value, relative to its pair's length: the angle is off by at most 2^-25 of half a
turn (its conversion to FP32) and 2^-33 of one (its lower bits), 2^-23 together, and the
tests' positions times frequencies by 2^-53 of up to 2^20 radians; sine and cosine by 2^-22;
mean and root by (D / 8 + 8) 2^-24; the products by 4 * 2^-24; and it is rounded once."""

from __future__ import annotations

import math

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib
from lesiondiffusion_mlx_b200.rotary import Rotary, grid_positions, qk_norm_rope
from oracle import rotary as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def check(got, ref, head_dim, dtype):
    loose = 2.0 ** -23 + 2.0 ** -22 + (head_dim / 8 + 12) * 2.0 ** -24 + 2.0 ** -33
    bound = loose * ref["size"] + UNIT[dtype] * (ref["out"].abs() + loose * ref["size"]) + TINY[dtype]
    err = (got.cpu().double() - ref["out"]).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


def inputs(batch, tokens, heads, kv_heads, dim, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, k = (3 * torch.randn(batch, tokens, n * dim, generator=g) for n in (heads, kv_heads))
    gammas = [1 + 0.2 * torch.randn(dim, generator=g) for _ in range(2)]
    return q.to(dtype), k.to(dtype), *gammas


def frequencies(dims, base=10000.0):
    pairs = [(base ** (-2 * i / d), a) for a, d in enumerate(dims) for i in range(d // 2)]
    return [f for f, _ in pairs], [a for _, a in pairs]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads,dim,dims,interleaved", [
    (1, 1, 1, 1, 64, (64,), False), (2, 5, 4, 2, 128, (128,), True), (3, 7, 3, 1, 80, (48,), False),
    (1, 33, 5, 5, 32, (8, 4, 4), True), (2, 9, 2, 2, 64, (16, 24, 24), False), (1, 4, 1, 0, 16, (16,), False),
    (1, 3, 9, 3, 256, (256,), False), (2, 3, 1, 2, 96, (10,), True), (1, 2, 7, 2, 112, (32, 0, 64), False),
    (1, 10007, 3, 3, 32, (16,), False), (2, 9001, 1, 1, 64, (64,), True), (7, 3001, 1, 2, 16, (10,), True),
    (3, 6500, 2, 0, 48, (16,), False), (1, 2, 2, 1, 48, (48,), True), (1, 700, 32, 8, 128, (64,), False), (40, 1, 16, 4, 128, (128,), False)])
def test_against_the_definition(cuda_device, dtype, batch, tokens, heads, kv_heads, dim, dims, interleaved):
    q, k, q_gamma, k_gamma = inputs(batch, tokens, heads, max(kv_heads, 1), dim, dtype)
    g = torch.Generator().manual_seed(2)
    at = torch.randint(0, 5000, (batch, tokens, len(dims)), generator=g, dtype=torch.int32)
    plan = Rotary.build(dims, interleaved=interleaved, device=cuda_device)
    args = {"head_dim": dim, "eps": 1e-5, "rotary": plan, "positions": at.to(cuda_device),
            "q_gamma": q_gamma.to(cuda_device), "k_gamma": k_gamma.to(cuda_device)}
    q_got, k_got = qk_norm_rope(q.to(cuda_device), k.to(cuda_device) if kv_heads else None, **args)
    assert q_got.dtype == dtype and q_got.shape == q.shape
    f = frequencies(dims)
    check(q_got, oracle.qk_norm_rope(q, dim, q_gamma, 1e-5, True, *f, interleaved, at), dim, dtype)
    if kv_heads:
        check(k_got, oracle.qk_norm_rope(k, dim, k_gamma, 1e-5, True, *f, interleaved, at), dim, dtype)
    else:
        assert k_got is None
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("position", [0, 1, 131071, 2 ** 24 + 1, 2 ** 31 - 1, -1, -(2 ** 31)])
def test_far_positions_keep_their_angle(cuda_device, position):
    """Against exact rational turns: the position's product with the plan's 64-bit fraction."""
    dim, pairs = 64, 32
    plan = Rotary.build((dim,), device="cpu")
    x = torch.zeros(1, 1, dim)
    x[..., :pairs] = 1.0
    at = torch.tensor([[position]], dtype=torch.int32, device=cuda_device)
    got, _ = qk_norm_rope(x.to(cuda_device), None, head_dim=dim, norm=False, positions=at,
                          rotary=Rotary(plan.turns.to(cuda_device), plan.axis.to(cuda_device), 1, False))
    got = got.cpu().double().view(-1)
    for i, t in enumerate(plan.turns.tolist()):
        part = (t * position) % 2 ** 64 / 2 ** 64
        want = (math.cos(2 * math.pi * part), math.sin(2 * math.pi * part))
        assert abs(got[i] - want[0]) <= 2.0 ** -21 and abs(got[i + pairs] - want[1]) <= 2.0 ** -21


def test_norm_alone_rotation_alone_and_neither(cuda_device):
    dtype, dim = torch.bfloat16, 64
    q, k, q_gamma, k_gamma = inputs(2, 6, 2, 1, dim, dtype)
    at = torch.arange(6, dtype=torch.int32)[None, :, None]  # one row of positions for both items
    plan = Rotary.build((dim,), device=cuda_device)
    f = frequencies((dim,))
    dev = [t.to(cuda_device) for t in (q, k)]
    got = qk_norm_rope(*dev, head_dim=dim, q_gamma=q_gamma.to(cuda_device))
    check(got[0], oracle.qk_norm_rope(q, dim, q_gamma, 1e-6, True, [], [], False, None), dim, dtype)
    check(got[1], oracle.qk_norm_rope(k, dim, None, 1e-6, True, [], [], False, None), dim, dtype)
    got = qk_norm_rope(*dev, head_dim=dim, norm=False, rotary=plan, positions=at.to(cuda_device))
    for x, y in zip(got, (q, k)):
        check(x, oracle.qk_norm_rope(y, dim, None, 0, False, *f, False, at.expand(2, 6, 1)), dim, dtype)
    got = qk_norm_rope(*dev, head_dim=dim, norm=False)
    assert torch.equal(got[0], dev[0]) and torch.equal(got[1], dev[1])


@pytest.mark.parametrize("lo", [0, 3])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_in_place_and_streams(cuda_device, lo, interleaved):
    """Slices of one projection at odd offsets, turned in place on another stream; their neighbours stay."""
    dim, heads, kv_heads, dtype = 32, 3, 1, torch.float16
    wide = torch.randn(2, 5, 5 * dim + 7, generator=torch.Generator().manual_seed(3)).to(dtype)
    q, k = wide[..., lo: lo + 96], wide[..., lo + 96: lo + 128]
    at = torch.randint(0, 100, (2, 5), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    f = frequencies((16,))
    want = [oracle.qk_norm_rope(t, dim, None, 1e-6, True, *f, interleaved, at[..., None]) for t in (q, k)]
    dev, plan = wide.to(cuda_device), Rotary.build((16,), interleaved=interleaved, device=cuda_device)
    views = dev[..., lo: lo + 96], dev[..., lo + 96: lo + 128]
    fat = torch.zeros(2, 5, 9, dtype=torch.int32, device=cuda_device)
    fat[..., 4] = at.to(cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qk_norm_rope(*views, head_dim=dim, rotary=plan, positions=fat[..., 4], q_out=views[0], k_out=views[1])
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(views, want):
        check(x, y, dim, dtype)
    rest = torch.ones(wide.shape[2], dtype=torch.bool)
    rest[lo: lo + 128] = False
    assert torch.equal(dev.cpu()[..., rest], wide[..., rest])


def test_what_does_not_turn_is_not_touched_by_what_is_not_finite(cuda_device):
    """Without the norm an infinity stays in its own pair."""
    for interleaved in (False, True):
        x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(5)).to(torch.float16)
        x[0, 0, 10], x[0, 1, 45] = float("inf"), float("nan")
        plan = Rotary.build((32 if not interleaved else 22,), interleaved=interleaved, device=cuda_device)
        at = torch.full((1, 2), 7, dtype=torch.int32, device=cuda_device)
        got, _ = qk_norm_rope(x.to(cuda_device), None, head_dim=64, norm=False, rotary=plan, positions=at)
        bad = (~torch.isfinite(got.cpu())).nonzero().tolist()
        pair = [10, 11] if interleaved else [10, 26]
        assert bad == [[0, 0, c] for c in pair] + [[0, 1, 45]]


def test_captured_and_replayed_with_new_positions(cuda_device):
    dim, dtype = 64, torch.bfloat16
    q, k, q_gamma, _ = inputs(2, 1, 4, 2, dim, dtype)
    plan = Rotary.build((dim,), device=cuda_device)
    dev = [t.to(cuda_device) for t in (q, k)]
    at = torch.zeros(2, 1, dtype=torch.int32, device=cuda_device)
    gamma = q_gamma.to(cuda_device)
    call = lambda: qk_norm_rope(*dev, head_dim=dim, q_gamma=gamma, rotary=plan, positions=at)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in (3, 90000):
        at.fill_(step)
        graph.replay()
        torch.cuda.synchronize()
        pos = torch.full((2, 1, 1), step, dtype=torch.int32)
        check(out[0], oracle.qk_norm_rope(q, dim, q_gamma, 1e-6, True, *frequencies((dim,)), False, pos), dim, dtype)
        check(out[1], oracle.qk_norm_rope(k, dim, None, 1e-6, True, *frequencies((dim,)), False, pos), dim, dtype)


def test_empty_batches_and_volumes(cuda_device):
    plan = Rotary.build((8, 4, 4), device=cuda_device)
    at = grid_positions(2, 3, 4, device=cuda_device)
    assert at.shape == (1, 24, 3) and at[0, 23].tolist() == [1, 2, 3] and at[0, 5].tolist() == [0, 1, 1]
    for batch, tokens in ((0, 24), (2, 0)):
        x = torch.zeros(batch, tokens, 32, device=cuda_device, dtype=torch.float16)
        before = _lib.launch_count()
        q, _ = qk_norm_rope(x, None, head_dim=32, rotary=plan, positions=at[:, :tokens])
        assert q.shape == x.shape and _lib.launch_count() == before


def test_refusals(cuda_device):
    q = torch.zeros(1, 4, 64, device=cuda_device, dtype=torch.float16)
    plan = Rotary.build((32,), device=cuda_device)
    at = torch.zeros(1, 4, dtype=torch.int32, device=cuda_device)
    for args, text in (({"head_dim": 24}, "multiple of 16"), ({"head_dim": 48}, "heads of 48"),
                       ({"head_dim": 32, "rotary": plan}, "positions must be int32"),
                       ({"head_dim": 32, "rotary": plan, "positions": at.long()}, "positions must be int32"),
                       ({"head_dim": 32, "rotary": plan, "positions": at[:, :3]}, "positions must be"),
                       ({"head_dim": 16, "rotary": plan, "positions": at}, "16 pairs"),
                       ({"head_dim": 32, "positions": at}, "without a plan"),
                       ({"head_dim": 32, "q_gamma": torch.ones(64, device=cuda_device)}, "q_gamma"),
                       ({"head_dim": 32, "q_out": q[:, :2]}, "q_out"), ({"head_dim": 32, "k_out": q}, "without k")):
        with pytest.raises(ValueError, match=text):
            qk_norm_rope(q, None, **args)
    with pytest.raises(ValueError, match="k must be"):
        qk_norm_rope(q, q.float(), head_dim=32)
    with pytest.raises(_lib.LdbError, match="item stride"):
        x = q.expand(2, 4, 64)
        qk_norm_rope(x, None, head_dim=32, q_out=x)
