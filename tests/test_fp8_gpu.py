"""8-bit norm, row quantization and product against their definitions in 64 bits.

Tolerances: quantization of given values is exact (bitwise).  The norm's FP32
statistics lie within d = 2^-18 relative of their 64-bit value (at most 32
sequential and 10 tree additions of squares, a division, a reciprocal square
root and two products, each 2^-24), so a scale may differ only where the block
maximum is within d of a power's edge, and a code is the rounding of a value
within d.  A product accumulates in FP32: 8 * 2^-23 of the terms' magnitudes
(the bound of the convolution tests), and one rounding to the output type."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import _lib, fp8
from oracle import fp8 as oracle

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def exponents(scales: torch.Tensor) -> torch.Tensor:
    return scales.view(torch.uint8).cpu().to(torch.int64) - 127


def values(rows) -> tuple[torch.Tensor, torch.Tensor]:
    return rows.codes.cpu().double().flatten(0, -2), exponents(rows.scales).flatten(0, -2)


def activations(rows: int, k: int, seed: int) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    x[:, ::17] *= 12
    if rows > 2:
        x[1] = 0
    return x


def test_every_call_is_clean(cuda_device):
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 128), (17, 129), (9, 250), (4, 512), (33, 1000), (2, 1032),
                                    (3, 4104), (2, 8192), (2, 10000)])
def test_quantize_rows_is_exact(cuda_device, dtype, rows, k):
    x = activations(rows, k, 3 * k + rows).to(dtype)
    got = fp8.quantize_rows(x.to(cuda_device))
    codes, e = values(got)
    want, want_e = oracle.quantize_rows(x)
    assert torch.equal(e, want_e) and torch.equal(codes, want)


def test_quantize_rows_edges(cuda_device):
    """Infinities and NaN become NaN codes without touching their block's scale; zeros, subnormals
    and the range's ends keep to the definition."""
    x = torch.randn(8, 256, generator=torch.Generator().manual_seed(1))
    x[0, 3], x[1, 5], x[2, 7] = float("inf"), float("-inf"), float("nan")
    x[3, :128] = float("inf")
    x[4] = 0
    x[5] *= 1e-42
    x[6] *= 3e38 / x[6].abs().max()
    x[7, :128] = 448.0
    x[7, 128:] = 448.0 * 1.0000001
    got = fp8.quantize_rows(x.to(cuda_device))
    codes, e = values(got)
    want, want_e = oracle.quantize_rows(x)
    assert torch.equal(e, want_e)
    assert torch.equal(torch.isnan(codes), torch.isnan(want))
    assert torch.equal(codes.nan_to_num(0.0), want.nan_to_num(0.0))


def check_rounding(codes, e, y, d=2.0 ** -18):
    rows, k = y.shape
    blocks = e.shape[1]
    padded = torch.nn.functional.pad(y, (0, blocks * 128 - k)).view(rows, blocks, 128)
    amax = padded.abs().amax(-1)
    low, high = oracle.exponent(amax * (1 - d)), oracle.exponent(amax * (1 + d))
    assert ((e >= low) & (e <= high)).all()
    scale = torch.exp2(e.double()).repeat_interleave(128, 1)[:, :k]
    _, power = torch.frexp(codes)
    power = torch.where(codes == 0, torch.full_like(power, -5), power)
    half = torch.exp2((power - 1).clamp(min=-6).double() - 4)
    assert ((codes * scale - y).abs() <= half * scale * (1 + 2.0 ** -20) + d * y.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,c,residual,gamma", [(1, 8, True, True), (1, 2048, True, True), (70, 256, True, True),
                                                   (9, 300, False, True), (33, 1000, True, False), (5, 1024, True, True),
                                                   (6, 1031, True, True), (3, 4096, False, False), (2, 8200, True, True),
                                                   (4, 1, True, True), (5000, 64, True, True)])
def test_rms_norm_rounds_the_norm(cuda_device, dtype, rows, c, residual, gamma):
    x = activations(rows, c, rows + c).to(dtype)
    r = (2 * activations(rows, c, rows + c + 1)).to(dtype) if residual else None
    g = 1 + 0.1 * torch.randn(c, generator=torch.Generator().manual_seed(c)) if gamma else None
    xd = x.to(cuda_device)
    got, h = fp8.rms_norm_fp8(xd, None if g is None else g.to(cuda_device),
                              residual=None if r is None else r.to(cuda_device), eps=1e-6)
    want_h, y = oracle.rms_norm(x, g, r, 1e-6)
    if residual:
        assert torch.equal(h.cpu(), (x.float() + r.float()).to(dtype))
    else:
        assert h is xd
    check_rounding(*values(got), y)


def test_rms_norm_strides_shapes_and_streams(cuda_device):
    """Channel slices of wider rows, unaligned starts, leading axes, and a call on a side stream."""
    wide = activations(24, 700, 5).to(cuda_device, torch.bfloat16)
    for lo, c in ((0, 640), (8, 640), (3, 333)):
        x = wide[:, lo : lo + c]
        got, h = fp8.rms_norm_fp8(x, None, residual=wide[:, 8 : 8 + c])
        _, y = oracle.rms_norm(x.cpu(), None, wide[:, 8 : 8 + c].cpu(), 1e-6)
        check_rounding(*values(got), y)
        assert torch.equal(h, (x.float() + wide[:, 8 : 8 + c].float()).to(torch.bfloat16))
    x = wide[:, :640].reshape(2, 3, 4, 640)
    got, _ = fp8.rms_norm_fp8(x, None)
    assert got.codes.shape == (2, 3, 4, 640) and got.scales.shape == (2, 3, 4, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, _ = fp8.rms_norm_fp8(x, None)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again.codes.view(torch.uint8), got.codes.view(torch.uint8))


def test_rms_norm_non_finite_rows_stay_by_themselves(cuda_device):
    x = activations(6, 512, 9)
    x[2, 40], x[4, 3] = float("inf"), float("nan")
    got, _ = fp8.rms_norm_fp8(x.to(cuda_device), None)
    codes, e = values(got)
    _, y = oracle.rms_norm(x, None, None, 1e-6)
    clean = [0, 1, 3, 5]
    check_rounding(codes[clean], e[clean], y[clean])
    assert torch.isnan(codes[2, 40]) and (codes[2, 41:] == 0).all() and torch.isnan(codes[4]).all()


def test_empty_rows(cuda_device):
    rows = fp8.quantize_rows(torch.zeros(0, 256, device=cuda_device))
    assert rows.codes.shape == (0, 256)
    w = fp8.pack_weight_fp8(torch.ones(16, 256, device=cuda_device))
    assert fp8.matmul_fp8(rows, w).shape == (0, 16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 257), (300, 1000)])
def test_pack_weight_is_exact(cuda_device, dtype, n, k):
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n)).to(dtype)
    got = fp8.pack_weight_fp8(w.to(cuda_device))
    want, want_e = oracle.quantize_weight(w)
    assert torch.equal(exponents(got.scales), want_e) and torch.equal(got.codes.cpu().double(), want)


def operands(m: int, n: int, k: int, dev, seed: int):
    """Operands with uneven scales, and NaN codes in the padding that no product may read."""
    g = torch.Generator().manual_seed(seed)
    a = activations(m, k, seed) * torch.exp2(torch.randint(-3, 4, (m, 1), generator=g))
    w = torch.randn(n, k, generator=g) * torch.exp2(torch.randint(-2, 3, (n, 1), generator=g)) * k ** -0.5
    rows, weight = fp8.quantize_rows(a.to(dev)), fp8.pack_weight_fp8(w.to(dev))
    for t in (rows.codes, weight.codes):
        if t.shape[1] != t.stride(0):
            full = t.view(torch.uint8).as_strided((t.shape[0], t.stride(0)), (t.stride(0), 1))
            full[:, t.shape[1]:] = 0x7F
    av = oracle.dequantize_rows(*values(rows))
    wv = oracle.dequantize_weight(weight.codes.cpu().double(), exponents(weight.scales))
    return rows, weight, av, wv


def check_product(got, want, size, dtype, slope=1.0):
    err = (got.cpu().double() - want).abs()
    bound = slope * 8 * 2.0 ** -23 * size + UNIT[dtype] * want.abs() * (1 + 2.0 ** -10) + TINY[dtype]
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,bias,residual,gelu", [
    (1, 1, 1, True, True, False), (1, 32, 16, False, False, False), (1, 40, 8192, True, True, True),
    (2, 8192, 300, False, True, False), (7, 24, 129, True, False, False), (16, 520, 2049, True, True, False),
    (127, 96, 640, False, False, True), (128, 128, 128, False, False, False), (129, 224, 256, True, True, False),
    (200, 1000, 1000, True, False, True), (400, 2048, 96, False, True, False), (1030, 456, 520, True, True, False),
    (300, 7000, 512, False, False, False), (2500, 1100, 384, True, False, False)])
def test_matmul(cuda_device, dtype, m, n, k, bias, residual, gelu):
    rows, weight, av, wv = operands(m, n, k, cuda_device, m + n + k)
    g = torch.Generator().manual_seed(1)
    b = torch.randn(n, generator=g) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    got = fp8.matmul_fp8(rows, weight, None if b is None else b.to(cuda_device),
                         residual=None if r is None else r.to(cuda_device),
                         act=_lib.LDB_ACT_GELU if gelu else _lib.LDB_ACT_NONE, out_dtype=dtype)
    want, size = oracle.matmul(av, wv, b, r, gelu)
    assert got.shape == (m, n) and got.dtype == dtype
    # |gelu'| <= 1.13, and erff within 2 units: 2^-22 of |y| <= size, inside the slope's margin
    check_product(got, want, size, dtype, slope=1.5 if gelu else 1.0)
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype,m,n,k,bias,residual,gelu", [
    (torch.float16, 513, 2304, 2048, True, False, True), (torch.bfloat16, 2050, 4100, 1024, False, True, False),
    (torch.float32, 700, 1600, 1500, True, True, False), (torch.float16, 1025, 1001, 2050, False, False, False),
    (torch.bfloat16, 300, 520, 4096, True, True, True)])
def test_matmul_many_rows_over_a_long_k(cuda_device, dtype, m, n, k, bias, residual, gelu):
    """Sizes at which two CTAs share a tile, with ragged last tiles on every side."""
    rows, weight, av, wv = operands(m, n, k, cuda_device, m + n + k)
    g = torch.Generator().manual_seed(1)
    b = torch.randn(n, generator=g) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    args = dict(residual=None if r is None else r.to(cuda_device),
                act=_lib.LDB_ACT_GELU if gelu else _lib.LDB_ACT_NONE, out_dtype=dtype)
    got = fp8.matmul_fp8(rows, weight, None if b is None else b.to(cuda_device), **args)
    want, size = oracle.matmul(av, wv, b, r, gelu)
    check_product(got, want, size, dtype, slope=1.5 if gelu else 1.0)
    assert torch.equal(fp8.matmul_fp8(rows, weight, None if b is None else b.to(cuda_device), **args), got)
    assert _lib.device_status(reset=True) == 0


def test_matmul_leading_axes_strides_and_repeats(cuda_device):
    rows, weight, av, wv = operands(60, 72, 256, cuda_device, 4)
    shaped = fp8.Fp8Rows(rows.codes.view(3, 20, 256), rows.scales.view(torch.uint8).as_strided((3, 20, 2), (80, 4, 1))
                         .view(fp8.SCALES))
    want, size = oracle.matmul(av, wv, None, None, False)
    got = fp8.matmul_fp8(shaped, weight, out_dtype=torch.float32)
    assert got.shape == (3, 20, 72)
    check_product(got.view(60, 72), want, size, torch.float32)
    wide = torch.full((60, 101), 7.0, device=cuda_device, dtype=torch.float16)
    out = wide[:, 5:77]  # an odd start and an odd row stride: narrow accesses
    fp8.matmul_fp8(rows, weight, out=out)
    check_product(out, want, size, torch.float16)
    assert (wide[:, :5] == 7).all() and (wide[:, 77:] == 7).all()
    # K ranges are added in order: the same bits every time
    rows, weight, _, _ = operands(5, 64, 8192, cuda_device, 6)
    first = fp8.matmul_fp8(rows, weight, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(fp8.matmul_fp8(rows, weight, out_dtype=torch.float32), first)


def test_matmul_scale_extremes_and_nan_rows(cuda_device):
    """The smallest row scales times the largest weight scales, and a NaN that stays in its row."""
    a = torch.randn(130, 384, generator=torch.Generator().manual_seed(2))
    a[3] *= 1e-38
    w = torch.randn(48, 384, generator=torch.Generator().manual_seed(3)) * 1e30
    rows, weight = fp8.quantize_rows(a.to(cuda_device)), fp8.pack_weight_fp8(w.to(cuda_device))
    rows.codes.view(torch.uint8)[7, 200] = 0x7F
    got = fp8.matmul_fp8(rows, weight, out_dtype=torch.float32).cpu()
    assert torch.isnan(got[7]).all()
    av = oracle.dequantize_rows(*values(rows))
    wv = oracle.dequantize_weight(weight.codes.cpu().double(), exponents(weight.scales))
    keep = [i for i in range(130) if i != 7]
    want, size = oracle.matmul(av[keep], wv, None, None, False)
    check_product(got[keep], want, size, torch.float32)


def test_matmul_in_a_graph_on_a_side_stream(cuda_device):
    rows, weight, av, wv = operands(300, 512, 512, cuda_device, 11)
    out = torch.empty(300, 512, device=cuda_device, dtype=torch.bfloat16)
    fp8.matmul_fp8(rows, weight, out_dtype=torch.bfloat16, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fp8.matmul_fp8(rows, weight, out_dtype=torch.bfloat16, out=out)
    out.zero_()
    graph.replay()
    want, size = oracle.matmul(av, wv, None, None, False)
    check_product(out, want, size, torch.bfloat16)


def test_refusals(cuda_device):
    x = torch.zeros(4, 64, device=cuda_device, dtype=torch.float16)
    with pytest.raises(ValueError, match="gamma"):
        fp8.rms_norm_fp8(x, torch.ones(63, device=cuda_device))
    with pytest.raises(ValueError, match="residual"):
        fp8.rms_norm_fp8(x, None, residual=x.float())
    with pytest.raises(ValueError, match="unit stride"):
        fp8.quantize_rows(x.t())
    with pytest.raises(_lib.LdbError, match="32768"):
        fp8.quantize_rows(torch.zeros(1, 32769, device=cuda_device))
    rows = fp8.quantize_rows(x)
    weight = fp8.pack_weight_fp8(torch.ones(32, 64, device=cuda_device))
    with pytest.raises(ValueError, match="64 channels"):
        fp8.matmul_fp8(rows, fp8.pack_weight_fp8(torch.ones(32, 80, device=cuda_device)))
    with pytest.raises(ValueError, match="bias"):
        fp8.matmul_fp8(rows, weight, torch.ones(32, device=cuda_device, dtype=torch.float16))
    with pytest.raises(ValueError, match="residual"):
        fp8.matmul_fp8(rows, weight, residual=torch.zeros(4, 32, device=cuda_device))
    with pytest.raises(ValueError, match="out shape"):
        fp8.matmul_fp8(rows, weight, out=torch.zeros(4, 31, device=cuda_device, dtype=torch.float16))
    with pytest.raises(ValueError, match="scales"):
        fp8.matmul_fp8(fp8.Fp8Rows(rows.codes, rows.scales[:3]), weight)
    with pytest.raises(_lib.LdbError, match="16-byte"):
        odd = torch.zeros(4, 200, device=cuda_device, dtype=torch.uint8)[:, 1:65].view(fp8.CODES)
        fp8.matmul_fp8(fp8.Fp8Rows(odd, rows.scales), weight)


def test_rms_norm_reads_gamma_after_its_producer(cuda_device):
    """gamma written by the launch right before: the norm has to wait for it."""
    c = 2048
    g = torch.Generator(device=cuda_device).manual_seed(1)
    x = torch.randn(1, c, device=cuda_device, generator=g)
    rows = fp8.quantize_rows(torch.randn(1, c, device=cuda_device, generator=g))
    for seed in range(20):
        weight = fp8.pack_weight_fp8(torch.randn(c, c, device=cuda_device, generator=g))
        torch.cuda.synchronize()
        gamma = fp8.matmul_fp8(rows, weight, out_dtype=torch.float32)
        got, _ = fp8.rms_norm_fp8(x, gamma[0])
        torch.cuda.synchronize()
        want, _ = fp8.rms_norm_fp8(x, gamma[0])
        assert torch.equal(got.codes.view(torch.uint8), want.codes.view(torch.uint8)), seed
        assert torch.equal(got.scales.view(torch.uint8), want.scales.view(torch.uint8)), seed


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k,residual,gelu", [(1, 33, 130, True, False), (37, 61, 4096, True, True),
                                                 (130, 257, 2500, False, False), (333, 999, 200, True, True),
                                                 (1030, 1027, 2050, True, False), (2051, 1601, 140, False, True)])
def test_matmul_narrow_outputs(cuda_device, dtype, m, n, k, residual, gelu):
    """Outputs and residuals without 16-byte rows, inside wider ones whose other values stay."""
    rows, weight, av, wv = operands(m, n, k, cuda_device, m + n + k)
    g = torch.Generator().manual_seed(2)
    b = torch.randn(n, generator=g)
    r = torch.randn(m, n + 2, generator=g).to(dtype)[:, 1 : n + 1] if residual else None
    wide = torch.full((m + 1, n + 4), 3.0, dtype=dtype, device=cuda_device)
    out = wide[:m, 1 : n + 1]
    wide_r = None
    if residual:
        wide_r = torch.zeros(m, n + 2, dtype=dtype, device=cuda_device)
        wide_r[:, 1 : n + 1] = r.to(cuda_device)
        wide_r = wide_r[:, 1 : n + 1]
    fp8.matmul_fp8(rows, weight, b.to(cuda_device), residual=wide_r, out=out, out_dtype=dtype,
                   act=_lib.LDB_ACT_GELU if gelu else _lib.LDB_ACT_NONE)
    want, size = oracle.matmul(av, wv, b, r, gelu)
    check_product(out, want, size, dtype, slope=1.5 if gelu else 1.0)
    assert (wide[m:] == 3).all() and (wide[:, :1] == 3).all() and (wide[:, n + 1:] == 3).all()
    assert _lib.device_status(reset=True) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,c", [(3, 127), (9, 129), (40, 257), (5, 1023), (6, 2051), (3, 8191), (2, 20003)])
def test_quantize_narrow_rows_is_exact(cuda_device, dtype, rows, c):
    """Rows without 16-byte accesses, with infinities and NaN, inside wider ones whose other values stay."""
    wide = torch.randn(rows, c + 3, generator=torch.Generator().manual_seed(rows + c)) * 2.0 ** 3
    wide[:, 1 + c // 2], wide[rows - 1, c] = float("inf"), float("nan")
    wide = wide.to(dtype)
    x = wide[:, 1 : c + 1]
    got = fp8.quantize_rows(wide.to(cuda_device)[:, 1 : c + 1])
    codes, e = oracle.quantize_rows(x.double())
    have = got.codes.cpu().double()
    assert torch.equal(torch.isnan(have), torch.isnan(codes))
    assert torch.equal(have.nan_to_num(0.0), codes.nan_to_num(0.0))
    assert torch.equal(got.scales.view(torch.uint8).cpu().long() - 127, e.long())
    assert _lib.device_status(reset=True) == 0
