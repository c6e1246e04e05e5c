"""Microscaled 4-bit floating point on the GPU, through fluke_b200.ops, against oracle/fp4.py.

Codes, scales, row scales and what is read back are compared bit for bit, and so are the stream and the
next input of the fused norms (their operations are defined one by one). Products are held to half
a step of the 16-bit type plus the bound of an f32 sum of K products, K * 2^-24 * sum |a b|."""
import numpy as np
import pytest
import torch

from fluke_b200 import ops
from oracle import fp4

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
QUANT = {"mx": ops.quant_mxfp4, "nv": ops.quant_nvfp4}
DEQUANT = {"mx": ops.dequant_mxfp4, "nv": ops.dequant_nvfp4}


def rows(g, m, k, dtype):
    """Normal values with some large channels, a zero block and zero row, signed zeros and values on ties."""
    x = torch.randn(m, k, generator=g)
    x[:, torch.rand(k, generator=g) < 0.02] *= 20
    x[m // 2, :] = 0
    x[0, :32] = torch.tensor([0.25, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0, 7.9, -0.0, 0.0, 0.5, 1e-6, -1e-6] * 2)
    if k > 64:
        x[m - 1, 32:64] *= 1e-5
    return x.to(dtype)


def f64(t):
    return t.cpu().double().numpy()


def check_quantised(got, want, fmt, m, k):
    codes, scales, row = want
    assert np.array_equal(got[0].cpu().numpy(), fp4.pack(codes))
    tiles = got[1].cpu().numpy()
    blocks = k // fp4.BLOCK[fmt]
    assert np.array_equal(fp4.untile_scales(tiles, m, blocks), scales)
    assert not fp4.untile_scales(tiles, m, tiles.shape[1] * 4)[:, blocks:].any()
    if fmt == "nv":
        assert np.array_equal(got[2].cpu().numpy(), row, equal_nan=True)


SHAPES = [(1, 32), (1, 64), (3, 96), (127, 512), (130, 544), (33, 1024), (5, 2048), (200, 4096), (2, 8192), (3, 16384), (700, 160), (1, 4096)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,k", SHAPES)
def test_quantisation_and_reading_back(m, k, fmt, dtype):
    g = torch.Generator().manual_seed(m * 31 + k)
    x = rows(g, m, k, TYPES[dtype])
    want = fp4.quantise(f64(x), fmt)
    got = QUANT[fmt](x.to(DEV))
    check_quantised(got, want, fmt, m, k)
    back = DEQUANT[fmt](*got, dtype=TYPES[dtype]).cpu()
    exact = torch.from_numpy(fp4.values(*want, fmt)).to(torch.float32).to(TYPES[dtype])
    assert torch.equal(back.view(torch.int16), exact.view(torch.int16))


def matrices(g, m, n, k, fmt):
    a = fp4.quantise(f64(rows(g, m, k, torch.bfloat16)), fmt)
    b = fp4.quantise(f64((torch.randn(n, k, generator=g) / k ** 0.5).half()), fmt)
    return a, b


def on_gpu(q, fill=0xFF):
    """Scales of the rows behind the last are NaN codes: nothing may depend on them."""
    out = (torch.from_numpy(fp4.pack(q[0])).to(DEV), torch.from_numpy(fp4.tile_scales(q[1], fill)).to(DEV))
    return out if q[2] is None else out + (torch.from_numpy(q[2]).to(DEV),)


def half_step(want, dtype):
    t = TYPES[dtype]
    return np.abs(want) * torch.finfo(t).eps / 2 + (2.0 ** -25 if dtype == "f16" else 0)


PRODUCTS = [(1, 64, 64), (1, 8, 32), (5, 136, 96), (127, 128, 256), (128, 128, 512), (129, 256, 288), (300, 1536, 512), (1000, 72, 2048), (77, 264, 4128), (2, 4096, 1024),
            (2600, 1032, 544), (2561, 1096, 2080), (10300, 200, 96)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, fmt, dtype):
    g = torch.Generator().manual_seed(m + n + k)
    a, b = matrices(g, m, n, k, fmt)
    va, vb = fp4.values(*a, fmt), fp4.values(*b, fmt)
    want = va @ vb.T
    got = f64((ops.gemm_mxfp4 if fmt == "mx" else ops.gemm_nvfp4)(*on_gpu(a), *on_gpu(b), dtype=TYPES[dtype]))
    tol = half_step(want, dtype) + k * 2.0 ** -24 * (np.abs(va) @ np.abs(vb).T)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_gated_product(m, n, k, fmt, dtype):
    g = torch.Generator().manual_seed(m + n + k + 1)
    a, b = matrices(g, m, n, k, fmt)
    u = matrices(g, 1, n, k, fmt)[1]
    va, vb, vu = (fp4.values(*q, fmt) for q in (a, b, u))
    gate, up = va @ vb.T, va @ vu.T
    silu = gate / (1 + np.exp(-gate))
    want = silu * up
    got = f64((ops.gated_mlp_mxfp4 if fmt == "mx" else ops.gated_mlp_nvfp4)(*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=TYPES[dtype]))
    # silu = h + h tanh(h), h = gate / 2, with a tanh of relative error 2^-11; the derivative of silu is below 1.1
    dg, du = (k * 2.0 ** -24 * (np.abs(va) @ np.abs(w).T) for w in (vb, vu))
    h = np.abs(gate) / 2
    tol = half_step(want, dtype) + np.abs(up) * (h * np.tanh(h) * 2.0 ** -11 + 1.1 * dg + 4 * h * 2.0 ** -24) + np.abs(silu) * du + 1.1 * dg * du
    assert (np.abs(got - want) <= tol * (1 + 1e-3)).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", [None, "mx", "nv"])
@pytest.mark.parametrize("m,k,seqlen", [(1, 32, 0), (3, 96, 1), (130, 512, 0), (77, 544, 10), (40, 1024, 40), (5, 2048, 2), (700, 1024, 100), (9, 4096, 0), (2, 16384, 1)])
def test_norms_around_a_block(m, k, seqlen, fmt, dtype):
    g = torch.Generator().manual_seed(m + k)
    t = TYPES[dtype]
    x, res = rows(g, m, k, t), torch.randn(m, k, generator=g).to(t)
    post, pre = ((1 + 0.1 * torch.randn(k, generator=g)).to(t) for _ in range(2))
    gate = (0.5 * torch.randn(-(-m // seqlen) if seqlen else 1, k, generator=g)).to(t)
    num = lambda v: v.float().numpy()
    round16 = lambda v: torch.from_numpy(v).to(t).float().numpy()
    stream, h = fp4.rmsnorm_block(num(x), num(res), num(post), num(gate), num(pre), 0.75, 1e-5, seqlen, round16)
    got = ops.rmsnorm_block(*(v.to(DEV) for v in (x, res, post, gate, pre)), 0.75, 1e-5, seqlen=seqlen,
                            quant=None if fmt is None else fmt + "fp4")
    assert np.array_equal(num(got[0].cpu()), stream)
    if fmt is None:
        assert np.array_equal(num(got[1].cpu()), round16(h))
    else:
        check_quantised(got[1:], fp4.quantise(h, fmt), fmt, m, k)
