"""The norms around a block with an 8-bit output and a scale per row, bit for bit: their f32 operations are defined one by one."""
import numpy as np
import pytest
import torch

from fluke_b200 import ops
from oracle import fp4

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def codes_of(h, fmt):
    """f32 rows -> (codes as int8 or e4m3 bytes, scales)."""
    f = np.float32
    most = f(127 if fmt == "int8" else 448)
    with np.errstate(invalid="ignore"):
        top = np.abs(h).max(-1, keepdims=True)
    bad = ~np.isfinite(top)
    top = np.maximum(np.where(bad, f(1), top), f(1e-12))
    scale = np.where(bad, f(np.nan), top / most)[:, 0]
    q = np.where(bad, f(0), h) * (most / top)
    if fmt == "int8":
        return np.rint(q).astype(np.int8), scale
    c = fp4.to_e4m3(np.minimum(np.abs(q), 448).astype(np.float64))
    return np.where(bad, 0, c | (np.signbit(q).astype(np.uint8) << 7)).astype(np.uint8), scale


SHAPES = [(1, 32), (1, 4096), (3, 96), (130, 544), (33, 1024), (5, 2048), (200, 4096), (3, 16384), (700, 160), (700, 256), (1500, 512), (700, 768), (1300, 1024), (900, 1536), (700, 2048), (700, 2080)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k", SHAPES)
def test_pre_norm(m, k, dtype, fmt):
    g = torch.Generator().manual_seed(m + k)
    t = lambda *s: torch.randn(*s, generator=g).to(TYPES[dtype])
    x, res, w = t(m, k), t(m, k), 1 + t(k)
    x[:, ::17] *= 20
    if m > 4:
        x[1], res[1] = 0, 0
        x[2, 5], x[3, k - 1] = float("nan"), float("inf")
    num = lambda v: v.float().numpy()
    round16 = lambda v: torch.from_numpy(v).to(TYPES[dtype]).float().numpy()
    stream, h = fp4.rmsnorm_block(num(x), num(res), None, None, num(w), 1.25, 1e-5, 0, round16)
    got = ops.rmsnorm_block(x.to(DEV), res.to(DEV), None, None, w.to(DEV), 1.25, 1e-5, quant=fmt)
    assert len(got) == 3 and got[1].dtype == (torch.int8 if fmt == "int8" else torch.uint8) and got[2].shape == (m,)
    codes, scale = codes_of(h, fmt)
    assert np.array_equal(num(got[0].cpu()), stream, equal_nan=True)
    assert np.array_equal(got[2].cpu().numpy(), scale, equal_nan=True)
    assert np.array_equal(got[1].cpu().numpy(), codes)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("m,k,seqlen", [(2, 512, 1), (300, 512, 100), (1300, 1024, 0), (40, 4096, 7)])
def test_around_a_block_and_in_place(m, k, seqlen, fmt):
    g = torch.Generator().manual_seed(m)
    t = lambda *s: torch.randn(*s, generator=g).half()
    x, res, post, pre = t(m, k), t(m, k), t(k), t(k)
    gate = t(-(-m // seqlen), k) if seqlen else t(k)
    num = lambda v: v.float().numpy()
    round16 = lambda v: torch.from_numpy(v).half().float().numpy()
    stream, h = fp4.rmsnorm_block(num(x), num(res), num(post), num(gate), num(pre), 0.75, 1e-5, seqlen, round16)
    dev = [v.to(DEV) for v in (x, res, post, gate, pre)]
    got = ops.rmsnorm_block(*dev, 0.75, 1e-5, seqlen=seqlen, quant=fmt, residual_out=dev[1])
    codes, scale = codes_of(h, fmt)
    assert got[0].data_ptr() == dev[1].data_ptr() and np.array_equal(num(got[0].cpu()), stream)
    assert np.array_equal(got[1].cpu().numpy(), codes) and np.array_equal(got[2].cpu().numpy(), scale)


def test_feeds_the_8_bit_products():
    g = torch.Generator(device=DEV).manual_seed(1)
    t = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x, res, w = t(500, 512).half(), t(500, 512).half(), (1 + 0.1 * t(512)).half()
    _, q, s = ops.rmsnorm_block(x, res, None, None, w, 1.0, 1e-5, quant="e4m3")
    wq = (t(256, 512) * 8).to(torch.float8_e4m3fn)
    sb = torch.rand(256, generator=g, device=DEV) / 100
    got = ops.gemm_fp8(q, wq.view(torch.uint8), s, sb)
    exact = (q.view(torch.float8_e4m3fn).double() @ wq.double().T) * s.double()[:, None] * sb.double()
    size = (q.view(torch.float8_e4m3fn).double().abs() @ wq.double().abs().T) * s.double()[:, None] * sb.double()
    assert ((got.double() - exact).abs() <= exact.abs() * 2.0 ** -11 + 2.0 ** -25 + 516 * 2.0 ** -24 * size).all()


def test_empty_and_refusals():
    x, w = torch.zeros(0, 64, dtype=torch.float16, device=DEV), torch.ones(64, dtype=torch.float16, device=DEV)
    assert [v.shape for v in ops.rmsnorm_block(x, x, None, None, w, 1.0, 1e-5, quant="int8")] == [(0, 64), (0, 64), (0,)]
    with pytest.raises(ValueError):
        ops.rmsnorm_block(x, x, None, None, w, 1.0, 1e-5, quant="e5m2")
