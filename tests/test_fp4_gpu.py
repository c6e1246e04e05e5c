"""Microscaled 4-bit floating point on the GPU, through fluke_b200.ops, against oracle/fp4.py.

Codes, scales, row scales and what is read back are compared bit for bit, and so are the stream and the
next input of the fused norms (their operations are defined one by one). Products are held to half
a step of the 16-bit type plus the bound of an f32 sum of K products, K * 2^-24 * sum |a b|."""
import ctypes

import numpy as np
import pytest
import torch

from fluke_b200 import lib as L, ops
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


# ---- K between the forms, and what no size reaches on its own ---------------------------------

@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,n,k", [(2600, 1032, 1024), (2600, 1032, 768), (2600, 2056, 512), (16, 2048, 8192), (33, 520, 4096), (65, 136, 8192), (64, 264, 2080), (300, 4096, 32)])
def test_products_of_every_form(m, n, k, fmt):
    """Resident weights of two to four stages, a change of columns inside a pair's run, K split over up to eight CTAs of 1 to 64 rows."""
    g = torch.Generator().manual_seed(m * 3 + n + k)
    a, b = matrices(g, m, n, k, fmt)
    u = matrices(g, 1, n, k, fmt)[1]
    va, vb, vu = (fp4.values(*q, fmt) for q in (a, b, u))
    bound = lambda w: k * 2.0 ** -24 * (np.abs(va) @ np.abs(w).T)
    want, up = va @ vb.T, va @ vu.T
    got = f64((ops.gemm_mxfp4 if fmt == "mx" else ops.gemm_nvfp4)(*on_gpu(a), *on_gpu(b), dtype=torch.bfloat16))
    assert (np.abs(got - want) <= half_step(want, "bf16") + bound(vb)).all()
    silu, h = want / (1 + np.exp(-want)), np.abs(want) / 2
    got = f64((ops.gated_mlp_mxfp4 if fmt == "mx" else ops.gated_mlp_nvfp4)(*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=torch.bfloat16))
    tol = half_step(silu * up, "bf16") + np.abs(up) * (h * np.tanh(h) * 2.0 ** -11 + 1.1 * bound(vb) + 4 * h * 2.0 ** -24) + np.abs(silu) * bound(vu) + 1.1 * bound(vb) * bound(vu)
    assert (np.abs(got - silu * up) <= tol * (1 + 1e-3)).all()


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def small(m, n, k, fmt, dtype=torch.float16, seed=0):
    """(a, b, up) of random rows, quantised on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = QUANT[fmt]
    return [q(torch.randn(r, k, generator=g, device=DEV).to(dtype)) for r in (m, n, n)]


GEMM = {"mx": ops.gemm_mxfp4, "nv": ops.gemm_nvfp4}
GATED = {"mx": ops.gated_mlp_mxfp4, "nv": ops.gated_mlp_nvfp4}


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,n,k", [(3, 256, 2048), (300, 512, 512), (3000, 2048, 512), (3000, 2048, 1088)])
def test_products_give_the_same_bits_every_time(m, n, k, fmt):
    a, b, u = small(m, n, k, fmt)
    for call in (lambda: GEMM[fmt](*a, *b), lambda: GATED[fmt](*a, *b, *u)):
        first = bits(call())
        assert all(torch.equal(first, bits(call())) for _ in range(5))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_blocks_and_rows_without_a_value(fmt):
    """An infinity or a NaN: its block (mx) or its row (nv) reads back as NaN, products of the row are NaN, other rows are what they were."""
    for dtype in (torch.float16, torch.bfloat16):
        x = torch.randn(70, 160, generator=torch.Generator().manual_seed(5)).to(dtype)
        x[3, 40], x[60, 0], x[69, 159] = float("nan"), float("inf"), float("-inf")
        want = fp4.quantise(f64(x), fmt)
        got = QUANT[fmt](x.to(DEV))
        check_quantised(got, want, fmt, 70, 160)
        back = DEQUANT[fmt](*got, dtype=dtype).cpu()
        value = fp4.values(*want, fmt)
        assert np.array_equal(np.isnan(back.double().numpy()), np.isnan(value))
        w = QUANT[fmt](torch.randn(64, 160, generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV))
        for out in (GEMM[fmt](*got, *w, dtype=dtype), GATED[fmt](*got, *w, *w, dtype=dtype)):
            bad = torch.isnan(out).cpu()
            assert bad[[3, 60, 69]].all() and not bad[[r for r in range(70) if r not in (3, 60, 69)]].any()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-20, 1e20, 1e30, 1e37])
def test_bf16_of_every_magnitude(fmt, scale):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(9, 96, generator=g) * scale).clamp(-3e38, 3e38).bfloat16()
    check_quantised(QUANT[fmt](x.to(DEV)), fp4.quantise(f64(x), fmt), fmt, 9, 96)
    num = lambda v: v.float().numpy()
    round16 = lambda v: torch.from_numpy(v).bfloat16().float().numpy()
    w = torch.ones(96).bfloat16()
    stream, h = fp4.rmsnorm_block(num(x), num(x), num(w), None, num(w), 0.5, 0.0, 0, round16)
    got = ops.rmsnorm_block(x.to(DEV), x.to(DEV), w.to(DEV), None, w.to(DEV), 0.5, 0.0)
    assert np.array_equal(num(got[0].cpu()), stream) and np.array_equal(num(got[1].cpu()), round16(h))


def test_norms_of_rows_that_have_none():
    """A zero row with eps = 0 (0 * inf), a row with an infinity, a row with a NaN: what the formula gives."""
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(1)).half()
    x[1], x[2, 7], x[3, 9] = 0, float("inf"), float("nan")
    w, res = torch.ones(64).half(), torch.zeros(4, 64).half()
    num = lambda v: v.float().numpy()
    round16 = lambda v: torch.from_numpy(v).half().float().numpy()
    stream, h = fp4.rmsnorm_block(num(x), num(res), num(w), None, num(w), 1.0, 0.0, 0, round16)
    got = ops.rmsnorm_block(x.to(DEV), res.to(DEV), w.to(DEV), None, w.to(DEV), 1.0, 0.0)
    assert np.array_equal(num(got[0].cpu()), stream, equal_nan=True) and np.array_equal(num(got[1].cpu()), round16(h), equal_nan=True)
    for fmt in ("mx", "nv"):
        got = ops.rmsnorm_block(x.to(DEV), res.to(DEV), w.to(DEV), None, w.to(DEV), 1.0, 0.0, quant=fmt + "fp4")
        check_quantised(got[1:], fp4.quantise(h, fmt), fmt, 4, 64)


@pytest.mark.parametrize("post,gate,pre", [(False, False, True), (True, False, False), (False, True, False), (True, True, False), (False, True, True)])
@pytest.mark.parametrize("m,k", [(5, 64), (300, 512), (40, 4096)])
def test_norms_without_one_of_their_parts(m, k, post, gate, pre):
    g = torch.Generator().manual_seed(m)
    t = lambda *s: torch.randn(*s, generator=g).half()
    x, res = t(m, k), t(m, k)
    post, gate, pre = (t(k) if on else None for on in (post, gate, pre))
    num = lambda v: None if v is None else v.float().numpy()
    round16 = lambda v: torch.from_numpy(v).half().float().numpy()
    stream, h = fp4.rmsnorm_block(num(x), num(res), num(post), num(gate), num(pre), 1.5, 1e-6, 0, round16)
    dev = lambda v: None if v is None else v.to(DEV)
    got = ops.rmsnorm_block(*(dev(v) for v in (x, res, post, gate, pre)), 1.5, 1e-6)
    assert len(got) == (2 if pre is not None else 1)
    assert np.array_equal(num(got[0].cpu()), stream)
    if pre is not None:
        assert np.array_equal(num(got[1].cpu()), round16(h))


@pytest.mark.parametrize("quant", [None, "mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,k", [(7, 1024), (1300, 512)])
def test_norms_in_place_on_the_stream(m, k, quant):
    g = torch.Generator(device=DEV).manual_seed(m)
    t = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()
    x, res, w, gate = t(m, k), t(m, k), t(k), t(-(-m // 100), k)
    want = ops.rmsnorm_block(x, res, w, gate, w, 0.5, 1e-5, seqlen=100, quant=quant)
    got = ops.rmsnorm_block(x, res, w, gate, w, 0.5, 1e-5, seqlen=100, quant=quant, residual_out=res)
    assert got[0].data_ptr() == res.data_ptr()
    same = lambda a, b: torch.equal(bits(a), bits(b)) if a.dim() != 3 else torch.equal(*(torch.from_numpy(fp4.untile_scales(v.cpu().numpy(), m, k // 32)) for v in (a, b)))
    assert all(same(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("m,k", [(7, 1024), (1300, 512), (1300, 2080)])
def test_norms_in_place_of_the_input(flib, m, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    t = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
    x, res, w = t(m, k), t(m, k), t(k)
    want = ops.rmsnorm_block(x, res, w, None, w, 0.5, 1e-5)
    a = x.clone()
    got = ops.rmsnorm_block(a, res, w, None, w, 0.5, 1e-5, residual_out=a)
    assert got[0].data_ptr() == a.data_ptr() and all(torch.equal(bits(u), bits(v)) for u, v in zip(want, got))
    a, r = x.clone(), res.clone()   # the stream in the place of the residual, the next input in that of x
    torch.cuda.synchronize()
    b = L.fluke_rmsnorm_block_t(m, k, 0, 0, a.data_ptr(), r.data_ptr(), w.data_ptr(), 0, w.data_ptr(), 0.5, 1e-5, r.data_ptr(), 0, a.data_ptr(), 0, 0)
    assert flib.fluke_rmsnorm_block_gpu(ctypes.byref(b)) == 0
    torch.cuda.synchronize()
    assert torch.equal(bits(r), bits(want[0])) and torch.equal(bits(a), bits(want[1]))
    with pytest.raises(RuntimeError):
        rows_ = torch.zeros(m + 1, k, dtype=torch.float16, device=DEV)
        ops.rmsnorm_block(x, rows_[1:], w, None, w, 0.5, 1e-5, residual_out=rows_[:-1])


def test_nothing_is_written_behind_the_rows(flib):
    """Guard bytes behind every output, and scales of rows behind the last, through the C entry points."""
    m, n, k = 37, 72, 96
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    p = lambda t: t.data_ptr()
    guard = lambda size: torch.full((size + 256,), 0xA5, dtype=torch.uint8, device=DEV)
    for fmt in ("mx", "nv"):
        nv = fmt == "nv"
        tile_bytes = flib.fluke_fp4_scale_bytes(m, k, 2 if nv else 1)
        codes, scale, row = guard(m * k // 2), guard(tile_bytes), guard(4 * m)
        if nv:
            assert flib.fluke_quant_nvfp4_gpu(p(x), p(codes), p(scale), p(row), m, k, 0) == 0
        else:
            assert flib.fluke_quant_mxfp4_gpu(p(x), p(codes), p(scale), m, k, 0) == 0
        assert (codes[m * k // 2:] == 0xA5).all() and (scale[tile_bytes:] == 0xA5).all() and (row[4 * m if nv else 0:] == 0xA5).all()
        tiles = scale[:tile_bytes].cpu().numpy().reshape(1, -1, 512)
        assert (fp4.untile_scales(tiles, 128, tiles.shape[1] * 4)[m:] == 0xA5).all()
        back, out, gated = guard(m * k * 2), guard(m * n * 2), guard(m * n * 2)
        w = QUANT[fmt](torch.randn(n, k, generator=torch.Generator().manual_seed(3)).half().to(DEV))
        if nv:
            assert flib.fluke_dequant_nvfp4_gpu(p(codes), p(scale), p(row), p(back), m, k, 0) == 0
            assert flib.fluke_gemm_nvfp4_gpu(p(out), p(codes), p(scale), p(row), *(p(t) for t in w), m, n, k, 0) == 0
            assert flib.fluke_gated_mlp_nvfp4_gpu(p(gated), p(codes), p(scale), p(row), *(p(t) for t in w), *(p(t) for t in w), m, n, k, 0) == 0
        else:
            assert flib.fluke_dequant_mxfp4_gpu(p(codes), p(scale), p(back), m, k, 0) == 0
            assert flib.fluke_gemm_mxfp4_gpu(p(out), p(codes), p(scale), *(p(t) for t in w), m, n, k, 0) == 0
            assert flib.fluke_gated_mlp_mxfp4_gpu(p(gated), p(codes), p(scale), *(p(t) for t in w), *(p(t) for t in w), m, n, k, 0) == 0
        assert (back[m * k * 2:] == 0xA5).all() and (out[m * n * 2:] == 0xA5).all() and (gated[m * n * 2:] == 0xA5).all()
        ref = GEMM[fmt](*QUANT[fmt](x), *w)
        assert torch.equal(out[:m * n * 2].view(torch.float16).view(m, n), ref)


@pytest.mark.parametrize("m,n,k", [(2600, 1032, 512), (2600, 1032, 1088), (1500, 72, 512)])
def test_products_write_their_rows_only(flib, m, n, k):
    a, b, u = small(m, n, k, "mx")
    for gated in (False, True):
        out = torch.full((m * n * 2 + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        args = [t.data_ptr() for t in (*a, *b, *(u if gated else ()))]
        fn = flib.fluke_gated_mlp_mxfp4_gpu if gated else flib.fluke_gemm_mxfp4_gpu
        assert fn(out.data_ptr(), *args, m, n, k, 0) == 0
        torch.cuda.synchronize()
        assert (out[m * n * 2:] == 0xA5).all()


def test_operators_refuse_wrong_arguments():
    x = torch.randn(8, 64, device=DEV).half()
    mx, nv = ops.quant_mxfp4(x), ops.quant_nvfp4(x)
    wide = ops.quant_mxfp4(torch.randn(8, 128, device=DEV).half())
    odd = ops.quant_mxfp4(torch.randn(12, 64, device=DEV).half())
    w = torch.ones(64, device=DEV).half()
    flat = torch.zeros(8 * 64 + 1, device=DEV).half()
    bad = [
        lambda: ops.quant_mxfp4(x.float()), lambda: ops.quant_mxfp4(x[:, :48].contiguous()), lambda: ops.quant_nvfp4(x[0]), lambda: ops.quant_mxfp4(x.t()),
        lambda: ops.quant_mxfp4(flat[1:].view(8, 64)), lambda: ops.quant_nvfp4(torch.zeros(1, 16416, device=DEV).half()),
        lambda: ops.dequant_mxfp4(*mx, dtype=torch.float32), lambda: ops.dequant_mxfp4(*mx, dtype=1), lambda: ops.dequant_mxfp4(wide[0], ops.quant_nvfp4(torch.zeros(8, 128, device=DEV).half())[1]),
        lambda: ops.dequant_mxfp4(mx[0].int(), mx[1]), lambda: ops.dequant_nvfp4(*nv[:2], nv[2].half()), lambda: ops.dequant_nvfp4(*nv[:2], nv[2][:4]),
        lambda: ops.gemm_mxfp4(*mx, *wide), lambda: ops.gemm_mxfp4(*mx, *odd), lambda: ops.gemm_mxfp4(mx[0], mx[1][:, :, :256].contiguous(), *mx),
        lambda: ops.gemm_nvfp4(*nv, *nv[:2], None), lambda: ops.gemm_mxfp4(*mx, mx[0].cpu(), mx[1]), lambda: ops.gated_mlp_mxfp4(*mx, *mx, *odd),
        lambda: ops.gated_mlp_mxfp4(*mx, *mx, *wide), lambda: ops.gemm_mxfp4(*mx, *mx, dtype=torch.int8),
        lambda: ops.rmsnorm_block(x, x[:4], w, None, w, 1.0, 1e-5), lambda: ops.rmsnorm_block(x, x.bfloat16(), w, None, w, 1.0, 1e-5),
        lambda: ops.rmsnorm_block(x, x, w[:32], None, w, 1.0, 1e-5), lambda: ops.rmsnorm_block(x, x, w, None, w.bfloat16(), 1.0, 1e-5),
        lambda: ops.rmsnorm_block(x, x, w, w, w, 1.0, 1e-5, seqlen=3), lambda: ops.rmsnorm_block(x, x, w, x[:2], w, 1.0, 1e-5, seqlen=3),
        lambda: ops.rmsnorm_block(x, x, w, w, w, 1.0, 1e-5, seqlen=-1), lambda: ops.rmsnorm_block(x, x, w, x, w, 1.0, 1e-5),
        lambda: ops.rmsnorm_block(x, x, w, None, w, 1.0, 1e-5, residual_out=x.float()), lambda: ops.rmsnorm_block(x, x, w, None, w, 1.0, 1e-5, residual_out=x.t()),
        lambda: ops.rmsnorm_block(x, x, flat[1:65], None, w, 1.0, 1e-5),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            call()
            pytest.fail(f"case {i} was taken")


def test_empty_batches():
    z = torch.zeros(0, 64, device=DEV).half()
    w = ops.quant_mxfp4(torch.randn(8, 64, device=DEV).half())
    q, n = ops.quant_mxfp4(z), ops.quant_nvfp4(z)
    assert q[0].shape == (0, 32) and q[1].shape == (0, 1, 512) and n[2].shape == (0,)
    assert ops.dequant_mxfp4(*q).shape == (0, 64) and ops.gemm_mxfp4(*q, *w).shape == (0, 8) and ops.gated_mlp_mxfp4(*q, *w, *w).shape == (0, 8)
    assert [t.shape[0] for t in ops.rmsnorm_block(z, z, None, None, torch.ones(64, device=DEV).half(), 1.0, 1e-5, quant="nvfp4")] == [0, 0, 0, 0]


def chain(x, res, gate, w, fmt):
    """One transformer layer between its norms, as a program would run it; what every step gave."""
    q = fmt + "fp4"
    s1, *h1 = ops.rmsnorm_block(x, res, w["post"], gate, w["pre"], 0.75, 1e-5, seqlen=50, quant=q)
    qkv = GEMM[fmt](*h1, *w["qkv"])
    attn = qkv[:, :512].contiguous()                # the attention itself is the caller's
    proj = GEMM[fmt](*QUANT[fmt](attn), *w["out"])
    s2, *h2 = ops.rmsnorm_block(proj, s1, w["post"], gate, w["pre"], 0.75, 1e-5, seqlen=50, quant=q)
    mlp = GATED[fmt](*h2, *w["gate"], *w["up"])
    down = GEMM[fmt](*QUANT[fmt](mlp), *w["down"])
    s3, out = ops.rmsnorm_block(down, s2, w["post"], None, w["pre"], 0.75, 1e-5)
    return dict(s1=s1, h1=h1, qkv=qkv, attn=attn, proj=proj, s2=s2, h2=h2, mlp=mlp, down=down, s3=s3, out=out)


def layer(fmt, m, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    w = {name: QUANT[fmt]((r(n, k) / k ** 0.5).half()) for name, n, k in
         (("qkv", 1536, 512), ("out", 512, 512), ("gate", 2048, 512), ("up", 2048, 512), ("down", 512, 2048))}
    w["post"], w["pre"] = ((1 + 0.1 * r(512)).half() for _ in range(2))
    return r(m, 512).half(), r(m, 512).half(), (0.5 * r(-(-m // 50), 512)).half(), w


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m", [1, 130, 2100])
def test_a_layer_step_by_step(m, fmt):
    """Every step of a layer against the oracle on the step's own inputs."""
    x, res, gate, w = layer(fmt, m)
    c = chain(x, res, gate, w, fmt)
    val = lambda q, k: fp4.values(*unpacked(q, k, fmt), fmt)
    def product(got, a, b, k):
        want = val(a, k) @ val(b, k).T
        assert (np.abs(f64(got) - want) <= half_step(want, "f16") + k * 2.0 ** -24 * (np.abs(val(a, k)) @ np.abs(val(b, k)).T)).all()
    num = lambda v: v.float().cpu().numpy()
    round16 = lambda v: torch.from_numpy(v).half().float().numpy()
    for xs, rs, gs, s, h in ((x, res, gate, c["s1"], c["h1"]), (c["proj"], c["s1"], gate, c["s2"], c["h2"]), (c["down"], c["s2"], None, c["s3"], c["out"])):
        stream, nxt = fp4.rmsnorm_block(num(xs), num(rs), num(w["post"]), None if gs is None else num(gs), num(w["pre"]), 0.75, 1e-5, 50, round16)
        assert np.array_equal(num(s), stream)
        if isinstance(h, list):
            check_quantised(h, fp4.quantise(nxt, fmt), fmt, m, 512)
        else:
            assert np.array_equal(num(h), round16(nxt))
    product(c["qkv"], c["h1"], w["qkv"], 512)
    product(c["proj"], QUANT[fmt](c["attn"]), w["out"], 512)
    product(c["down"], QUANT[fmt](c["mlp"]), w["down"], 2048)


def unpacked(q, k, fmt):
    codes = q[0].cpu().numpy()
    c = np.stack((codes & 15, codes >> 4), -1).reshape(len(codes), k)
    return c, fp4.untile_scales(q[1].cpu().numpy(), len(codes), k // fp4.BLOCK[fmt]), q[2].cpu().numpy() if fmt == "nv" else None


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_a_layer_captured_and_replayed(fmt):
    """Two layers of different sizes captured into two graphs and replayed in turns with new inputs, beside eager calls."""
    graphs, stream = [], torch.cuda.Stream()
    for m in (37, 2100):
        x, res, gate, w = layer(fmt, m, seed=m)
        ops.set_stream(stream)
        try:
            with torch.cuda.stream(stream):
                chain(x, res, gate, w, fmt)
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    outs = chain(x, res, gate, w, fmt)
        finally:
            ops.set_stream(None)
        graphs.append((graph, x, res, gate, w, outs))
    torch.cuda.synchronize()
    for turn in range(3):
        for graph, x, res, gate, w, outs in graphs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(turn)).half())
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, res, gate, w, outs in graphs:
            eager = chain(x, res, gate, w, fmt)
            assert all(torch.equal(bits(outs[k]), bits(eager[k])) for k in ("s1", "qkv", "proj", "s2", "mlp", "down", "s3", "out"))


def test_two_threads_with_a_stream_each():
    import threading
    inputs = [layer("nv", m, seed=m) for m in (300, 1000)]
    want = [bits(chain(*i, "nv")["out"]) for i in inputs]
    torch.cuda.synchronize()
    failed = []
    def run(k):
        s = torch.cuda.Stream()
        ops.set_stream(s)
        try:
            with torch.cuda.stream(s):
                for _ in range(20):
                    out = chain(*inputs[k], "nv")["out"]
                    s.synchronize()
                    if not torch.equal(bits(out), want[k]):
                        failed.append(k)
        finally:
            ops.set_stream(None)
    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed


def test_more_than_2_pow_31_values():
    """[270001, 8192] in and out again: the last rows, whose offsets pass 32 bits."""
    m, k = 270001, 8192
    x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    w = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    for fmt in ("mx", "nv"):
        q = QUANT[fmt](x)
        back = DEQUANT[fmt](*q, dtype=torch.bfloat16)
        for lo in (0, 262144, m - 3):
            want = fp4.quantise(f64(x[lo:lo + 3]), fmt)
            assert np.array_equal(f64(back[lo:lo + 3]), fp4.values(*want, fmt))
        del q, back
    s, h = ops.rmsnorm_block(x, x, w, None, w, 1.0, 1e-5)
    ref = ops.rmsnorm_block(x[-3:], x[-3:], w, None, w, 1.0, 1e-5)
    assert torch.equal(s[-3:], ref[0]) and torch.equal(h[-3:], ref[1])


def test_a_product_of_more_than_2_pow_31_values():
    m, n, k = 300100, 8192, 64
    a, b, u = small(m, n, k, "mx")
    for gated in (False, True):
        out = GATED["mx"](*a, *b, *u) if gated else GEMM["mx"](*a, *b)
        tail = ops.dequant_mxfp4(*a, dtype=torch.bfloat16)[-200:].contiguous()
        q = ops.quant_mxfp4(tail)   # values of the format come back as they are
        want = GATED["mx"](*q, *b, *u) if gated else GEMM["mx"](*q, *b)
        torch.testing.assert_close(out[-200:].float(), want.float(), rtol=2.0 ** -10, atol=1e-4)
        del out
