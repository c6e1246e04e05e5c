"""4-bit operators where ordinary values do not take them, against oracle/fp4.py as in test_fp4_gpu.py."""
import numpy as np
import pytest
import torch

from fluke_b200 import ops
from oracle import fp4
from test_fp4_gpu import DEV, GATED, GEMM, TYPES, half_step, on_gpu

pytestmark = pytest.mark.gpu

# (rows, weight rows, K) of the split, the resident and the streamed form of the products
FORMS = [(5, 264, 96), (64, 136, 2080), (2600, 1032, 96), (2600, 1032, 1024), (2600, 1032, 2080)]


def one_term(m, n, k, fmt, values, weights):
    """a with values[r % len] and b with weights[c % len] in the last column and zeros elsewhere: sums are single products, which f32 holds."""
    a, b = np.zeros((m, k), np.float32), np.zeros((n, k), np.float32)
    a[:, -1] = np.resize(np.asarray(values, np.float32), m)
    b[:, -1] = np.resize(np.asarray(weights, np.float32), n)
    return fp4.quantise(a, fmt), fp4.quantise(b, fmt)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_gates_at_which_silu_is_small(m, n, k, fmt, dtype):
    """Gates from -80 (bf16; -12 in f16) to 40, under an up that brings the result back into the type. Gate and up are exact, so what is left is the rounding and the
    relative error of silu * up in f32: ex2.approx 2^-22 and its argument's 2^-23 |g|, 1 + exp(-g) 2^-24, rcp.approx 2^-23 and two products of
    2^-24 each, below (|g| + 5) 2^-23. Some gates lie below -87, where silu may be zero: it is less than 2^-119 there."""
    low, high = (80, 40) if dtype == "bf16" else (12, 12)
    steps = np.concatenate(([-1000, -100], -np.geomspace(low, 1e-3, 61), np.geomspace(1e-3, high, 30)))
    up = np.exp2(np.round(np.where(steps < -1, np.minimum(-steps * 1.4427, 115), 1))) if dtype == "bf16" else np.where(np.arange(len(steps)) % 2, 8.0, -3.0)
    a, b = one_term(m, n, k, fmt, (1.0, 0.75, 0.5, 1.0), steps)
    u = one_term(m, n, k, fmt, (1.0,), up)[1]
    va, vb, vu = (fp4.values(*q, fmt) for q in (a, b, u))
    gate, lift = np.outer(va[:, -1], vb[:, -1]), np.outer(va[:, -1], vu[:, -1])
    want = gate * np.exp(np.minimum(gate, 0)) / (1 + np.exp(-np.abs(gate))) * lift
    got = GATED[fmt](*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=TYPES[dtype]).cpu().double().numpy()
    err = np.abs(want) * (np.abs(gate) + 5) * 2.0 ** -23
    tol = half_step(np.abs(want) + err, dtype) + err + np.where(gate < -87, np.abs(lift) * 2.0 ** -119, 0)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_a_weight_row_without_a_value_stays_alone(m, n, k, fmt):
    """A gate row, an up row with an infinity: its column is NaN, the neighbours are what they are without it."""
    g = torch.Generator().manual_seed(n)
    a, b, u = (fp4.quantise(torch.randn(r, k, generator=g).numpy(), fmt) for r in (m, n, n))
    want = GATED[fmt](*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=torch.bfloat16)

    def spoiled(q, rows_):
        codes, scale, row = (None if t is None else t.copy() for t in q)
        for r in rows_:
            codes[r, :fp4.BLOCK[fmt]], scale[r, 0] = 0, 255 if fmt == "mx" else 0x7F
            if row is not None:
                row[r] = np.nan
        return codes, scale, row
    got = GATED[fmt](*on_gpu(a), *on_gpu(spoiled(b, (6, 37))), *on_gpu(spoiled(u, (101, n - 2))), dtype=torch.bfloat16)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[6, 37, 101, n - 2]] = True
    assert torch.isnan(got[:, bad.to(DEV)]).all()
    assert torch.equal(got[:, ~bad.to(DEV)], want[:, ~bad.to(DEV)])


def random_rows(seed, m, k, scale, fmt="nv"):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(seed))
    x[m // 3] = 0
    return fp4.quantise((x * scale).bfloat16().double().numpy(), fmt)


def gated_bound(va, vb, vu, gate, up, k):
    """Of silu(gate) * up with sums of K products in f32 (the derivative of silu is below 1.1)."""
    dg, du = (k * 2.0 ** -24 * (np.abs(va) @ np.abs(w).T) for w in (vb, vu))
    silu = gate * np.exp(np.minimum(gate, 0)) / (1 + np.exp(-np.abs(gate)))
    return silu * up, np.abs(up) * 1.1 * dg + np.abs(silu) * du + 1.1 * dg * du + np.abs(silu * up) * (np.minimum(np.abs(gate), 87) + 5) * 2.0 ** -23


def close(got, want, tol, dtype):
    """Within tol and half a step, or infinite where the type holds no such number (from half a step above its largest one on)."""
    top = torch.finfo(TYPES[dtype]).max * (1 + torch.finfo(TYPES[dtype]).eps / 4)
    return ((np.abs(got - want) <= tol + half_step(want, dtype)) | (np.isinf(got) & (got * want > 0) & (np.abs(want) + tol >= top))).all()


@pytest.mark.parametrize("sa,sb", [(1e36, 0.01), (0.01, 1e36), (1e37, 1e-30), (1e-30, 1e37), (1e-22, 1e-12)])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_row_scales_that_are_far_apart(m, n, k, sa, sb):
    """nvfp4 rows and weights of very different magnitudes: finite results stay finite, in either operand's favour."""
    a, b = random_rows(m, m, k, sa), random_rows(n + 1, n, k, sb)
    va, vb = fp4.values(*a, "nv"), fp4.values(*b, "nv")
    want = va @ vb.T
    assert np.abs(want).max() < 3e38
    got = GEMM["nv"](*on_gpu(a), *on_gpu(b), dtype=torch.bfloat16).cpu().double().numpy()
    tol = half_step(want, "bf16") + k * 2.0 ** -24 * (np.abs(va) @ np.abs(vb).T)
    assert (np.abs(got - want) <= tol).all()
    # gates of that size, finite and mostly far below zero or above, under an up near one; rows of zeros give a gate of zero
    u = random_rows(n + 2, n, k, 1.0 / sa)
    vu = fp4.values(*u, "nv")
    up = va @ vu.T
    want, tol = gated_bound(va, vb, vu, va @ vb.T, up, k)
    keep = np.abs(want) < 3e38
    got = GATED["nv"](*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=torch.bfloat16).cpu().double().numpy()
    assert np.isfinite(got[keep]).all() and (np.abs(got - want) <= tol + half_step(want, "bf16"))[keep].all()


@pytest.mark.parametrize("m,n,k", FORMS)
def test_an_up_of_any_size_under_a_gate_of_zero(m, n, k):
    a, b, u = random_rows(1, m, k, 1e36), random_rows(2, n, k, 0.0), random_rows(3, n, k, 0.01)
    got = GATED["nv"](*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=torch.bfloat16)
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_row_scales_that_are_no_powers_of_two(m, n, k, dtype):
    """Published nvfp4 weights carry one f32 per tensor: repeated per row it is a row scale like any other (two more roundings of 2^-24)."""
    a, b, u = random_rows(1, m, k, 1.0), random_rows(2, n, k, 1.0 / k ** 0.5), random_rows(3, n, k, 1.0 / k ** 0.5)
    g = np.random.default_rng(4)
    a = (a[0], a[1], (a[2] * g.uniform(0.5, 2, m)).astype(np.float32))
    b, u = ((q[0], q[1], np.full(n, q[2].max() * f, np.float32)) for q, f in ((b, 0.7), (u, 1.3)))
    va, vb, vu = (fp4.values(*q, "nv") for q in (a, b, u))
    gate, up = va @ vb.T, va @ vu.T
    got = GEMM["nv"](*on_gpu(a), *on_gpu(b), dtype=TYPES[dtype]).cpu().double().numpy()
    assert close(got, gate, k * 2.0 ** -24 * (np.abs(va) @ np.abs(vb).T) + np.abs(gate) * 2.0 ** -23, dtype)
    want, tol = gated_bound(va, vb, vu, gate, up, k + 2)   # two more roundings in either sum
    got = GATED["nv"](*on_gpu(a), *on_gpu(b), *on_gpu(u), dtype=TYPES[dtype]).cpu().double().numpy()
    assert close(got, want, tol, dtype)


def test_a_missing_part_is_not_another_operator():
    """Without row scales nvfp4 bytes are not mxfp4 bytes (up to 64 columns their scales have the same shape), and without an up there is no gated product."""
    x, w = (torch.randn(8, 64, device=DEV).half() for _ in range(2))
    nv, wn, mx, wm = ops.quant_nvfp4(x), ops.quant_nvfp4(w), ops.quant_mxfp4(x), ops.quant_mxfp4(w)
    for call in (lambda: ops.dequant_nvfp4(*nv[:2], None), lambda: ops.gemm_nvfp4(*nv[:2], None, *wn[:2], None), lambda: ops.gemm_nvfp4(*nv, *wn[:2], None),
                 lambda: ops.gemm_nvfp4(*nv[:2], None, *wn), lambda: ops.gated_mlp_nvfp4(*nv[:2], None, *wn[:2], None, *wn[:2], None),
                 lambda: ops.gated_mlp_nvfp4(*nv, *wn, *wn[:2], None), lambda: ops.gated_mlp_nvfp4(*nv, *wn, None, None, None),
                 lambda: ops.gated_mlp_mxfp4(*mx, *wm, None, None), lambda: ops.gated_mlp_mxfp4(*mx, *wm, None, wm[1]), lambda: ops.gemm_mxfp4(*mx, None, None)):
        with pytest.raises((TypeError, ValueError)):
            call()


# ---- rows that walk: more rows than are resident at once, every width of lane and unit -----------

def sample(m):
    """Rows of the first turn, of later ones and of the ragged end."""
    return np.unique(np.concatenate((np.arange(20), np.random.default_rng(m).integers(0, m, 90), np.arange(m - 20, m))))


def stream_of(m, k, t, seed):
    """Normal values with some large channels; rows and blocks of zeros and rows without a value among them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=DEV)
    x[:, torch.rand(k, generator=g, device=DEV) < 0.02] *= 20
    x[5], x[m - 2, :32], x[m - 7, k - 1], x[m - 11, 40 % k] = 0, 0, float("inf"), float("nan")
    return x.to(t)


def check_rows(got, want, fmt, rows_, m, k):
    codes, scales, row = want
    blocks = k // fp4.BLOCK[fmt]
    assert np.array_equal(got[0][torch.from_numpy(rows_).to(DEV)].cpu().numpy(), fp4.pack(codes))
    tiles = fp4.untile_scales(got[1].cpu().numpy(), m, got[1].shape[1] * 4)[rows_]
    assert np.array_equal(tiles[:, :blocks], scales) and not tiles[:, blocks:].any()
    if fmt == "nv":
        assert np.array_equal(got[2].cpu().numpy()[rows_], row, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,k", [(20011, 32), (20011, 256), (9331, 480), (9331, 512), (9331, 736), (9331, 768), (9331, 992), (9331, 1024), (9331, 1504), (9331, 1536), (9331, 2016),
                                 (9331, 2048), (700, 2080), (700, 4096), (700, 4128), (700, 16384)])
def test_nvfp4_quantiser_of_many_rows(m, k, dtype):
    x, rows_ = stream_of(m, k, TYPES[dtype], k), sample(m)
    check_rows(ops.quant_nvfp4(x), fp4.quantise(x[torch.from_numpy(rows_).to(DEV)].cpu().double().numpy(), "nv"), "nv", rows_, m, k)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fmt", [None, "mx", "nv"])
@pytest.mark.parametrize("m,k,seqlen", [(20011, 32, 0), (9331, 256, 1333), (9331, 480, 0), (9331, 512, 1333), (9331, 736, 1), (9331, 768, 0), (9331, 992, 1333), (9331, 1024, 7),
                                        (9331, 1504, 0), (9331, 1536, 1333), (9331, 2016, 1000), (9331, 2048, 0), (700, 2080, 100), (700, 4096, 7), (700, 16384, 1)])
def test_norms_of_many_rows(m, k, seqlen, fmt, dtype):
    """In place of the residual, which a later turn of the same warp must not have read too late."""
    t = TYPES[dtype]
    x, res = stream_of(m, k, t, k), stream_of(m, k, t, k + 1)
    g = torch.Generator(device=DEV).manual_seed(k + 2)
    post, pre = ((1 + 0.1 * torch.randn(k, generator=g, device=DEV)).to(t) for _ in range(2))
    gate = (0.5 * torch.randn(-(-m // seqlen) if seqlen else 1, k, generator=g, device=DEV)).to(t)
    rows_ = sample(m)
    at = torch.from_numpy(rows_).to(DEV)
    num = lambda v: v.float().cpu().numpy()
    round16 = lambda v: torch.from_numpy(v).to(t).float().numpy()
    own = num(gate[at // seqlen] if seqlen else gate.expand(len(rows_), k))
    stream, h = fp4.rmsnorm_block(num(x[at]), num(res[at]), num(post), own, num(pre), 0.75, 1e-5, 1, round16)
    got = ops.rmsnorm_block(x, res, post, gate, pre, 0.75, 1e-5, seqlen=seqlen, quant=None if fmt is None else fmt + "fp4", residual_out=res)
    assert np.array_equal(num(got[0][at]), stream, equal_nan=True)
    if fmt is None:
        assert np.array_equal(num(got[1][at]), round16(h), equal_nan=True)
    else:
        check_rows(got[1:], fp4.quantise(h, fmt), fmt, rows_, m, k)


@pytest.mark.parametrize("fmt", ["mx", "nv"])
@pytest.mark.parametrize("m,k", [(7, 1024), (1300, 512), (9331, 1056)])
def test_quantised_norms_in_place_of_the_input(m, k, fmt):
    """Codes, every block scale and row scales of a call whose stream goes to x, against those of a call with a stream of its own."""
    g = torch.Generator(device=DEV).manual_seed(m)
    t = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()
    x, res, w, gate = t(m, k), t(m, k), t(k), t(-(-m // 100), k)
    want = ops.rmsnorm_block(x, res, w, gate, w, 0.5, 1e-5, seqlen=100, quant=fmt + "fp4")
    got = ops.rmsnorm_block(x, res, w, gate, w, 0.5, 1e-5, seqlen=100, quant=fmt + "fp4", residual_out=x)
    assert got[0].data_ptr() == x.data_ptr()
    blocks = k // fp4.BLOCK[fmt]
    for a, b in zip(want, got):
        if a.dim() == 3:
            a, b = (torch.from_numpy(fp4.untile_scales(v.cpu().numpy(), m, blocks).copy()) for v in (a, b))
        assert torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_more_than_2_pow_31_units(flib, fmt):
    """[4194433, 8192]: 2^31 + 66048 units of 16 values, which the mxfp4 quantiser and both read-backs work through in two runs of rows. 69 GB, read back in place."""
    m, k = (1 << 22) + 129, 8192
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 110e9:
        pytest.skip("needs 110 GB of free memory")
    x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    rows_ = np.concatenate((np.arange(3), np.arange((1 << 22) - 140, (1 << 22) - 120), np.arange((1 << 22) - 3, (1 << 22) + 3), np.arange(m - 3, m)))
    at = torch.from_numpy(rows_).to(DEV)
    want = fp4.quantise(x[at].cpu().double().numpy(), fmt)
    q = ops.quant_mxfp4(x) if fmt == "mx" else ops.quant_nvfp4(x)
    assert np.array_equal(q[0][at].cpu().numpy(), fp4.pack(want[0]))
    x.fill_(float("nan"))
    torch.cuda.synchronize()
    args = [t.data_ptr() for t in (*q, x)]
    assert (flib.fluke_dequant_mxfp4_gpu if fmt == "mx" else flib.fluke_dequant_nvfp4_gpu)(*args, m, k, 1) == 0
    torch.cuda.synchronize()
    assert np.array_equal(x[at].cpu().double().numpy(), fp4.values(*want, fmt))
    assert not torch.isnan(x[:, 0]).any() and not torch.isnan(x[:, -1]).any()
    del x, q
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_quotients_of_every_16_bit_mantissa(dtype):
    """Rows whose blocks have each of the eight mantissas of an e4m3 scale, with every mantissa of the type in four binades under it, and every block maximum."""
    t = TYPES[dtype]
    bits_ = 10 if dtype == "f16" else 7
    mantissas = 1 + torch.arange(1 << bits_) / (1 << bits_)
    values = torch.cat([mantissas * 2.0 ** e for e in (-2, -1, 0, 1)] + [-mantissas])   # below 4
    values = torch.cat((values, torch.zeros(-len(values) % 15)))
    blocks = []
    for eighth in range(8):   # a block maximum of 6 (1 + i / 8) gives the scale 1 + i / 8 in a row of scale 1
        blocks.append(torch.cat((torch.full((len(values) // 15, 1), 6 * (1 + eighth / 8)), values.view(-1, 15)), 1))
    tops = torch.cat([mantissas * 2.0 ** e for e in (-8, -3, 0, 2, 7, 11)])
    blocks.append(torch.cat((tops.clamp_max(2688)[:, None], torch.rand(len(tops), 15, generator=torch.Generator().manual_seed(1)) * tops[:, None]), 1))
    x = torch.cat(blocks)
    x = torch.cat((x, torch.zeros(-len(x) % 63, 16))).view(-1, 63 * 16)
    x = torch.cat((torch.full((len(x), 16), 2688.0), x), 1).to(t)   # the row's scale is 1 (some of the last rows hold larger values)
    want = fp4.quantise(x.double().numpy(), "nv")
    assert (want[2][:len(values) * 8 // 15 // 63] == 1).all()
    check_rows(ops.quant_nvfp4(x.to(DEV)), want, "nv", np.arange(len(x)), *x.shape)
