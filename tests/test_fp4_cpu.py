"""Microscaled 4-bit floating point without a GPU: the oracle against published tables, the preparation
functions against the oracle, sizes, and what the entry points refuse before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from fluke_b200 import lib as L, ops, prep
from oracle import fp4


def test_oracle_elements_round_to_nearest_ties_to_even():
    v = np.array([0, .25, .26, .5, .75, .74, 1.25, 1.26, 1.75, 1.74, 2.5, 2.51, 3.5, 3.49, 5, 5.01, 6, 7.9, 1e9])
    want = np.array([0, 0, .5, .5, 1, .5, 1, 1.5, 2, 1.5, 2, 3, 4, 3, 4, 6, 6, 6, 6])
    assert np.array_equal(fp4.element(fp4.e2m1(v)), want)
    assert np.array_equal(fp4.e2m1(-v), fp4.e2m1(v) | 8)


def test_oracle_e4m3_agrees_with_torch():
    t = torch.cat((torch.linspace(0, 448, 20001), 2.0 ** torch.linspace(-12, 8.8, 5001)))
    assert np.array_equal(fp4.to_e4m3(t.double().numpy()), t.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", ["mx", "nv"])
def test_oracle_error_is_that_of_the_format(fmt):
    """Half a step of the element grid, plus what saturates (mx: up to 8 / 6 of the largest element) and what the block scale's own
    rounding moves (nv: 2^-4 of the block's largest value)."""
    x = np.random.default_rng(1).standard_normal((64, 256))
    q = fp4.quantise(x.astype(np.float32), fmt)
    v, b = fp4.values(*q, fmt), np.repeat(np.abs(x.reshape(64, -1, fp4.BLOCK[fmt])).max(-1), fp4.BLOCK[fmt], axis=1)
    assert (np.abs(v - x) <= b * (1 / 4 if fmt == "mx" else 1 / 6 + 1 / 16)).all()


def rows(m, k):
    g = torch.Generator().manual_seed(m + k)
    x = torch.randn(m, k, generator=g)
    x[m // 2] = 0
    x[0, :32] = torch.tensor([0.25, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, 6.0, 7.9, -0.0, 0.0, 0.5, 1e-6, -1e-6] * 2)
    x[m - 1, 5] = float("nan")
    x[m - 2, 7] = float("inf")
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(4, 32), (5, 96), (130, 160), (9, 1024)])
def test_preparation_agrees_with_the_oracle(m, k, dtype):
    x = rows(m, k).to(dtype)
    for fmt, fn in (("mx", prep.quantize_mxfp4), ("nv", prep.quantize_nvfp4)):
        codes, scales, row = fp4.quantise(x.double().numpy(), fmt)
        got = fn(x)
        assert np.array_equal(got[0].numpy(), fp4.pack(codes)) and np.array_equal(got[1].numpy(), fp4.tile_scales(scales))
        if fmt == "nv":
            assert np.array_equal(got[2].numpy(), row, equal_nan=True)
    with pytest.raises(ValueError):
        prep.quantize_mxfp4(torch.zeros(2, 48))


def test_scale_bytes(flib):
    for rows_, cols, fmt, want in ((1, 32, 1, 512), (128, 128, 1, 512), (129, 160, 1, 2048), (128, 64, 2, 512), (1, 96, 2, 1024), (0, 32, 1, 0),
                                   (1, 32, 0, 0), (1, 32, 3, 0), (1, -32, 1, 0), (1 << 20, 1 << 15, 2, (1 << 13) * (1 << 9) * 512)):
        assert flib.fluke_fp4_scale_bytes(rows_, cols, fmt) == want


P = 1 << 20   # an address that is aligned and never followed: every call below is refused before a launch


def test_c_entries_refuse(flib):
    ok = 0
    invalid, misaligned = 1, 716   # cudaErrorInvalidValue, cudaErrorMisalignedAddress
    q = flib.fluke_quant_mxfp4_gpu
    assert q(P, P, P, 0, 64, 0) == ok                     # nothing to do
    for args in ((P, P, P, 4, 48, 0), (P, P, P, 4, 0, 0), (P, P, P, -1, 64, 0), (P, P, P, 4, 64, 2), (0, P, P, 4, 64, 0), (P, 0, P, 4, 64, 0), (P, P, 0, 4, 64, 0)):
        assert q(*args) == invalid
        assert b"invalid argument" in flib.fluke_last_error()
    for args in ((P + 16, P, P, 4, 64, 0), (P, P + 8, P, 4, 64, 0), (P, P, P + 4, 4, 64, 0)):
        assert q(*args) == misaligned
    assert flib.fluke_quant_nvfp4_gpu(P, P, P, 0, 4, 64, 0) == invalid
    assert flib.fluke_quant_nvfp4_gpu(P, P, P, P, 4, 16416, 0) == invalid
    assert flib.fluke_dequant_mxfp4_gpu(P, P, P, 4, 40, 0) == invalid
    assert flib.fluke_dequant_mxfp4_gpu(P, P, P + 16, 4, 64, 1) == misaligned
    assert flib.fluke_dequant_nvfp4_gpu(P, P, 0, P, 4, 64, 0) == invalid
    g = flib.fluke_gemm_mxfp4_gpu
    assert g(P, P, P, P, P, 0, 64, 64, 0) == ok
    for args in ((P, P, P, P, P, 4, 64, 48, 0), (P, P, P, P, P, 4, 60, 64, 0), (P, P, P, P, P, 4, 0, 64, 0), (P, P, P, P, P, -4, 64, 64, 0),
                 (P, P, P, P, P, 4, 64, 64, 7), (0, P, P, P, P, 4, 64, 64, 0), (P, P, 0, P, P, 4, 64, 64, 0), (P, P, P, P, 0, 4, 64, 64, 0)):
        assert g(*args) == invalid
    for k in range(5):
        args = [P] * 5 + [4, 64, 64, 0]
        args[k] += 8
        assert g(*args) == misaligned
    assert flib.fluke_gemm_nvfp4_gpu(P, P, P, 0, P, P, P, 4, 64, 64, 0) == invalid
    assert flib.fluke_gemm_nvfp4_gpu(P, P, P, P, P, P, P + 4, 4, 64, 64, 0) == misaligned
    assert flib.fluke_gated_mlp_mxfp4_gpu(P, P, P, P, P, 0, P, 4, 64, 64, 0) == invalid
    assert flib.fluke_gated_mlp_mxfp4_gpu(P, P, P, P, P, P, 0, 4, 64, 64, 0) == invalid
    assert flib.fluke_gated_mlp_nvfp4_gpu(P, P, P, P, P, P, P, P, P, 0, 4, 64, 64, 0) == invalid


def test_sizes_next_to_the_largest_int_are_refused(flib):
    # rounding such a size up to a tile, or a step from the last row, does not fit 32 bits
    most, wide = (1 << 31) - 1, (1 << 31) - 32
    for rows_ in (most, most - 127, most - (1 << 20) + 1):
        assert flib.fluke_quant_mxfp4_gpu(P, P, P, rows_, 32, 0) == 1
        assert flib.fluke_quant_nvfp4_gpu(P, P, P, P, rows_, 32, 0) == 1
        assert flib.fluke_dequant_nvfp4_gpu(P, P, P, P, rows_, 32, 0) == 1
        assert flib.fluke_gemm_mxfp4_gpu(P, P, P, P, P, rows_, 8, 32, 0) == 1
        b = L.fluke_rmsnorm_block_t(rows_, 32, 0, 0, P, P, P, P, P, 1.0, 1e-5, P, 0, P, P, P)
        assert flib.fluke_rmsnorm_block_gpu(ctypes.byref(b)) == 1
    assert flib.fluke_gemm_mxfp4_gpu(P, P, P, P, P, 1, most - 7, 32, 0) == 1
    assert flib.fluke_gemm_mxfp4_gpu(P, P, P, P, P, 1, 8, wide, 0) == 1
    assert flib.fluke_gated_mlp_mxfp4_gpu(P, P, P, P, P, P, P, 1, most - 7, 32, 0) == 1
    assert flib.fluke_quant_mxfp4_gpu(P, P, P, 1, wide, 0) == 1


def test_scale_bytes_of_columns_that_no_operator_takes(flib):
    for fmt in (1, 2):
        assert flib.fluke_fp4_scale_bytes(4, 48, fmt) == 0
        assert flib.fluke_fp4_scale_bytes(4, 31, fmt) == 0


def test_c_entry_of_the_norms_refuses(flib):
    def call(**change):
        b = L.fluke_rmsnorm_block_t(4, 64, 0, 0, P, P, P, P, P, 1.0, 1e-5, P, 0, P, P, P)
        for k, v in change.items():
            setattr(b, k, v)
        return flib.fluke_rmsnorm_block_gpu(ctypes.byref(b))
    assert flib.fluke_rmsnorm_block_gpu(None) == 1
    assert call(n_tokens=0) == 0
    for change in (dict(n_tokens=-1), dict(hidden_dim=48), dict(hidden_dim=0), dict(hidden_dim=16416), dict(dtype=2), dict(seqlen=-1), dict(out_format=3),
                   dict(out_format=-1), dict(x=0), dict(residual=0), dict(residual_out=0), dict(out=0), dict(out_format=1, scale=0),
                   dict(out_format=2, row_scale=0)):
        assert call(**change) == 1, change
    for change in (dict(x=P + 16), dict(residual=P + 16), dict(residual_out=P + 16), dict(out=P + 16), dict(post_weight=P + 16), dict(gate=P + 2),
                   dict(pre_weight=P + 16), dict(out_format=1, out=P + 8), dict(out_format=2, scale=P + 8)):
        assert call(**change) == 716, change


def test_norms_refuse_outputs_that_overlap_other_rows(flib):
    # [4, 64]: 512 bytes. A row's output may take the place of its own input, not of another row's.
    def call(**change):
        b = L.fluke_rmsnorm_block_t(4, 64, 0, 0, P, P + 4096, P + 8192, 0, P + 8192, 1.0, 1e-5, P + 16384, 0, P + 20480, P + 24576, P + 28672)
        for k, v in change.items():
            setattr(b, k, v)
        return flib.fluke_rmsnorm_block_gpu(ctypes.byref(b))
    for change in (dict(residual_out=P + 128), dict(residual_out=P + 4096 + 128), dict(residual_out=P + 4096 - 128), dict(residual=P + 16384 + 384),
                   dict(out=P + 128), dict(out=P + 4096 - 32), dict(out=P + 16384), dict(out=P + 16384 + 384),
                   dict(out_format=1, out=P), dict(out_format=1, out=P + 4096), dict(out_format=2, out=P + 16384 + 496)):
        assert call(**change) == 1, change


def test_operators_refuse_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.float16)
    codes, scale = prep.quantize_mxfp4(x)
    for call in (lambda: ops.quant_mxfp4(x), lambda: ops.quant_nvfp4(x), lambda: ops.dequant_mxfp4(codes, scale), lambda: ops.gemm_mxfp4(codes, scale, codes, scale),
                 lambda: ops.gated_mlp_mxfp4(codes, scale, codes, scale, codes, scale), lambda: ops.rmsnorm_block(x, x, None, None, None, 1.0, 1e-5)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        ops.rmsnorm_block(x, x, None, None, None, 1.0, 1e-5, quant="fp8")
