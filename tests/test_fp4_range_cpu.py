"""Host-side parts of the 4-bit operators that need no GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from fluke_b200 import lib as L, prep

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_failed_capacity_query_is_asked_again(tmp_path):
    """Answers 0, -1, 7: the failures are returned and not kept, the 7 is (a fourth question would get a 9)."""
    exe = str(tmp_path / "kept_test")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-pthread", os.path.join(ROOT, "tests", "csrc", "kept_test.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout
    assert out.split() == ["0/1", "-1/2", "7/3", "7/3", "7/3", "0"]


P = 1 << 20   # an address that is aligned and never followed: every call below is refused before a launch


def test_norms_refuse_outputs_over_what_every_row_reads(flib):
    """[256, 64], a gate per 100 rows: 32768 bytes of rows, 128 of a weight, 384 of gates, 8192 of codes, 1024 of scales, 1024 of row scales."""
    at = {name: P + i * 65536 for i, name in enumerate(("x", "residual", "post_weight", "gate", "pre_weight", "residual_out", "out", "scale", "row_scale"))}

    def call(**change):
        b = L.fluke_rmsnorm_block_t()
        for k, v in {**at, **dict(n_tokens=256, hidden_dim=64, seqlen=100, alpha=1.0, eps=1e-5), **change}.items():
            setattr(b, k, v)
        return flib.fluke_rmsnorm_block_gpu(ctypes.byref(b))

    def over(out, n_out, other, n_other, fmt):
        for delta in (0, -(n_out - 32), n_other - 32):   # the same start, the output's last and first bytes
            assert call(**{"out_format": fmt, out: at[other] + delta}) == 1, (out, other, delta, fmt)
    for fmt, n_out, n_scale in ((0, 32768, 0), (1, 8192, 1024), (2, 8192, 1024)):
        assert not n_scale or flib.fluke_fp4_scale_bytes(256, 64, fmt) == n_scale
        for other, n in (("post_weight", 128), ("gate", 384), ("pre_weight", 128)):
            over("residual_out", 32768, other, n, fmt)
            over("out", n_out, other, n, fmt)
        if n_scale:
            for other, n in (("x", 32768), ("residual", 32768), ("post_weight", 128), ("gate", 384), ("residual_out", 32768), ("out", n_out)):
                over("scale", n_scale, other, n, fmt)
        if fmt == 2:
            for other, n in (("x", 32768), ("pre_weight", 128), ("gate", 384), ("residual_out", 32768), ("out", n_out), ("scale", n_scale)):
                over("row_scale", 1024, other, n, fmt)


def test_row_scales_on_odd_addresses_are_refused(flib):
    """Row scales are f32: an address that is no multiple of 4 faults on the device. cudaErrorMisalignedAddress (716) before a launch."""
    Q = P + 2
    assert flib.fluke_quant_nvfp4_gpu(P, P, P, Q, 4, 64, 0) == 716
    assert flib.fluke_dequant_nvfp4_gpu(P, P, Q, P, 4, 64, 0) == 716
    assert flib.fluke_gemm_nvfp4_gpu(P, P, P, Q, P, P, P, 4, 64, 64, 0) == 716
    assert flib.fluke_gated_mlp_nvfp4_gpu(P, P, P, Q, P, P, P, P, P, P, 4, 64, 64, 0) == 716
    b = L.fluke_rmsnorm_block_t(4, 64, 0, 0, P, P + 4096, P + 8192, 0, P + 8192, 1.0, 1e-5, P + 16384, 2, P + 20480, P + 24576, P + 28674)
    assert flib.fluke_rmsnorm_block_gpu(ctypes.byref(b)) == 716


def fma32(a, b, c):
    """Correctly rounded f32 a * b + c where 64 bits hold it exactly, which the asserts of its callers' operands say."""
    return (a.astype(np.longdouble) * np.longdouble(b) + c.astype(np.longdouble)).astype(np.float32)


@pytest.mark.skipif(np.finfo(np.longdouble).nmant < 63, reason="needs 64-bit mantissas")
@pytest.mark.parametrize("divisor", [6.0] + [1 + i / 8 for i in range(8)])
def test_every_quotient_of_the_nvfp4_quantiser(divisor):
    """x / 6 and x / s with s of four significant bits, as nv_codes computes them (fp4_rows_sm100.cu: a correctly rounded reciprocal and one residual), for
    every f32 mantissa against the correctly rounded division. Exponents only shift both sides."""
    d = np.float32(divisor)
    r = np.float32(1) / d
    for part in range(8):
        x = ((np.arange(1 << 20, dtype=np.uint32) + np.uint32(part << 20)) | np.uint32(0x3F800000)).view(np.float32)
        want = x / d
        # the reciprocal's sign is turned for s, so that a zero keeps its sign; the signs of 6 are written the other way round
        q = x * r if divisor == 6 else x * -r
        residual = fma32(q, -d if divisor == 6 else d, x)
        # the residual has few bits, so its product with r and the sum with q fit 64
        assert (np.abs(residual) < 2.0 ** -20).all() and (residual * np.float32(2.0 ** 30) == np.rint(residual * np.float32(2.0 ** 30))).all()
        got = fma32(residual, r if divisor == 6 else -r, q)
        assert np.array_equal(got if divisor == 6 else -got, want)


def test_preparation_of_no_rows():
    z = torch.zeros(0, 96)
    codes, scale = prep.quantize_mxfp4(z)
    assert codes.shape == (0, 48) and scale.shape == (0, 1, 512)
    codes, scale, row = prep.quantize_nvfp4(z)
    assert codes.shape == (0, 48) and scale.shape == (0, 2, 512) and row.shape == (0,)
