"""Input and weight preparation that the reference does in torch, outside the hot path:
symmetric quantisers, rotary tables, fp8 weight pre-shuffle. These run on whatever device the
tensors are on; none of them is a GPU kernel of the library.
"""
import torch

E4M3_MAX = 448.0


def quantize_int8_rows(t, dim=-1):
    """Symmetric per-row int8 (amax/127): returns (int8, f32 dequant scale).
    Restates cute/common.py:63-69 of the reference (scale = 1/(127/amax))."""
    qm = 127
    fr = t.abs().amax(dim=dim).clamp_min(1e-8)
    qs = qm / fr
    ti = (t * qs.unsqueeze(dim)).round().clamp(-qm, qm).to(torch.int8)
    return ti, qs.to(torch.float32).reciprocal()


def quantize_fp8_rows(t):
    """Per-row e4m3 (amax/448): returns (float8_e4m3fn, f32 scale [rows]).
    Restates fp8_quantize_per_token, fly/rdna4/gemm/rdna_fp8_preshuffle_gemm.py:57-70."""
    amax = t.abs().amax(dim=-1, keepdim=True).clamp(min=1e-12)
    scale = amax / E4M3_MAX
    q = (t / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q, scale.squeeze(-1).to(torch.float32)


def preshuffle_fp8_weight(w_nk):
    """Row-major [N, K] e4m3 weight -> the [N/16, K/16, 2, 16, 8] byte layout the fp8 ABI takes
    (preshuffle_b_fp8 of fly/rdna4/gemm/rdna_fp8_preshuffle_gemm.py:40-54 applied to w^T)."""
    n, k = w_nk.shape
    assert n % 16 == 0 and k % 16 == 0
    b = w_nk.view(torch.uint8).reshape(n // 16, 16, k // 16, 2, 8)  # n0, nl, k0, kl, kp
    return b.permute(0, 2, 3, 1, 4).contiguous()


def rotary_tables(seq_len, head_dim=64, theta=10000.0, device="cpu"):
    """(sin, cos) f32 [seq_len, head_dim/2] built in f64 like test/test_rotary_gpu.py:53-58."""
    inv_freq = torch.pow(theta, torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim).reciprocal()
    freqs = torch.outer(torch.arange(seq_len, dtype=torch.float64), inv_freq)
    return (torch.sin(freqs).to(torch.float32).contiguous().to(device),
            torch.cos(freqs).to(torch.float32).contiguous().to(device))


# ---- microscaled 4-bit floating point (the formats of fluke.h, part 6) ------------------------

def _e2m1(v):
    """Codes of the nearest E2M1 values, ties to the even code, saturating at 6."""
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=v.dtype, device=v.device)
    m = v.abs()
    code = torch.bucketize(m, bounds, right=False)     # values on a bound go down ...
    up = torch.isin(m, bounds[1::2])                   # ... and up where the code above is the even one
    return (code + up).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)


def _fp4_tiles(scale):
    """[rows, blocks] bytes -> [ceil(rows / 128), ceil(blocks / 4), 512], zeros where there is no block."""
    rows, blocks = scale.shape
    t = torch.zeros(-(-rows // 128) * 128, -(-blocks // 4) * 4, dtype=torch.uint8, device=scale.device)
    t[:rows, :blocks] = scale
    return t.view(-1, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(t.shape[0] // 128, t.shape[1] // 4, 512).contiguous()


def _fp4_blocks(t, size):
    rows, cols = t.shape
    if cols % 32 != 0:
        raise ValueError(f"{cols} columns: 4-bit formats need a multiple of 32")
    b = t.float().reshape(rows, cols // size, size)
    return b, torch.isfinite(b).all(-1)


def quantize_mxfp4(t):
    """[rows, cols] of any float type -> (codes uint8 [rows, cols / 2], block scales in tiles): what
    ops.quant_mxfp4 gives for 16-bit rows, on any device."""
    b, ok = _fp4_blocks(t, 32)
    amax = torch.where(ok, b.abs().amax(-1), 0.0)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp_(-127, 127)
    factor = ((127 - e) << 23).to(torch.int32).view(torch.float32)   # e is at most 126 below the largest f32
    q = torch.where(ok[..., None], _e2m1(torch.where(ok[..., None], b, 0.0) * factor[..., None]), 0).flatten(1)
    return q[:, 0::2] | (q[:, 1::2] << 4), _fp4_tiles(torch.where(ok, e + 127, 255).to(torch.uint8))


def quantize_nvfp4(t):
    """[rows, cols] of any float type -> (codes, block scales in tiles, row scales f32 [rows]): what
    ops.quant_nvfp4 gives for 16-bit rows, on any device."""
    b, ok = _fp4_blocks(t, 16)
    ok = ok.all(-1)
    b = torch.where(ok[:, None, None], b, 0.0)
    amax = b.abs().amax(-1)
    top = amax.amax(-1)
    f, e = torch.frexp(top)
    e = torch.where(f <= 0.65625, e - 12, e - 11).clamp_min(-100)   # 2688 = 0.65625 * 2^12
    g = torch.where(top > 0, ((e + 127) << 23).to(torch.int32).view(torch.float32), 1.0)
    s8 = (amax / (6.0 * g)[:, None]).to(torch.float8_e4m3fn)
    s = (s8.float() * g[:, None])[..., None]
    q = torch.where((s > 0) & ok[:, None, None], _e2m1(torch.where(s > 0, b / s, 0.0)), 0).flatten(1)
    scale = torch.where(ok[:, None], s8.view(torch.uint8), 0x7F)
    return q[:, 0::2] | (q[:, 1::2] << 4), _fp4_tiles(scale), torch.where(ok, g, float("nan"))
