"""Workloads of the 4-bit floating-point operators and of the fused norms around a block.

Four kinds of pass, each at several sizes, in the two formats (`mx`: blocks of 32 under a power of
two, `nv`: blocks of 16 under an e4m3 scale and a power of two per row) and the two activation types:

  quant   rows are quantised and read back (what a consumer of the stored values sees)
  gemm    out = a @ b^T of two quantised matrices
  gated   out = silu(a @ gate^T) * (a @ up^T)
  norm    a block's output is normalised, gated and added to the scaled residual stream, and the
          stream is normalised for the next block, plain or quantised (and read back)

Scales of quantised matrices lie in tiles of 128 rows x 4 blocks: block c of row r is byte
(r % 32) * 16 + (r / 32 % 4) * 4 + c % 4 of tile (r / 128, c / 4).
"""
import math

import torch

own = False

BLOCK = {"mx": 32, "nv": 16}
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
ALPHA, EPS = 0.75, 1e-5
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # The residual stream of a batch of 32 chunks of 1000 positions, in front of a product of
        # its own, and the wide hidden activations of seven chunks of 1333.
        {"name": "quant_mx_32000x512", "kind": "quant", "format": "mx", "type": "f16", "M": 32000, "K": 512},
        {"name": "quant_nv_9331x2048", "kind": "quant", "format": "nv", "type": "bf16", "M": 9331, "K": 2048},
        # Between two blocks: the ordinary batch with a gate per channel; one token of a wider
        # model; chunks that carry a gate each, where the next block takes 16-bit input.
        {"name": "norm_mx_32000x512", "kind": "norm", "format": "mx", "type": "f16", "M": 32000, "K": 512, "seq": 0},
        {"name": "norm_nv_1x4096", "kind": "norm", "format": "nv", "type": "bf16", "M": 1, "K": 4096, "seq": 1},
        {"name": "norm_plain_9331x1024", "kind": "norm", "format": "none", "type": "f16", "M": 9331, "K": 1024, "seq": 1333},
        # Products: QKV of the ordinary batch; one token (weights are all there is to read); an
        # odd remainder against the second matrix of the MLP; the largest, bound by arithmetic.
        {"name": "gemm_mx_32000x1536x512", "kind": "gemm", "format": "mx", "type": "f16", "M": 32000, "N": 1536, "K": 512},
        {"name": "gemm_nv_1x4096x4096", "kind": "gemm", "format": "nv", "type": "bf16", "M": 1, "N": 4096, "K": 4096},
        {"name": "gemm_mx_333x512x2048", "kind": "gemm", "format": "mx", "type": "f16", "M": 333, "N": 512, "K": 2048},
        {"name": "gemm_nv_8192x8192x4096", "kind": "gemm", "format": "nv", "type": "bf16", "M": 8192, "N": 8192, "K": 4096},
        # The gated MLP: the ordinary batch, five tokens of a wider model, and a ragged prompt of it.
        {"name": "gated_mx_32000x2048x512", "kind": "gated", "format": "mx", "type": "f16", "M": 32000, "N": 2048, "K": 512},
        {"name": "gated_mx_5x8192x4096", "kind": "gated", "format": "mx", "type": "bf16", "M": 5, "N": 8192, "K": 4096},
        {"name": "gated_nv_1803x4096x2048", "kind": "gated", "format": "nv", "type": "bf16", "M": 1803, "N": 4096, "K": 2048},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("quant", "norm", "gemm", "gated"))
    case = {"kind": kind, "format": rng.choice(("mx", "nv")), "type": rng.choice(("f16", "bf16")),
            "M": _log(rng, 1, 32768), "K": 32 * _log(rng, 2, 256)}
    if kind in ("gemm", "gated"):
        case["N"] = 8 * _log(rng, 8, 1024)
        while (2 if kind == "gated" else 1) * case["M"] * case["N"] * case["K"] > 8192 * 8192 * 4096 or case["M"] * max(case["N"], case["K"]) > 1 << 26:
            case["M"] = (case["M"] + 1) // 2
    else:
        while case["M"] * case["K"] > 1 << 25:
            case["M"] = (case["M"] + 1) // 2
        if kind == "norm":
            case["format"] = rng.choice(("mx", "nv", "none"))
            case["seq"] = rng.choice((0, rng.randint(1, case["M"])))
    return case


# ---- the format, in elementary operations ----------------------------------------------------

def _blocks(x, fmt):
    return x.unflatten(-1, (-1, BLOCK[fmt]))


def _round_e2m1(v):
    """Nearest E2M1 value, ties to the even code, saturating at 6; also the code."""
    m = v.abs()
    code = (m > 0.25).to(torch.uint8)
    code += m >= 0.75
    code += m > 1.25
    code += m >= 1.75
    code += m > 2.5
    code += m >= 3.5
    code += m > 5.0
    code |= torch.signbit(v).to(torch.uint8) << 3
    return code


def _table(device, dtype=torch.float32):
    t = torch.tensor(E2M1, dtype=dtype, device=device)
    return torch.cat((t, -t))


def _power(e, dtype=torch.float32):
    """2^e of whole numbers -127 .. 127, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64).to(dtype)


def _quantise(x, fmt):
    """x f32 [M, K] -> codes [M, K / B, B], block scales as bytes [M, K / B], row scales f32 [M] or None."""
    b = _blocks(x, fmt)
    amax = b.abs().amax(-1)
    if fmt == "mx":
        e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp_(-127, 127)
        return _round_e2m1(b * _power(-e)[..., None]), (e + 127).to(torch.uint8), None
    top = amax.amax(-1)
    f, e = torch.frexp(top)
    g = torch.where(top > 0, _power(torch.where(f <= 0.65625, e - 12, e - 11).clamp_min(-100)), 1.0)
    s8 = (amax / (6.0 * g)[:, None]).to(torch.float8_e4m3fn)
    s = (s8.float() * g[:, None])[..., None]
    return _round_e2m1(torch.where(s > 0, b / s, torch.copysign(torch.zeros_like(b), b))), s8.view(torch.uint8), g


def _scale_values(scale, fmt, dtype=torch.float32):
    if fmt == "mx":
        return _power(scale.long() - 127, dtype)
    return scale.view(torch.float8_e4m3fn).to(dtype)


def _read_back(codes, scale, row_scale, fmt, dtype):
    v = _table(codes.device)[codes.int()] * _scale_values(scale, fmt)[..., None]
    v = v.flatten(-2)
    return (v if row_scale is None else v * row_scale[:, None]).to(dtype)


def _pack(codes, scale, row_scale):
    """Two codes a byte, the lower of a pair in the low half; scales in tiles of 128 rows x 4 blocks."""
    c = codes.flatten(-2)
    m, k = c.shape
    rows, blocks = -(-m // 128) * 128, -(-scale.shape[1] // 4) * 4
    t = torch.zeros(rows, blocks, dtype=torch.uint8, device=c.device)
    t[:m, :scale.shape[1]] = scale
    t = t.view(rows // 128, 4, 32, blocks // 4, 4).permute(0, 3, 2, 1, 4).reshape(rows // 128, blocks // 4, 512)
    return c[:, 0::2] | (c[:, 1::2] << 4), t.contiguous(), row_scale


def _unpack(packed, fmt, dtype=torch.float32):
    codes, tiles, row_scale = packed
    m, k = codes.shape[0], 2 * codes.shape[1]
    v = _table(codes.device, dtype)[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    t = tiles.view(tiles.shape[0], tiles.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)
    v = (_blocks(v, fmt) * _scale_values(t[:m, :k // BLOCK[fmt]], fmt, dtype)[..., None]).flatten(-2)
    return v if row_scale is None else v * row_scale.to(dtype)[:, None]


# ---- states ----------------------------------------------------------------------------------

def _activations(m, k, dtype, g):
    """Normal values; a few channels of each row are larger, as in a trained model's stream."""
    x = torch.randn(m, k, generator=g, device="cuda")
    gain = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return (x * gain).to(dtype)


def _weight(n, k, g):
    return torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, m, k, fmt = TYPES[case["type"]], case["M"], case["K"], case["format"]
    state = {"case": case, "dtype": dtype, "format": fmt}
    if case["kind"] == "quant":
        state["x"] = _activations(m, k, dtype, g)
    elif case["kind"] == "norm":
        gates = 1 if case["seq"] == 0 else -(-m // case["seq"])
        state["x"] = _activations(m, k, dtype, g)
        state["residual"] = _activations(m, k, dtype, g)
        state["post"] = (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(dtype)
        state["pre"] = (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(dtype)
        state["gate"] = (0.5 * torch.randn(gates, k, generator=g, device="cuda")).to(dtype)
        state["seq"] = case["seq"]
    else:
        def packed(x):
            return _pack(*_quantise(x.float(), fmt))
        state["a"] = packed(_activations(m, k, dtype, g))
        state["b"] = packed(_weight(case["N"], k, g))
        if case["kind"] == "gated":
            state["up"] = packed(_weight(case["N"], k, g))
    return state


# ---- passes ----------------------------------------------------------------------------------

def _norm(v, weight):
    # the mean of squares in 64 bits: what is quantised behind it lies next to borders
    eps = torch.tensor(EPS, dtype=torch.float32).item()
    r = (1.0 / torch.sqrt(v.double().square().mean(-1, keepdim=True) + eps)).float()
    return v.float() * r * weight.float()


def _plain(state):
    kind, dtype, fmt = state["case"]["kind"], state["dtype"], state["format"]
    if kind == "quant":
        return _read_back(*_quantise(state["x"].float(), fmt), fmt, dtype)
    if kind == "norm":
        gate, m = state["gate"].float(), state["x"].shape[0]
        if state["seq"] > 0:
            gate = gate[torch.arange(m, device=gate.device) // state["seq"]]
        y = (ALPHA * state["residual"].float() + gate * _norm(state["x"], state["post"])).to(dtype)
        h = _norm(y, state["pre"])
        return y, h.to(dtype) if fmt == "none" else _read_back(*_quantise(h, fmt), fmt, dtype)
    a = _unpack(state["a"], fmt)
    out = a @ _unpack(state["b"], fmt).T
    if kind == "gated":
        out = out / (1 + torch.exp(-out)) * (a @ _unpack(state["up"], fmt).T)
    return out.to(dtype)


def _own(state):
    from fluke_b200 import ops
    kind, dtype, fmt = state["case"]["kind"], state["dtype"], state["format"]
    if kind == "quant":
        if fmt == "mx":
            return ops.dequant_mxfp4(*ops.quant_mxfp4(state["x"]), dtype=dtype)
        return ops.dequant_nvfp4(*ops.quant_nvfp4(state["x"]), dtype=dtype)
    if kind == "norm":
        quant = {"mx": "mxfp4", "nv": "nvfp4", "none": None}[fmt]
        y, *h = ops.rmsnorm_block(state["x"], state["residual"], state["post"], state["gate"], state["pre"], ALPHA, EPS,
                                  seqlen=state["seq"], quant=quant)
        if fmt == "none":
            return y, h[0]
        return y, (ops.dequant_mxfp4 if fmt == "mx" else ops.dequant_nvfp4)(*h, dtype=dtype)
    a, b = state["a"], state["b"]
    if fmt == "mx":
        if kind == "gemm":
            return ops.gemm_mxfp4(*a[:2], *b[:2], dtype=dtype)
        return ops.gated_mlp_mxfp4(*a[:2], *b[:2], *state["up"][:2], dtype=dtype)
    if kind == "gemm":
        return ops.gemm_nvfp4(*a, *b, dtype=dtype)
    return ops.gated_mlp_nvfp4(*a, *b, *state["up"], dtype=dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass has to do -------------------------------------------------------------------

def work(case):
    m, k, fmt = case["M"], case["K"], case["format"]
    # bytes a value of the format takes, with its share of the scales
    held = 2.0 if fmt == "none" else 0.5 + 1.0 / BLOCK[fmt] + (4.0 / k if fmt == "nv" else 0.0)
    if case["kind"] == "quant":
        return {"bytes": m * k * (4 + 2 * held), "flops": 6 * m * k}
    if case["kind"] == "norm":
        gates = 1 if case["seq"] == 0 else -(-m // case["seq"])
        back = 0.0 if fmt == "none" else held + 2
        return {"bytes": m * k * (6 + held + back) + 2 * k * (2 + gates), "flops": 14 * m * k}
    n, weights = case["N"], 2 if case["kind"] == "gated" else 1
    return {"bytes": held * k * (m + weights * n) + 2 * m * n, "flops": 2 * weights * m * n * k}


# ---- the same from the definitions, in 64 bits -------------------------------------------------

def _nearest(v):
    """The E2M1 value nearest to v, ties to the value whose last mantissa bit is zero."""
    m = v.abs().clamp(max=6.0)
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return torch.copysign(torch.round(m / step) * step, v)


def _quantised64(h, fmt):
    size = BLOCK[fmt]
    b = h.reshape(h.shape[0], -1, size)
    top = b.abs().max(dim=2, keepdim=True).values
    if fmt == "mx":
        # exponent of the largest power of two not above the block's maximum
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -130)))
        e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double()
        step = torch.exp2((e - 2).clamp(-127, 127))
    else:
        # the least power of two under which the row's largest value needs no block scale above 448
        largest = h.abs().max(dim=1).values[:, None, None]
        least = torch.ceil(torch.log2(largest.clamp_min(2.0 ** -100) / (6 * 448)))
        least = least - (largest <= 6 * 448 * torch.exp2(least - 1)).double() + (largest > 6 * 448 * torch.exp2(least)).double()
        row = torch.where(largest > 0, torch.exp2(least.clamp_min(-100)), 1.0)
        step = (top / 6 / row).to(torch.float8_e4m3fn).double() * row
    q = torch.where(step > 0, _nearest(b / step.clamp_min(1e-300)), 0.0)
    return (q * step).reshape(h.shape)


def _matrix64(packed, fmt):
    codes, tiles, row_scale = packed
    m, half = codes.shape
    low, high = (codes & 15).long(), (codes >> 4).long()
    value = torch.tensor([(-1.0 if c & 8 else 1.0) * E2M1[c & 7] for c in range(16)], dtype=torch.float64, device=codes.device)
    v = torch.empty(m, 2 * half, dtype=torch.float64, device=codes.device)
    v[:, 0::2], v[:, 1::2] = value[low], value[high]
    r = torch.arange(m, device=codes.device)[:, None]
    c = torch.arange(2 * half // BLOCK[fmt], device=codes.device)[None, :]
    at = ((r // 128) * tiles.shape[1] + c // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4
    s = tiles.flatten()[at]
    s = torch.exp2(s.double() - 127) if fmt == "mx" else s.view(torch.float8_e4m3fn).double()
    v *= s.repeat_interleave(BLOCK[fmt], dim=1)
    return v if row_scale is None else v * row_scale.double()[:, None]


def exact(case, seed):
    state = prepare(case, seed)
    fmt = case["format"]
    if case["kind"] == "quant":
        return _quantised64(state["x"].double(), fmt)
    if case["kind"] == "norm":
        def unit(v):
            return v / torch.sqrt((v * v).sum(dim=1, keepdim=True) / v.shape[1] + EPS)
        x, res = state["x"].double(), state["residual"].double()
        gate = state["gate"].double()
        if case["seq"] > 0:
            gate = gate.repeat_interleave(case["seq"], dim=0)[:x.shape[0]]
        y = ALPHA * res + gate * (unit(x) * state["post"].double())
        # the stream is kept in 16 bits, and the next norm is of what is kept
        h = unit(y.to(state["dtype"]).double()) * state["pre"].double()
        return y, h if fmt == "none" else _quantised64(h, fmt)
    a = _matrix64(state["a"], fmt)
    p = torch.matmul(a, _matrix64(state["b"], fmt).t())
    if case["kind"] == "gated":
        p = p * torch.sigmoid(p) * torch.matmul(a, _matrix64(state["up"], fmt).t())
    return p
