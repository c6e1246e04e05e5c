"""Workloads of the 16-bit product with an epilogue, the gated linear recurrence and the norm with an
8-bit output.

  linear      out = act(x @ w^T + bias) + alpha * residual
  recurrence  h_t = f_t h_{t-1} + (1 - f_t) v_t with f = sigmoid(g), over time in either direction;
              forward (with the last state), or a training step: forward and the gradients of
              gates, values and the first state
  norm        stream = alpha * residual + x, and norm(stream) * weight as 8-bit values under a scale per row
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # Behind the attention of 32 chunks of 1000 positions; the MLP's second matrix there; one token of a
        # wider model; an odd remainder in front of a convolution's nonlinearity, read out of a wider tensor; gates of a
        # large batch, bound by arithmetic.
        {"name": "linear_32000x512x512", "kind": "linear", "type": "f16", "M": 32000, "N": 512, "K": 512, "act": "none", "bias": 1, "residual": 1, "wide": 0},
        {"name": "linear_32000x512x2048", "kind": "linear", "type": "bf16", "M": 32000, "N": 512, "K": 2048, "act": "none", "bias": 0, "residual": 1, "wide": 0},
        {"name": "linear_1x4096x4096", "kind": "linear", "type": "bf16", "M": 1, "N": 4096, "K": 4096, "act": "silu", "bias": 1, "residual": 0, "wide": 0},
        {"name": "linear_333x1536x512", "kind": "linear", "type": "f16", "M": 333, "N": 1536, "K": 512, "act": "gelu", "bias": 1, "residual": 0, "wide": 1},
        {"name": "linear_8192x8192x4096", "kind": "linear", "type": "bf16", "M": 8192, "N": 8192, "K": 4096, "act": "sigmoid", "bias": 1, "residual": 0, "wide": 0},
        # A layer over 32 chunks of 1000 steps with gates and values side by side as a product leaves them; one step
        # of a stream of 1024 chunks; one long read; training steps: a few odd chunks, batch-major, and a full batch.
        {"name": "recurrence_1000x32x512", "kind": "recurrence", "type": "f16", "T": 1000, "B": 32, "H": 512, "train": 0, "reverse": 0, "ragged": 0, "layout": "packed"},
        {"name": "recurrence_1x1024x768", "kind": "recurrence", "type": "f16", "T": 1, "B": 1024, "H": 768, "train": 0, "reverse": 0, "ragged": 0, "layout": "time"},
        {"name": "recurrence_65536x1x512", "kind": "recurrence", "type": "bf16", "T": 65536, "B": 1, "H": 512, "train": 0, "reverse": 1, "ragged": 0, "layout": "time"},
        {"name": "recurrence_train_333x7x520", "kind": "recurrence", "type": "bf16", "T": 333, "B": 7, "H": 520, "train": 1, "reverse": 0, "ragged": 1, "layout": "batch"},
        {"name": "recurrence_train_1000x256x768", "kind": "recurrence", "type": "f16", "T": 1000, "B": 256, "H": 768, "train": 1, "reverse": 1, "ragged": 0, "layout": "packed"},
        # In front of an 8-bit product: the ordinary batch, and wide activations of seven chunks of 1333.
        {"name": "norm_int8_32000x512", "kind": "norm", "type": "f16", "M": 32000, "K": 512, "format": "int8"},
        {"name": "norm_fp8_9331x2048", "kind": "norm", "type": "bf16", "M": 9331, "K": 2048, "format": "fp8"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    case = {"kind": rng.choice(("linear", "recurrence", "norm")), "type": rng.choice(("f16", "bf16"))}
    if case["kind"] == "linear":
        case |= {"M": _log(rng, 1, 32768), "N": 8 * _log(rng, 1, 1024), "K": 8 * _log(rng, 1, 1024),
                 "act": rng.choice(("none", "relu", "silu", "gelu", "tanh", "sigmoid")),
                 "bias": rng.randint(0, 1), "residual": rng.randint(0, 1), "wide": rng.randint(0, 1)}
        while case["M"] * case["N"] * case["K"] > 8192 * 8192 * 4096 or case["M"] * max(case["N"], case["K"]) > 1 << 26:
            case["M"] = (case["M"] + 1) // 2
    elif case["kind"] == "recurrence":
        case |= {"T": _log(rng, 1, 65536), "B": _log(rng, 1, 1024), "H": 8 * _log(rng, 1, 256), "train": rng.randint(0, 1),
                 "reverse": rng.randint(0, 1), "ragged": rng.randint(0, 1), "layout": rng.choice(("time", "batch", "packed"))}
        while case["T"] * case["B"] * case["H"] > 1 << 27:
            at = "B" if case["B"] > 1 and rng.random() < 0.5 else "T"
            case[at] = (case[at] + 1) // 2
    else:
        case |= {"M": _log(rng, 1, 32768), "K": 32 * _log(rng, 1, 512), "format": rng.choice(("int8", "fp8"))}
        while case["M"] * case["K"] > 1 << 25:
            case["M"] = (case["M"] + 1) // 2
    return case


# ---- states ----------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(m, k, dtype, g):
    """Normal values; a few channels of each row are larger, as in a trained model's stream."""
    gain = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return (_randn(g, m, k) * gain).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = TYPES[case["type"]], case["kind"]
    state = {"case": case, "dtype": dtype}
    if kind == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        # columns of a wider tensor (one of several outputs of the layer before) or a tensor of its own
        x = _randn(g, m, 2 * k if case["wide"] else k).to(dtype)
        state["x"] = x[:, k:] if case["wide"] else x
        state["weight"] = (_randn(g, n, k) / math.sqrt(k)).to(dtype)
        state["bias"] = (0.5 * _randn(g, n)).to(dtype) if case["bias"] else None
        state["residual"] = _randn(g, m, n).to(dtype) if case["residual"] else None
        state["alpha"] = 2.4494 if case["residual"] else 1.0
        state["act"] = None if case["act"] == "none" else case["act"]
    elif kind == "recurrence":
        t, b, h = case["T"], case["B"], case["H"]
        lead = (b, t) if case["layout"] == "batch" else (t, b)
        # channels that remember from a few steps to some thousand of them
        both = torch.empty(*lead, 2, h, dtype=dtype, device="cuda")
        both[:, :, 0] = 1.5 * _randn(g, *lead, h) + 7 * torch.rand(h, generator=g, device="cuda")
        both[:, :, 1] = _randn(g, *lead, h)
        parts = [both[:, :, 0], both[:, :, 1]]
        if case["layout"] != "packed":
            parts = [p.contiguous() for p in parts]
        if case["layout"] == "batch":
            parts = [p.transpose(0, 1) for p in parts]
        state["gate"], state["value"] = parts
        state["h0"] = 0.5 * _randn(g, b, h)
        state["reverse"] = bool(case["reverse"])
        state["lengths"] = None
        if case["ragged"]:
            lengths = 1 + (torch.rand(b, generator=g, device="cuda") * t).int()
            state["lengths"] = lengths.clamp_(max=t)
        if case["train"]:
            grad = _randn(g, *lead, h).to(dtype)
            state["grad"] = grad.transpose(0, 1) if case["layout"] == "batch" else grad
            state["grad_last"] = _randn(g, b, h)
    else:
        m, k = case["M"], case["K"]
        state["x"], state["residual"] = _activations(m, k, dtype, g), _activations(m, k, dtype, g)
        state["weight"] = (1 + 0.1 * _randn(g, k)).to(dtype)
    return state


# ---- passes ----------------------------------------------------------------------------------

def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _activation(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * _sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.erfc(v * -math.sqrt(0.5))
    if act == "tanh":
        return torch.tanh(v)
    return _sigmoid(v) if act == "sigmoid" else v


def _scan(c, b):
    """States h_t = (1 - c_t) h_{t-1} + b_t from zero, and what is left of an earlier state, as one minus it: steps are
    joined in pairs of doubling distance. One minus the product of many gates near one keeps its digits this way."""
    t, step = c.shape[0], 1
    while step < t:
        b = torch.cat((b[:step], b[step:] + b[:-step] - c[step:] * b[:-step]))
        c = torch.cat((c[:step], c[step:] + c[:-step] - c[step:] * c[:-step]))
        step *= 2
    return c, b


def _plain_recurrence(state):
    g, v, dtype = state["gate"].float(), state["value"].float(), state["dtype"]
    t, b, _ = g.shape
    inside = None
    if state["lengths"] is not None:
        inside = (torch.arange(t, device=g.device)[:, None] < state["lengths"][None, :])[..., None]
    if state["reverse"]:
        g, v = g.flip(0), v.flip(0)
        inside = None if inside is None else inside.flip(0)
    c = 1 / (1 + torch.exp(g))
    if inside is not None:
        c = torch.where(inside, c, 0.0)
    left, h = _scan(c, c * v)
    h = h + state["h0"] - left * state["h0"]
    last = h[-1]
    y = h if inside is None else torch.where(inside, h, 0.0)
    y = (y.flip(0) if state["reverse"] else y).to(dtype)
    if "grad" not in state:
        return y, last
    e = state["grad"].float()
    e = e.flip(0) if state["reverse"] else e
    if inside is not None:
        e = torch.where(inside, e, 0.0)
    e[-1] += state["grad_last"]
    # backwards in time, the gradient of step t passes through the gate of step t + 1
    after = torch.cat((torch.zeros_like(c[:1]), c[1:].flip(0)))
    _, e = _scan(after, e.flip(0))
    e = e.flip(0)
    first = e[0] - c[0] * e[0]
    before = torch.cat((state["h0"][None], h[:-1]))
    dv, dg = c * e, e * (before - v) * c * (1 - c)
    if state["reverse"]:
        dv, dg = dv.flip(0), dg.flip(0)
    return y, last, dg.to(dtype), dv.to(dtype), first


def _plain(state):
    kind, dtype = state["case"]["kind"], state["dtype"]
    if kind == "linear":
        out = state["x"].float() @ state["weight"].float().T
        if state["bias"] is not None:
            out += state["bias"].float()
        out = _activation(out, state["act"])
        if state["residual"] is not None:
            out = out + state["alpha"] * state["residual"].float()
        return out.to(dtype)
    if kind == "recurrence":
        return _plain_recurrence(state)
    stream = (state["x"].float() + state["residual"].float()).to(dtype)
    # the mean of squares in 64 bits: what is quantised behind it lies next to borders
    eps = torch.tensor(EPS, dtype=torch.float32).item()
    r = (1.0 / torch.sqrt(stream.double().square().mean(-1, keepdim=True) + eps)).float()
    h = stream.float() * r * state["weight"].float()
    most = 127.0 if state["case"]["format"] == "int8" else 448.0
    top = h.abs().amax(-1, keepdim=True).clamp_min(1e-12)
    scale = top / most
    q = (h * (most / top)).clamp(-most, most)
    if state["case"]["format"] == "int8":
        return stream, (torch.round(q) * scale).to(dtype), scale[:, 0]
    return stream, q.to(torch.float8_e4m3fn), scale[:, 0]


def _own(state):
    from fluke_b200 import ops
    kind = state["case"]["kind"]
    if kind == "linear":
        return ops.linear(state["x"], state["weight"], state["bias"], activation=state["act"], residual=state["residual"], alpha=state["alpha"])
    if kind == "recurrence":
        if "grad" not in state:
            return ops.linear_recurrence(state["gate"], state["value"], state["h0"], lengths=state["lengths"], reverse=state["reverse"])
        y, last, saved = ops.linear_recurrence(state["gate"], state["value"], state["h0"], lengths=state["lengths"], reverse=state["reverse"], save=True)
        return (y, last) + tuple(ops.linear_recurrence_backward(state["grad"], state["gate"], state["value"], saved, grad_last=state["grad_last"],
                                                                 lengths=state["lengths"], reverse=state["reverse"]))
    fmt = state["case"]["format"]
    stream, q, scale = ops.rmsnorm_block(state["x"], state["residual"], None, None, state["weight"], 1.0, EPS, quant="int8" if fmt == "int8" else "e4m3")
    if fmt == "int8":
        # the values that the codes stand for
        return stream, torch.mul(q, scale[:, None], out=torch.empty_like(stream)), scale
    return stream, q.view(torch.float8_e4m3fn), scale


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass has to do -------------------------------------------------------------------

def work(case):
    if case["kind"] == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        return {"bytes": 2 * (m * k + n * k + m * n * (1 + case["residual"]) + n * case["bias"]), "flops": 2 * m * n * k}
    if case["kind"] == "recurrence":
        n, state = case["T"] * case["B"] * case["H"], case["B"] * case["H"] * 4
        if case["train"]:
            return {"bytes": 12 * n + 4 * state, "flops": 24 * n}
        return {"bytes": 6 * n + 2 * state, "flops": 8 * n}
    m, k = case["M"], case["K"]
    return {"bytes": m * k * (7 + (3 if case["format"] == "int8" else 0)) + 4 * m + 2 * k, "flops": 10 * m * k}


# ---- the same from the definitions, in 64 bits -------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "linear":
        z = torch.matmul(state["x"].double(), state["weight"].double().t())
        if state["bias"] is not None:
            z = z + state["bias"].double()
        act = state["act"]
        if act == "relu":
            z = torch.where(z > 0, z, 0.0)
        elif act == "silu":
            z = z * torch.sigmoid(z)
        elif act == "gelu":
            z = z * torch.special.ndtr(z)
        elif act == "tanh":
            z = torch.tanh(z)
        elif act == "sigmoid":
            z = torch.sigmoid(z)
        return z if state["residual"] is None else z + state["alpha"] * state["residual"].double()
    if case["kind"] == "recurrence":
        f, v = torch.sigmoid(state["gate"].double()), state["value"].double()
        t = f.shape[0]
        lengths = state["lengths"]
        order = range(t - 1, -1, -1) if state["reverse"] else range(t)
        h = state["h0"].double()
        y, before = torch.zeros_like(v), torch.zeros_like(v)
        for i in order:
            before[i] = h
            new = f[i] * h + (1 - f[i]) * v[i]
            if lengths is None:
                y[i] = h = new
            else:
                live = (lengths > i)[:, None]
                y[i] = torch.where(live, new, 0.0)
                h = torch.where(live, new, h)
        if not case["train"]:
            return y, h
        e = state["grad_last"].double()
        dg, dv = torch.zeros_like(v), torch.zeros_like(v)
        for i in reversed(order):
            live = None if lengths is None else (lengths > i)[:, None]
            here = state["grad"][i].double() + e
            if live is not None:
                here = torch.where(live, here, 0.0)
            dv[i] = here * (1 - f[i])
            dg[i] = here * (before[i] - v[i]) * f[i] * (1 - f[i])
            e = here * f[i] if live is None else torch.where(live, here * f[i], e)
        return y, h, dg, dv, e
    # the stream is kept in 16 bits, and the norm is of what is kept
    stream = state["x"].double() + state["residual"].double()
    kept = stream.to(state["dtype"]).double()
    h = kept / torch.sqrt((kept * kept).sum(1, keepdim=True) / kept.shape[1] + EPS) * state["weight"].double()
    most = 127 if case["format"] == "int8" else 448
    scale = torch.clamp(h.abs().max(1, keepdim=True).values, min=1e-12) / most
    if case["format"] == "int8":
        return stream, torch.round(h / scale) * scale, scale[:, 0]
    return stream, (h / scale).float().to(torch.float8_e4m3fn).double(), scale[:, 0]
