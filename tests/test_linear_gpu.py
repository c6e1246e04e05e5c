"""16-bit products with an epilogue on the GPU, through fluke_b200.ops, against 64-bit products of the same values.

Tolerance: half a step of the type, the bound K 2^-24 sum |x w| of an f32 sum times the largest slope of the activation (1.13), roundings of what follows (4 * 2^-24 of
each term) and the activations' own errors: 2^-16 of the value (gelu 8e-6, tanh 2^-16 at its change of form, the others (|v| + 5) 2^-23 for |v| up to 100)."""
import ctypes

import numpy as np
import pytest
import torch

from fluke_b200 import lib as L, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
ACTS = [None, "relu", "silu", "gelu", "tanh", "sigmoid"]


def act64(v, act):
    return {None: lambda: v, "relu": lambda: v.clamp_min(0), "silu": lambda: v / (1 + torch.exp(-v)), "gelu": lambda: 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5),
            "tanh": lambda: torch.tanh(v), "sigmoid": lambda: 1 / (1 + torch.exp(-v))}[act]()


def check(got, x, w, bias=None, act=None, res=None, alpha=1.0):
    x, w = x.double(), w.double()
    z, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs() / max(1, x.shape[1])
    want = act64(z, act)
    err = 1.13 * (x.shape[1] + 4) * 2.0 ** -24 * size + (0 if act in (None, "relu") else 2.0 ** -16) * want.abs()
    if res is not None:
        want = want + alpha * res.double()
        err = err + 4 * 2.0 ** -24 * (want.abs() + abs(alpha) * res.double().abs())
    tol = (want.abs() + err) * (torch.finfo(got.dtype).eps / 2) + 2.0 ** -25 + err
    d = (got.double() - want).abs()
    assert (d <= tol).all(), f"off by {d.max().item()}, {(d / tol).max().item()} of the tolerance"


def tensors(g, m, n, k, dtype):
    t = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return t(m, k).to(dtype), (t(n, k) / k ** 0.5).to(dtype), (0.5 * t(n)).to(dtype), t(m, n).to(dtype)


SIZES = [(1, 8, 8), (1, 4096, 4096), (5, 24, 40), (16, 512, 1024), (17, 136, 72), (33, 1544, 200), (64, 512, 512), (130, 1536, 512), (333, 520, 2048), (1000, 2048, 512),
         (4097, 256, 64), (300, 72, 8192), (2600, 1032, 520), (9331, 1536, 96), (20000, 512, 512), (3000, 4104, 1032)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, dtype):
    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x, w, bias, res = tensors(g, m, n, k, TYPES[dtype])
    i = (m + n + k) % 6
    check(ops.linear(x, w), x, w)
    check(ops.linear(x, w, bias, activation=ACTS[i], residual=res, alpha=-1.5), x, w, bias, ACTS[i], res, -1.5)
    j = (i + 1 + (dtype == "bf16")) % 6
    check(ops.linear(x, w, activation=ACTS[j], residual=res), x, w, None, ACTS[j], res)
    check(ops.linear(x, w, bias, ACTS[(j + 1) % 6]), x, w, bias, ACTS[(j + 1) % 6])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 3000])
def test_activations_over_their_range(m, act):
    """Products that are single values, over the whole range of f16 and zero."""
    v = torch.cat((torch.linspace(-12, 12, 3001), torch.logspace(-7, 4.8, 3001), -torch.logspace(-7, 4.8, 3001), torch.zeros(1))).half()
    v = v[torch.isfinite(v)]
    n = 8 * (len(v) // 8)
    w = torch.zeros(n, 8, dtype=torch.float16)
    w[:, 0] = v[:n]
    x = torch.zeros(m, 8, dtype=torch.float16)
    x[:, 0] = 1
    x, w = x.to(DEV), w.to(DEV)
    check(ops.linear(x, w, activation=act), x, w, act=act)


@pytest.mark.parametrize("m,n,k", [(3, 64, 128), (150, 264, 72), (5000, 520, 136)])
def test_columns_of_wider_tensors(m, n, k):
    """Inputs and output are columns of wider tensors, whose other columns nothing reads (NaN) or writes."""
    g = torch.Generator(device=DEV).manual_seed(m)
    x, w, bias, res = tensors(g, m, n, k, torch.float16)
    wide = torch.full((m, k + 24), float("nan"), dtype=torch.float16, device=DEV)
    wide[:, 8:8 + k] = x
    both = torch.full((m, 2 * n + 8), float("nan"), dtype=torch.float16, device=DEV)
    both[:, :n] = res
    out = both[:, n:2 * n]
    got = ops.linear(wide[:, 8:8 + k], w, bias, "silu", both[:, :n], 0.5, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, ops.linear(x, w, bias, "silu", res, 0.5))
    assert torch.equal(both[:, :n], res) and both[:, 2 * n:].isnan().all()
    check(out, x, w, bias, "silu", res, 0.5)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 512), (200, 512, 2048), (9000, 512, 512)])
def test_in_place_on_the_residual(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    x, w, bias, res = tensors(g, m, n, k, torch.bfloat16)
    want = ops.linear(x, w, bias, None, res, 2.5)
    got = ops.linear(x, w, bias, None, res, 2.5, out=res)
    assert got.data_ptr() == res.data_ptr() and torch.equal(got, want)


def test_infinities_and_nans():
    x = torch.zeros(3, 8, dtype=torch.float16, device=DEV)
    x[0, 0], x[1, 0], x[2, 0] = float("inf"), float("-inf"), float("nan")
    w = torch.zeros(8, 8, dtype=torch.float16, device=DEV)
    w[:, 0] = 1
    for act, high, low in ((None, float("inf"), float("-inf")), ("relu", float("inf"), 0.0), ("tanh", 1.0, -1.0), ("sigmoid", 1.0, 0.0), ("silu", float("inf"), None), ("gelu", float("inf"), None)):
        y = ops.linear(x, w, activation=act)
        assert (y[0] == high).all() and (y[1].isnan().all() if low is None else (y[1] == low).all()) and y[2].isnan().all(), act
    big = torch.full((1, 8), 60000.0, dtype=torch.float16, device=DEV)
    assert (ops.linear(big, w) == 60000).all() and ops.linear(big, w * 2).isinf().all()


@pytest.mark.parametrize("m,n,k", [(1, 1024, 4096), (70, 512, 2048), (6000, 1024, 256)])
def test_the_same_bits_every_time_and_replayed(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    x, w, bias, res = tensors(g, m, n, k, torch.float16)
    want = ops.linear(x, w, bias, "gelu", res)
    assert all(torch.equal(ops.linear(x, w, bias, "gelu", res), want) for _ in range(5))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ops.set_stream(stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            a = ops.linear(x, w, bias, "gelu", res)
            b = ops.linear(a, a[:8].contiguous()) if m >= 8 else a
    finally:
        ops.set_stream(None)
    x.copy_(x.flip(0) * 0.5)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    want = ops.linear(x, w, bias, "gelu", res)
    assert torch.equal(a, want) and (m < 8 or torch.equal(b, ops.linear(want, want[:8].contiguous())))


def test_empty_and_refusals():
    t = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)
    assert ops.linear(t(0, 64), t(16, 64)).shape == (0, 16)
    x, w = t(4, 64), t(16, 64)
    for call in (lambda: ops.linear(x, t(16, 72)), lambda: ops.linear(x, t(12, 64)), lambda: ops.linear(t(4, 60), t(16, 60)), lambda: ops.linear(x, w.bfloat16()),
                 lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w, t(8)), lambda: ops.linear(x, w, residual=t(4, 8)), lambda: ops.linear(x, w, out=t(4, 8)),
                 lambda: ops.linear(x, w, activation="swish"), lambda: ops.linear(t(64, 4).T, w), lambda: ops.linear(x[0], w)):
        with pytest.raises(ValueError):
            call()
    shared = t(8, 64)
    for call in (lambda: ops.linear(t(4, 68)[:, :64], w), lambda: ops.linear(t(1, 64).expand(4, 64), w), lambda: ops.linear(t(4 * 64 + 1)[1:].view(4, 64), w),
                 lambda: ops.linear(shared[:4, :64], t(64, 64), out=shared[2:6]), lambda: ops.linear(x, t(64, 64), residual=shared[:4], out=shared[1:5]),
                 lambda: ops.linear(x, t(64, 64), out=x)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError):
        ops.linear(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError):
        ops.linear(x, t(64, 16).T)


def test_run_of_a_recurrent_block():
    """Gate and candidate from one product, the recurrence over views of it, the product back onto the stream, and the norm that
    feeds an 8-bit product of the next layer: a step as a layer makes it, against the same in 64 bits from the rounded intermediates."""
    g = torch.Generator(device=DEV).manual_seed(11)
    t, b, h = 130, 5, 512
    stream = torch.randn(t * b, h, generator=g, device=DEV).half()
    w_in, w_out = (torch.randn(2 * h, h, generator=g, device=DEV) / h ** 0.5).half(), (torch.randn(h, h, generator=g, device=DEV) / h ** 0.5).half()
    bias = torch.cat((torch.full((h,), 3.0), torch.zeros(h))).half().to(DEV)
    weight = (1 + 0.1 * torch.randn(h, generator=g, device=DEV)).half()
    both = ops.linear(stream, w_in, bias)
    check(both, stream, w_in, bias)
    gate, value = both.view(t, b, 2 * h).chunk(2, -1)
    y, last = ops.linear_recurrence(gate, value)
    from oracle import recurrence as ref
    want = ref.forward(gate.cpu().double().numpy(), value.cpu().double().numpy())[0]
    assert np.abs(y.cpu().double().numpy() - want).max() <= np.abs(want).max() * 2.0 ** -11 + 2.0 ** -14 * 4
    out = ops.linear(y.view(t * b, h), w_out, residual=stream, alpha=0.5)
    check(out, y.view(t * b, h), w_out, None, None, stream, 0.5)
    kept, q, s = ops.rmsnorm_block(y.view(t * b, h), out, None, None, weight, 1.0, 1e-5, quant="int8")
    w8 = torch.randint(-127, 128, (128, h), generator=g, device=DEV, dtype=torch.int8)
    sb = torch.rand(128, generator=g, device=DEV) / 1000
    p = ops.gemm_i8(q, w8, s, sb)
    exact = (q.double() @ w8.double().T) * (s.double()[:, None] * sb.double())
    assert ((p.double() - exact).abs() <= exact.abs() * (2.0 ** -11 + 2.0 ** -22) + 2.0 ** -25).all()


def test_more_than_2_pow_31_values():
    """Offsets beyond 32 bits in the output, the residual and x."""
    m, n, k = 270000, 8192, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float16)
    w, res = new(n, k), new(m, n)
    wide = new(m, 8192)
    x = wide[:, 5000:5000 + k]
    assert res.numel() > 1 << 31
    out = ops.linear(x, w, residual=res, alpha=0.5)
    rows = slice(m - 300, m)
    check(out[rows], x[rows], w, None, None, res[rows], 0.5)
    check(out[:300], x[:300], w, None, None, res[:300], 0.5)
