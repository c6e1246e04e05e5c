"""Gated linear recurrence and its gradients on the GPU, through fluke_b200.ops, against oracle/recurrence.py.

Tolerances. A state is a mean of the first state and the values, so no state and no difference of a state and a value is above
M = 2 max(|h0|, |v|). A step h += c (v - h) rounds three times, 3 * 2^-24 M at most, and is taken with a c that is (|g| + 8) 2^-24 of
itself off; a rounding fades with the gates behind it, so at most n = min(T, 1 / min c) of them add up, and an error of c, which moves h
by that part of c (v - h), adds up to as much of M. Joining runs is a step of the same kind per run and tile, fewer than T / 4 + 8. Together
    E = M 2^-24 (4 n + |g|max + 32)
for states, and the same with the largest |e| in the place of M for the gradients that go back. To that comes half a step of the type."""
import ctypes

import numpy as np
import pytest
import torch

from fluke_b200 import lib as L, ops
from oracle import recurrence as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def n64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def steps(g, layout, t, b, h, dtype):
    """gate and value as a caller has them: of their own, batch-major, or columns of a wider tensor."""
    lead = (b, t) if layout == "batch" else (t, b)
    both = torch.stack((1.5 * torch.randn(*lead, h, generator=g) + 8 * torch.rand(h, generator=g) - 1, torch.randn(*lead, h, generator=g)), 2).to(dtype).to(DEV)
    parts = [both[:, :, 0], both[:, :, 1]]
    if layout != "packed":
        parts = [p.contiguous() for p in parts]
    return [p.transpose(0, 1) if layout == "batch" else p for p in parts]


def bounds(gate, value, h0):
    g = n64(gate)
    c = ref.sigmoid(-g)
    n = min(g.shape[0], 1 / c.min()) if g.size else 1
    most = 2 * max(np.abs(n64(value)).max(), 0 if h0 is None else np.abs(n64(h0)).max())
    return most, 2.0 ** -24 * (4 * n + np.abs(g).max() + 32)


def half(want, dtype):
    return np.abs(want) * (torch.finfo(dtype).eps / 2) + 2.0 ** -25


def near(got, want, tol):
    d = np.abs(n64(got) - want)
    assert (d <= tol).all(), f"off by {d.max()}, {(d / np.maximum(tol, 1e-300)).max()} of the tolerance, at {np.unravel_index((d / np.maximum(tol, 1e-300)).argmax(), d.shape)}"


SIZES = [(1, 1, 2), (1, 5, 64), (7, 3, 66), (8, 2, 32), (9, 2, 30), (17, 300, 34), (63, 1, 64), (64, 2, 128), (65, 2, 130), (200, 3, 520), (1000, 2, 64),
         (4097, 1, 34), (333, 7, 520), (1161, 1, 512), (20000, 1, 64), (520, 40, 256), (50, 130, 136), (35, 700, 96), (100, 1030, 72), (3000, 2, 40), (1100, 5, 264), (1500, 8, 328)]


@pytest.mark.parametrize("t,b,h", SIZES)
@pytest.mark.parametrize("dtype,layout,reverse,ragged", [("f16", "time", False, False), ("bf16", "packed", True, True), ("f16", "batch", True, False), ("bf16", "time", False, True)])
def test_forward_and_gradients(t, b, h, dtype, layout, reverse, ragged):
    g = torch.Generator().manual_seed(t * 7 + b + h)
    dtype = TYPES[dtype]
    gate, value = steps(g, layout, t, b, h, dtype)
    h0 = torch.randn(b, h, generator=g).to(DEV)
    lengths = None
    if ragged:
        lengths = torch.randint(0, t + 1, (b,), generator=g).int().to(DEV)
        for i in range(b):   # what lies behind a chunk is nobody's
            gate[lengths[i]:, i] = float("nan")
            value[lengths[i]:, i] = float("inf")
    clean = (torch.nan_to_num(gate, nan=0.0), torch.nan_to_num(value, posinf=0.0))
    y, last, states = ops.linear_recurrence(gate, value, h0, lengths=lengths, reverse=reverse, save=True)
    assert y.shape == (t, b, h) and y.dtype == dtype and last.dtype == torch.float32 and states.shape == (-(-t // 16), b, h)
    num = None if lengths is None else lengths.cpu().numpy()
    want, want_last, before = ref.forward(n64(clean[0]), n64(clean[1]), n64(h0), num, reverse)
    most, unit = bounds(clean[0], clean[1], h0)
    near(last, want_last, most * unit)
    near(y, want, half(want, dtype) + most * unit * 2)
    order = before[::-1] if reverse else before
    near(states, order[::16], most * unit)
    plain = ops.linear_recurrence(gate, value, h0, lengths=lengths, reverse=reverse)
    assert len(plain) == 2 and torch.equal(plain[0], y) and torch.equal(plain[1], last)

    grad = torch.randn(t, b, h, generator=g).to(dtype).to(DEV)
    if ragged:
        for i in range(b):
            grad[lengths[i]:, i] = float("nan")
    grad_last = torch.randn(b, h, generator=g).to(DEV)
    dg, dv, dh = ops.linear_recurrence_backward(grad, gate, value, states, grad_last=grad_last, lengths=lengths, reverse=reverse)
    wg, wv, wh, e = ref.backward(n64(torch.nan_to_num(grad, nan=0.0)), n64(clean[0]), n64(clean[1]), before, n64(grad_last), num, reverse)
    back = e[None] * unit
    near(dh, wh, back[0])
    f, c = ref.sigmoid(n64(clean[0])), ref.sigmoid(-n64(clean[0]))
    near(dv, wv, half(wv, dtype) + 2 * c * back)
    # a product of e, h - v, f and c, each off by its own bound
    near(dg, wg, half(wg, dtype) + 2 * f * c * (back * most + e[None] * most * unit))


def test_parts_are_optional():
    g = torch.Generator().manual_seed(3)
    gate, value = steps(g, "time", 130, 2, 66, torch.float16)
    y, last, states = ops.linear_recurrence(gate, value, save=True)
    zero = ops.linear_recurrence(gate, value, torch.zeros(2, 66, device=DEV))
    assert torch.equal(y, zero[0]) and torch.equal(last, zero[1])
    full = torch.full((2,), 130, dtype=torch.int32, device=DEV)
    for n in (full, full + 1000):   # longer than the tensor: all of it
        got = ops.linear_recurrence(gate, value, lengths=n)
        assert torch.equal(got[0], y) and torch.equal(got[1], last)
    none = ops.linear_recurrence(gate, value, torch.ones(2, 66, device=DEV), lengths=full - 1000)   # below zero: nothing
    assert not none[0].any() and (none[1] == 1).all()
    grad = torch.randn(130, 2, 66, generator=g).half().to(DEV)
    a = ops.linear_recurrence_backward(grad, gate, value, states)
    b = ops.linear_recurrence_backward(grad, gate, value, states, grad_last=torch.zeros(2, 66, device=DEV))
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("t,b,h", [(0, 3, 8), (5, 0, 8), (5, 3, 0)])
def test_empty(t, b, h):
    x = torch.zeros(t, b, h, dtype=torch.bfloat16, device=DEV)
    h0 = torch.randn(b, h, device=DEV)
    y, last, states = ops.linear_recurrence(x, x.clone(), h0, save=True)
    assert y.shape == (t, b, h) and (t or torch.equal(last, h0))
    dg, dv, dh = ops.linear_recurrence_backward(y, x, x.clone(), states, grad_last=h0)
    assert dg.shape == dv.shape == (t, b, h) and (t or torch.equal(dh, h0))


@pytest.mark.parametrize("reverse", [False, True])
def test_a_stream_in_pieces(reverse):
    """A state handed from call to call, in place, gives what one call over everything gives, down to single steps."""
    g = torch.Generator().manual_seed(5)
    t, b, h = 300, 3, 96
    gate, value = steps(g, "time", t, b, h, torch.float16)
    h0 = torch.randn(b, h, generator=g).to(DEV)
    want, want_last, _ = ref.forward(n64(gate), n64(value), n64(h0), None, reverse)
    most, unit = bounds(gate, value, h0)
    state, out = h0.clone(), torch.empty_like(value)
    cuts = [0, 1, 2, 9, 73, 201, 299, 300]
    pieces = list(zip(cuts[:-1], cuts[1:]))
    for a, e in reversed(pieces) if reverse else pieces:
        y, last = ops.linear_recurrence(gate[a:e], value[a:e], state, reverse=reverse, out=out[a:e], h_last=state)
        assert last.data_ptr() == state.data_ptr() and y.data_ptr() == out[a:e].data_ptr()
    near(out, want, half(want, torch.float16) + 2 * most * unit)
    near(state, want_last, most * unit)


def test_gates_at_their_ends():
    """A gate of plus infinity keeps the state for good, one of minus infinity takes the value, and long memories keep their time constant."""
    inf = float("inf")
    gate = torch.tensor([inf, 200.0, -inf, -200.0, 0.0], device=DEV).half()[:, None, None].expand(5, 1, 2).contiguous()
    value = torch.tensor([5.0, 6.0, 3.0, 4.0, 2.0], device=DEV).half()[:, None, None].expand(5, 1, 2).contiguous()
    y, last = ops.linear_recurrence(gate, value, torch.full((1, 2), 9.0, device=DEV))
    assert y[:, 0, 0].tolist() == [9.0, 9.0, 3.0, 4.0, 3.0]
    t = 60000   # about one time constant of c = 1 / (1 + exp(11)); roundings of runs of eight steps
    gate, value = torch.full((t, 1, 2), 11.0, device=DEV).half(), torch.zeros(t, 1, 2, device=DEV).half()
    _, last = ops.linear_recurrence(gate, value, torch.ones(1, 2, device=DEV))
    want = np.exp(t * np.log1p(-ref.sigmoid(-11.0)))
    near(last, np.full((1, 2), want), want * 2.0 ** -24 * (11 + 8 + 3 * t / 8 + 16))


def test_the_same_bits_every_time_and_on_a_stream():
    g = torch.Generator().manual_seed(7)
    gate, value = steps(g, "packed", 700, 4, 192, torch.bfloat16)
    grad = torch.randn(700, 4, 192, generator=g).bfloat16().to(DEV)
    first = ops.linear_recurrence(gate, value, save=True)
    back = ops.linear_recurrence_backward(grad, gate, value, first[2])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ops.set_stream(stream)
    try:
        with torch.cuda.stream(stream):
            for _ in range(3):
                again = ops.linear_recurrence(gate, value, save=True)
                assert all(torch.equal(u, v) for u, v in zip(first, again))
                assert all(torch.equal(u, v) for u, v in zip(back, ops.linear_recurrence_backward(grad, gate, value, again[2])))
        # captured and replayed on new inputs in the same places
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y, last, states = ops.linear_recurrence(gate, value, save=True)
            grads = ops.linear_recurrence_backward(grad, gate, value, states)
    finally:
        ops.set_stream(None)
    new = steps(g, "packed", 700, 4, 192, torch.bfloat16)
    gate.copy_(new[0])
    value.copy_(new[1])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    want = ops.linear_recurrence(gate, value, save=True)
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
    assert all(torch.equal(u, v) for u, v in zip(grads, ops.linear_recurrence_backward(grad, gate, value, want[2])))


def test_nothing_is_written_beside_the_outputs():
    """Outputs as columns of a wider tensor, with guards around them."""
    g = torch.Generator().manual_seed(9)
    t, b, h = 77, 3, 34
    gate, value = steps(g, "time", t, b, h, torch.float16)
    wide = torch.full((t, b, h + 6), 7.0, dtype=torch.float16, device=DEV)
    y, _ = ops.linear_recurrence(gate, value, out=wide[:, :, 2:2 + h])
    want, _ = ops.linear_recurrence(gate, value)
    assert torch.equal(wide[:, :, 2:2 + h], want) and (wide[:, :, :2] == 7).all() and (wide[:, :, 2 + h:] == 7).all()


def test_refusals():
    t = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)
    gate, value = t(10, 2, 8), t(10, 2, 8)
    state = torch.zeros(2, 8, device=DEV)
    bad = [lambda: ops.linear_recurrence(gate, t(10, 2, 10)), lambda: ops.linear_recurrence(gate, value.bfloat16()), lambda: ops.linear_recurrence(gate.float(), value.float()),
           lambda: ops.linear_recurrence(t(10, 2, 7), t(10, 2, 7)), lambda: ops.linear_recurrence(gate, value, h0=state.half()), lambda: ops.linear_recurrence(gate, value, h0=state[:1]),
           lambda: ops.linear_recurrence(gate, value, lengths=torch.zeros(2, device=DEV)), lambda: ops.linear_recurrence(gate, value, lengths=torch.zeros(3, dtype=torch.int32, device=DEV)),
           lambda: ops.linear_recurrence(gate, t(10, 2, 16)[:, :, ::2]), lambda: ops.linear_recurrence(gate, value, out=t(9, 2, 8)), lambda: ops.linear_recurrence(gate[0], value[0]),
           lambda: ops.linear_recurrence_backward(gate, gate, value, torch.zeros(2, 2, 8, device=DEV)), lambda: ops.linear_recurrence_backward(gate, gate, value, None)]
    for call in bad:
        with pytest.raises((ValueError, TypeError)):
            call()
    run = [lambda: ops.linear_recurrence(t(1, 2, 8).expand(10, 2, 8), value), lambda: ops.linear_recurrence(t(21, 9)[:, 1:].unflatten(0, (7, 3)), t(7, 3, 8)),
           lambda: ops.linear_recurrence(t(162)[1:161].view(10, 2, 8), value), lambda: ops.linear_recurrence(gate, value, out=value), lambda: ops.linear_recurrence(gate, value, out=t(1, 2, 8).expand(10, 2, 8))]
    for call in run:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError):
        ops.linear_recurrence(gate.cpu(), value.cpu())


def test_more_than_2_pow_31_values():
    """Offsets beyond 32 bits: the last chunks of a tensor of 2^31 values and more give what they give by themselves, forwards and backwards."""
    t, b, h = 2100, 1024, 1000
    g = torch.Generator(device=DEV).manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float16)
    gate, value = new(t, b, h), new(t, b, h)
    assert gate.numel() > 1 << 31
    y, last, states = ops.linear_recurrence(gate, value, reverse=True, save=True)
    tail = slice(b - 64, b)   # 64 chunks of 32 runs of channels take the same form
    want = ops.linear_recurrence(gate[:, tail], value[:, tail], reverse=True, save=True)
    assert torch.equal(y[:, tail], want[0]) and torch.equal(last[tail], want[1]) and torch.equal(states[:, tail], want[2])
    dg, dv, dh = ops.linear_recurrence_backward(y, gate, value, states, reverse=True)
    part = ops.linear_recurrence_backward(y[:, tail], gate[:, tail], value[:, tail], want[2], reverse=True)
    assert torch.equal(dg[:, tail], part[0]) and torch.equal(dv[:, tail], part[1]) and torch.equal(dh[tail], part[2])


def test_two_threads_with_a_stream_each():
    import threading
    gens = [torch.Generator().manual_seed(20 + i) for i in range(2)]
    data = [steps(g, "time", 900, 3, 96, torch.float16) for g in gens]
    want = [ops.linear_recurrence(*d) for d in data]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        ops.set_stream(stream)   # of this thread
        with torch.cuda.stream(stream):
            for _ in range(50):
                y, last = ops.linear_recurrence(*data[i])
                z = ops.linear(y.view(2700, 96), data[i][1].view(2700, 96)[:64])
                stream.synchronize()
                if not (torch.equal(y, want[i][0]) and torch.equal(last, want[i][1])):
                    bad.append(i)
                if z.shape != (2700, 64):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


def test_autograd_around_the_calls():
    """A function as a training program writes it, against differentiated elementary operations in 64 bits."""
    class Recurrence(torch.autograd.Function):
        @staticmethod
        def forward(ctx, gate, value, h0):
            y, last, states = ops.linear_recurrence(gate, value, h0, save=True)
            ctx.save_for_backward(gate, value, states)
            return y, last

        @staticmethod
        def backward(ctx, dy, dlast):
            gate, value, states = ctx.saved_tensors
            return ops.linear_recurrence_backward(dy.contiguous(), gate, value, states, grad_last=dlast.contiguous())
    g = torch.Generator().manual_seed(31)
    gate, value = (t.detach().requires_grad_() for t in steps(g, "time", 21, 2, 16, torch.bfloat16))
    h0 = torch.randn(2, 16, generator=g).to(DEV).requires_grad_()
    wy, wl = torch.randn(21, 2, 16, generator=g).to(DEV), torch.randn(2, 16, generator=g).to(DEV)
    y, last = Recurrence.apply(gate, value, h0)
    ((y * wy).sum() + (last * wl).sum()).backward()
    leaves = [t.detach().double().requires_grad_() for t in (gate, value, h0)]
    h, total = leaves[2], 0
    for k in range(21):
        f = torch.sigmoid(leaves[0][k])
        h = f * h + (1 - f) * leaves[1][k]
        total = total + (h * wy[k].bfloat16().double()).sum()   # the gradient of y arrives in its type
    (total + (h * wl.double()).sum()).backward()
    for a, b in zip((gate, value, h0), leaves):
        # half a step of the gradient's type, and f32 roundings of sums of up to 21 terms
        assert ((a.grad.double() - b.grad).abs() <= b.grad.abs() * 2.0 ** -8 + b.grad.abs().max() * 2.0 ** -16).all()
