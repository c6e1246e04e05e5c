"""Gated linear recurrence on the GPU at the ends of what it takes, through fluke_b200.ops, against oracle/recurrence.py: calls without steps, gates
that close or are infinite, infinite and largest values.

Tolerances go with the result, by a bound that is carried along with the steps. 1 / (1 + exp |g|), the smaller of f and c = 1 - f, is
    D = 2^-21 + |g| 2^-23
of itself off (exponential 2^-22, its argument 2^-24 of itself and the constant in it as much, the reciprocal 2^-23, a sum 2^-24), so a step from h to f h + c v
is, beside f times what h was off, D min(f, c) (|h| + |v|) and its own roundings off. With A' = f A + c |v| from |h0|, which no
state and no part of a joined run is above, these are four at most (the difference, the step, the product of the gates of a run and its part in the joining):
    E' = f E + D min(f, c) (A + |v|) + 4 2^-24 A'
and the same backwards for x' = f (x + dy). Nothing here grows with a large state that a gate has let go."""
import ctypes

import numpy as np
import pytest
import torch

from fluke_b200 import lib as L, ops
from oracle import recurrence as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def c_call(fn, struct, **fields):
    s = struct()
    for k, v in fields.items():
        setattr(s, k, v.data_ptr() if torch.is_tensor(v) else v)
    torch.cuda.synchronize()
    ops.set_stream(None)
    assert getattr(L.load(), fn)(ctypes.byref(s)) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("b,h", [(1, 2), (3, 8), (70, 520)])
def test_no_steps_and_a_place_for_states(b, h):
    """The states of no steps are no values: what stands at their address is not written, and plays no part."""
    around = torch.full((3, b, h), 7.0, device=DEV)
    first, last = torch.randn(b, h, device=DEV), torch.empty(b, h, device=DEV)
    c_call("fluke_linear_recurrence_gpu", L.fluke_linear_recurrence_t, T=0, B=b, H=h, h0=first, h_last=last, states=around[1])
    assert torch.equal(last, first) and (around == 7).all()
    around.fill_(float("nan"))
    c_call("fluke_linear_recurrence_backward_gpu", L.fluke_linear_recurrence_grad_t, T=0, B=b, H=h, grad_last=first, grad_h0=last.zero_(), states=around[1])
    assert torch.equal(last, first) and around.isnan().all()
    # in place
    c_call("fluke_linear_recurrence_gpu", L.fluke_linear_recurrence_t, T=0, B=b, H=h, h0=last, h_last=last, states=around[1])
    assert torch.equal(last, first) and around.isnan().all()


@pytest.mark.parametrize("t,b,h", [(100, 3, 8), (5, 7, 34), (300, 9, 64), (1200, 4, 512)])
@pytest.mark.parametrize("chunks_outside", [False, True])
def test_gradients_as_columns_of_one_tensor(t, b, h, chunks_outside):
    """What the product in front takes back: the gradients of gates and values side by side, with columns that nobody writes around them."""
    g = torch.Generator().manual_seed(t)
    new = lambda *s: torch.randn(*s, generator=g).half().to(DEV)
    gate, value, grad = new(t, b, h), new(t, b, h), new(t, b, h)
    states = ops.linear_recurrence(gate, value, save=True)[2]
    want = ops.linear_recurrence_backward(grad, gate, value, states)
    wide = torch.full((b, t, 2 * h + 16) if chunks_outside else (t, b, 2 * h + 16), 7.0, dtype=torch.float16, device=DEV)
    both = wide.transpose(0, 1) if chunks_outside else wide
    dg, dv, dh = both[..., 8:8 + h], both[..., 8 + h:8 + 2 * h], torch.empty(b, h, device=DEV)
    strides = {n + s: x.stride(i) for n, x in (("gate", gate), ("value", value), ("grad", grad), ("grad_gate", dg), ("grad_value", dv)) for i, s in enumerate(("_step", "_chunk"))}
    c_call("fluke_linear_recurrence_backward_gpu", L.fluke_linear_recurrence_grad_t, T=t, B=b, H=h, gate=gate, value=value, grad=grad, grad_gate=dg, grad_value=dv,
           states=states, grad_h0=dh, **strides)
    assert torch.equal(dg, want[0]) and torch.equal(dv, want[1]) and torch.equal(dh, want[2])
    assert (both[..., :8] == 7).all() and (both[..., 8 + 2 * h:] == 7).all()


# one size at least for each form: few steps; a warp per run of channels, for short and for many chunks; segments of 4, 8 and 16 warps; clusters; through registers
FORMS = [(1, 3, 8), (5, 130, 34), (8, 2, 64), (50, 130, 136), (100, 1030, 72), (520, 40, 256), (3000, 8, 512), (333, 7, 520), (20000, 1, 64), (4097, 1, 34), (50, 3, 6)]
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def n64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def off(g):
    """D of the smaller of f and c."""
    return 2.0 ** -21 + np.minimum(np.abs(g), 128) * 2.0 ** -23


def rounded(want, dtype):
    """Half a step of the type, subnormal values included."""
    return np.maximum(np.abs(want) * (torch.finfo(dtype).eps / 2), 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def state_bounds(gate, value, h0, reverse):
    """(A, E) in front of every step, and behind the last."""
    f, c = ref.sigmoid(gate), ref.sigmoid(-gate)
    a, e = np.abs(h0), np.zeros_like(h0)
    bounds_a, bounds_e = np.zeros_like(f), np.zeros_like(f)
    for k in (range(len(f) - 1, -1, -1) if reverse else range(len(f))):
        bounds_a[k], bounds_e[k] = a, e
        new = f[k] * a + c[k] * np.abs(value[k])
        e = f[k] * e + off(gate[k]) * np.minimum(f[k], c[k]) * (a + np.abs(value[k])) + 2.0 ** -22 * new
        a = new
    return bounds_a, bounds_e, a, e


def grad_bounds(gate, grad, grad_last, reverse):
    """(A, E) of the gradient of every step's state, and in front of the first."""
    f, c = ref.sigmoid(gate), ref.sigmoid(-gate)
    a, e = np.abs(grad_last), np.zeros_like(grad_last)
    bounds_a, bounds_e = np.zeros_like(f), np.zeros_like(f)
    for k in (range(len(f)) if reverse else range(len(f) - 1, -1, -1)):
        a = a + np.abs(grad[k])
        bounds_a[k], bounds_e[k] = a, e + 2.0 ** -24 * a
        new = f[k] * a
        e = f[k] * bounds_e[k] + off(gate[k]) * np.minimum(f[k], c[k]) * a + 2.0 ** -22 * new
        a = new
    return bounds_a, bounds_e, a, e


def near(got, want, tol, what):
    d = np.abs(n64(got) - want)
    bad = ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}, first at {tuple(np.argwhere(bad)[0])}: {n64(got)[bad][0]} for {want[bad][0]}, tolerance {np.broadcast_to(tol, d.shape)[bad][0]}"


def check(gate, value, h0, grad, grad_last, reverse):
    """All outputs of both directions."""
    dtype = gate.dtype
    y, last, states = ops.linear_recurrence(gate, value, h0, reverse=reverse, save=True)
    g, v, s = n64(gate), n64(value), n64(h0)
    want, want_last, before = ref.forward(g, v, s, None, reverse)
    a, e, a_last, e_last = state_bounds(g, v, s, reverse)
    order = slice(None, None, -1) if reverse else slice(None)
    behind_a, behind_e = (np.concatenate((x[order][1:], last_x[None]))[order] for x, last_x in ((a, a_last), (e, e_last)))
    tiny = 2.0 ** -126   # a gate's f or c below it counts as zero
    near(last, want_last, e_last + tiny, "last")
    near(y, want, rounded(want, dtype) + behind_e * (1 + torch.finfo(dtype).eps) + tiny, "out")
    near(states, before[order][::16], e[order][::16] + tiny, "states")
    dg, dv, dh = ops.linear_recurrence_backward(grad, gate, value, states, grad_last=grad_last, reverse=reverse)
    wg, wv, wh, _ = ref.backward(n64(grad), g, v, before, n64(grad_last), None, reverse)
    x, ex, x_first, e_first = grad_bounds(g, n64(grad), n64(grad_last), reverse)
    f, c, d = ref.sigmoid(g), ref.sigmoid(-g), off(g)
    near(dh, wh, e_first + tiny, "dh")
    near(dv, wv, rounded(wv, dtype) + (c * ex + (d * np.minimum(f, c) + 2.0 ** -23 * c) * x) * (1 + torch.finfo(dtype).eps) + tiny, "dv")
    size = a + np.abs(v)
    near(dg, wg, rounded(wg, dtype) + f * c * (ex * size + 2 * x * e + (d + 8 * 2.0 ** -24) * x * size) * (1 + torch.finfo(dtype).eps) + tiny, "dg")


def closing(seed, t, b, h, dtype):
    """Gates that mostly keep, of which one in ten closes (0 to -16), values of a thousandth, and now and then one of a hundred that is let in."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g)
    gate = torch.where(rand(t, b, h) < 0.1, -16 * rand(t, b, h), 2 + 8 * rand(t, b, h))
    value = 1e-3 * torch.randn(t, b, h, generator=g)
    large = rand(t, b, h) < 0.02
    gate, value = torch.where(large, torch.full_like(gate, -3.0), gate), torch.where(large, 1e5 * value, value)
    return gate.to(dtype).to(DEV), value.to(dtype).to(DEV), (100 * torch.randn(b, h, generator=g)).to(DEV)


@pytest.mark.parametrize("t,b,h", FORMS)
@pytest.mark.parametrize("dtype,reverse", [("f16", False), ("bf16", True)])
def test_gates_that_close_on_large_states(t, b, h, dtype, reverse):
    """What is left of a large state behind a gate that closes, and what reaches a gradient through one, keeps its digits."""
    gate, value, h0 = closing(t + b + h, t, b, h, TYPES[dtype])
    g = torch.Generator().manual_seed(t)
    grad_last = torch.randn(b, h, generator=g).to(DEV)
    # a gradient of the step that is taken last, and of it alone
    grad = torch.zeros(t, b, h, dtype=TYPES[dtype], device=DEV)
    grad[0 if reverse else t - 1] = 1.5
    check(gate, value, h0, grad, grad_last, reverse)
    check(gate, value, h0, torch.randn(t, b, h, generator=g).to(TYPES[dtype]).to(DEV), 100 * grad_last, reverse)


@pytest.mark.parametrize("gate", [-8.0, -12.0, -16.0, -1.0, 0.0, -0.0])
def test_one_step_through_a_closed_gate(gate):
    """f h by itself: the value is zero, and the gradient comes from behind."""
    x = lambda v: torch.full((1, 1, 8), v, dtype=torch.bfloat16, device=DEV)
    check(x(gate), x(0.0), torch.full((1, 8), 100.0, device=DEV), x(0.0), torch.full((1, 8), 3.0, device=DEV), False)
    check(x(gate), x(0.125), torch.full((1, 8), 100.0, device=DEV), x(2.0), torch.full((1, 8), 3.0, device=DEV), False)


@pytest.mark.parametrize("t,b,h", [(333, 7, 520), (3000, 8, 512), (520, 40, 256), (20000, 1, 64), (4097, 1, 34), (50, 130, 136)])
def test_a_large_first_state_that_fades(t, b, h):
    """Runs of steps that are joined leave nothing of a state that they have let go: behind a few steps of gates of -1 the small values stand by themselves."""
    g = torch.Generator().manual_seed(t)
    gate = torch.full((t, b, h), -1.0, dtype=torch.bfloat16, device=DEV)
    value = (1e-3 * torch.randn(t, b, h, generator=g)).bfloat16().to(DEV)
    big = torch.full((b, h), 3e4, device=DEV)
    zero = torch.zeros(t, b, h, dtype=torch.bfloat16, device=DEV)
    check(gate, value, big, zero, big, False)
    check(gate, value, big, (1e-3 * torch.randn(t, b, h, generator=g)).bfloat16().to(DEV), big, True)


def same(got, want, tol, what):
    """Infinities and NaN in the same places, and the rest within the tolerance."""
    got = n64(got)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN at {tuple(np.argwhere(np.isnan(got) != np.isnan(want))[0])}, {(np.isnan(got) != np.isnan(want)).sum()} differ"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities"
    ok = ~inf & ~np.isnan(want)
    d = np.abs(got - want, where=ok, out=np.zeros_like(got))
    with np.errstate(invalid="ignore"):
        bad = ok & ~(d <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())}, first at {tuple(np.argwhere(bad)[0])}: {got[bad][0]} for {want[bad][0]}"


@pytest.mark.parametrize("t,b,h", FORMS)
@pytest.mark.parametrize("dtype,reverse,ragged", [("f16", False, True), ("bf16", True, False)])
def test_gates_at_their_ends_in_every_form(t, b, h, dtype, reverse, ragged):
    """Gates of both infinities and far beyond where an exponential overflows, anywhere and at the borders of tiles and segments, on finite states."""
    g = torch.Generator().manual_seed(t + 3 * b + h)
    gate = 3 * torch.randn(t, b, h, generator=g)
    some = torch.rand(t, b, h, generator=g)
    for i, end in enumerate((float("inf"), float("-inf"), 200.0, -200.0)):
        gate[(some > 0.02 * i) & (some < 0.02 * i + 0.02)] = end
    gate[::16, :, ::3], gate[15::16, :, 1::3] = float("-inf"), float("inf")
    gate = gate.to(TYPES[dtype]).to(DEV)
    value, grad = (torch.randn(t, b, h, generator=g).to(TYPES[dtype]).to(DEV) for _ in range(2))
    h0, grad_last = (torch.randn(b, h, generator=g).to(DEV) for _ in range(2))
    check(gate, value, 50 * h0, grad, grad_last, reverse)
    if ragged:   # behind a chunk's end a gate closes nothing
        lengths = torch.randint(0, t + 1, (b,), generator=g).int().to(DEV)
        y, last, states = ops.linear_recurrence(gate, value, h0, lengths=lengths, reverse=reverse, save=True)
        for i in range(b):
            n = int(lengths[i])
            part = slice(0, n)
            if n and i < 4:
                one = ops.linear_recurrence(gate[part, i:i + 1], value[part, i:i + 1], h0[i:i + 1], reverse=reverse)
                want, want_last, _ = ref.forward(n64(gate[part, i:i + 1]), n64(value[part, i:i + 1]), n64(h0[i:i + 1]), None, reverse)
                for got, got_last in ((y[part, i:i + 1], last[i:i + 1]), one):
                    near(got, want, rounded(want, TYPES[dtype]) + 2.0 ** -16 * 8, "out")
                    near(got_last, want_last, 2.0 ** -16 * 8, "last")
            elif not n:
                assert torch.equal(last[i], h0[i])
            assert not y[n:, i].any()


@pytest.mark.parametrize("t,b,h", FORMS)
@pytest.mark.parametrize("dtype,reverse", [("f16", True), ("bf16", False)])
def test_infinities_and_the_largest_values(t, b, h, dtype, reverse):
    """An infinite state stays one, and values of opposite sign whose difference is too large for f32 have a mean all the same."""
    dtype = TYPES[dtype]
    g = torch.Generator().manual_seed(5 * t + b + h)
    gate = (4 * torch.randn(t, b, h, generator=g)).clamp(-30, 30).to(dtype)
    value, grad = (torch.randn(t, b, h, generator=g).to(dtype) for _ in range(2))
    h0, grad_last = (torch.randn(b, h, generator=g) for _ in range(2))
    kind = torch.arange(b * h).view(b, h) % 8   # of a channel
    at = lambda: torch.randint(0, t, (b, h), generator=g)
    put = lambda x, where, when, v: x.scatter_(0, when[None], torch.where(where, torch.tensor(v, dtype=x.dtype), x.gather(0, when[None])[0])[None])
    inf, largest = float("inf"), torch.finfo(dtype).max
    put(value, kind == 1, at(), inf)
    put(value, kind == 2, at(), -inf)
    put(value, kind == 2, at(), inf)
    h0[kind == 3] = -inf
    put(value, kind == 4, at(), float("nan"))
    value[:, kind == 5] = torch.where(torch.rand(t, b, h, generator=g) < 0.5, largest, -largest)[:, kind == 5].to(dtype)
    h0[kind == 5] = -float(largest)
    put(grad, kind == 6, at(), -inf)
    grad_last[kind == 7] = inf
    gate, value, grad, h0, grad_last = (x.to(DEV) for x in (gate, value, grad, h0, grad_last))
    lengths = torch.randint(0, t + 1, (b,), generator=g).int()
    lengths[:1] = t
    for lens in (None, lengths.to(DEV)):
        num = None if lens is None else lens.cpu().numpy()
        y, last, states = ops.linear_recurrence(gate, value, h0, lengths=lens, reverse=reverse, save=True)
        with np.errstate(all="ignore"):
            want, want_last, before = ref.forward(n64(gate), n64(value), n64(h0), num, reverse)
            # E of a state is below this part of the largest that its channel has seen
            top = np.maximum(np.nanmax(np.where(np.isfinite(n64(value)), np.abs(n64(value)), 0), 0), np.where(np.isfinite(n64(h0)), np.abs(n64(h0)), 0))
            part = top * 2.0 ** -24 * (4 * min(t, 1 / ref.sigmoid(-n64(gate)).min()) + 256)
            same(last, want_last, part, "last")
            same(y, want, rounded(want, dtype) + part * 1.01, "out")
            order = slice(None, None, -1) if reverse else slice(None)
            same(states, before[order][::16], part, "states")
            dg, dv, dh = ops.linear_recurrence_backward(grad, gate, value, states, grad_last=grad_last, lengths=lens, reverse=reverse)
            wg, wv, wh, e = ref.backward(n64(grad), n64(gate), n64(value), before, n64(grad_last), num, reverse)
            back = np.nanmax(np.where(np.isfinite(e), e, 0)) * 2.0 ** -24 * (4 * min(t, 1 / ref.sigmoid(-n64(gate)).min()) + 256)
            same(dh, wh, back, "dh")
            same(dv, wv, rounded(wv, dtype) + 1.01 * back, "dv")
            # A factor that is smaller than its own error may as well be zero or of the other sign, so that its product with an infinite one is any infinity or NaN:
            # a state that f32 holds as the value itself (f of 1e-13), say, whose difference is zero there
            x, here, dy, f = n64(grad_last), np.zeros_like(wg), n64(grad), ref.sigmoid(n64(gate))
            for k in (range(t) if reverse else range(t - 1, -1, -1)):
                live = (k < (np.full(b, t) if num is None else num))[:, None]
                here[k] = np.where(live, dy[k] + x, 0)
                x = np.where(live, f[k] * here[k], x)
            d = before - n64(value)
            any_of = (np.isinf(here) & (np.abs(d) <= part)) | (np.isinf(d) & (np.abs(here) <= back))
            wg[any_of] = n64(dg)[any_of]
            # where the product is near the end of the type its rounding decides
            edge = np.abs(wg) > 0.99 * float(largest)
            wg[edge & ~np.isinf(wg)] = n64(dg)[edge & ~np.isinf(wg)]
            same(dg, wg, rounded(wg, dtype) + 1.01 * (2 * back * top + 64 * part * (1 + np.nanmax(np.where(np.isfinite(e), e, 0)))), "dg")
