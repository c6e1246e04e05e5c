"""What the gated linear recurrence refuses of calls without steps, before anything is launched."""
import ctypes

from fluke_b200 import lib as L

P = 1 << 20   # an address that is aligned and never followed


def call(flib, fn, struct, base, **change):
    s = struct()
    for k, v in {**base, **change}.items():
        setattr(s, k, v)
    return getattr(flib, fn)(ctypes.byref(s))


def test_no_steps_and_overlapping_states(flib):
    """Without steps the first state is still read and the last one written: one that half overlaps the other, or the lengths, is refused as with steps."""
    run = lambda **c: call(flib, "fluke_linear_recurrence_gpu", L.fluke_linear_recurrence_t, {**dict(T=0, B=3, H=8, h0=P, h_last=2 * P), **c})
    for delta in (8, 88, -8, -88):
        assert run(h_last=P + delta) == 1, delta
    assert run(lengths=2 * P + 92) == 1
    back = lambda **c: call(flib, "fluke_linear_recurrence_backward_gpu", L.fluke_linear_recurrence_grad_t, {**dict(T=0, B=3, H=8, grad_last=P, grad_h0=2 * P), **c})
    for delta in (8, 88, -8, -88):
        assert back(grad_h0=P + delta) == 1, delta
    assert back(lengths=2 * P + 92) == 1


def test_gradients_side_by_side_one_column_too_near(flib):
    """Both gradients as columns of one tensor, on addresses that the alignment allows: the second begins inside the first's eight columns, or ends inside its next row's."""
    base = dict(T=100, B=3, H=8, gate=P, value=2 * P, grad=3 * P, grad_gate=4 * P, grad_value=4 * P, states=6 * P, grad_last=7 * P, grad_h0=8 * P)
    for name in ("gate", "value", "grad"):
        base |= {name + "_step": 24, name + "_chunk": 8}
    for name in ("grad_gate", "grad_value"):
        base |= {name + "_step": 48, name + "_chunk": 16}
    for delta in (4, 8, 12, 20, 24, 28, -4, -12):
        assert call(flib, "fluke_linear_recurrence_backward_gpu", L.fluke_linear_recurrence_grad_t, {**base, "grad_value": 4 * P + delta}) == 1, delta
