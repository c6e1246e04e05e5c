"""What the 16-bit product, the gated linear recurrence and the 8-bit norms refuse before anything is launched, and the formulas of the
gradients, without a GPU."""
import ctypes

import numpy as np
import pytest

from fluke_b200 import lib as L
from oracle import recurrence as ref

P = 1 << 20   # an address that is aligned and never followed


def call(flib, fn, struct, base, **change):
    s = struct()
    for k, v in {**base, **change}.items():
        setattr(s, k, v)
    return getattr(flib, fn)(ctypes.byref(s))


def test_linear_refuses(flib):
    base = dict(M=100, N=64, K=32, x=P, weight=2 * P, out=3 * P, ld_x=32, ld_out=64, alpha=1.0)
    run = lambda **c: call(flib, "fluke_linear_gpu", L.fluke_linear_t, base, **c)
    assert flib.fluke_linear_gpu(None) == 1
    for bad in (dict(M=-1), dict(N=0), dict(N=60), dict(K=0), dict(K=36), dict(dtype=2), dict(activation=6), dict(activation=-1), dict(x=0), dict(weight=0), dict(out=0),
                dict(ld_x=24), dict(ld_x=36), dict(ld_out=56), dict(residual=4 * P, ld_residual=8), dict(M=2 ** 31 - 1), dict(N=2 ** 31 - 8), dict(ld_x=1 << 40)):
        assert run(**bad) == 1, bad
    for name in ("x", "weight", "out"):
        assert run(**{name: P * 5 + 8}) == 716, name
    assert run(bias=P + 8) == 716 and run(residual=P * 5 + 2, ld_residual=64) == 716
    # the output over an input: the same start, its first and its last bytes
    size = {"x": 100 * 64, "weight": 64 * 64, "bias": 128, "residual": 100 * 128}
    for name, n in size.items():
        extra = dict(bias=6 * P, residual=7 * P, ld_residual=64)
        at = {**base, **extra}[name]
        for delta in (0, 16 - 100 * 128, n - 16):
            if name != "residual" or delta:
                assert run(**extra, out=at + delta) == 1, (name, delta)
    # columns of one wider tensor: apart side by side, not one column over
    assert run(x=P, ld_x=128, out=P + 16, ld_out=128) == 1
    assert run(M=0) == 0 and run(M=0, x=0) == 0


def test_recurrence_refuses(flib):
    base = dict(T=100, B=3, H=8, gate=P, value=2 * P, out=3 * P, h_last=4 * P, gate_step=24, gate_chunk=8, value_step=24, value_chunk=8, out_step=24, out_chunk=8)
    run = lambda **c: call(flib, "fluke_linear_recurrence_gpu", L.fluke_linear_recurrence_t, base, **c)
    assert flib.fluke_linear_recurrence_gpu(None) == 1
    for bad in (dict(T=-1), dict(B=-1), dict(H=-2), dict(H=7), dict(dtype=2), dict(gate=0), dict(value=0), dict(out=0), dict(gate_step=6), dict(gate_step=25), dict(value_chunk=0), dict(out_step=16),
                dict(out_step=8), dict(gate=P + 2), dict(T=2 ** 31 - 1), dict(out=P), dict(out=2 * P + 64), dict(h_last=P), dict(h0=4 * P + 8), dict(states=P), dict(states=4 * P), dict(lengths=3 * P)):
        assert run(**bad) == 1, bad
    for bad in (dict(h0=P + 4), dict(h_last=4 * P + 4), dict(states=5 * P + 4), dict(lengths=5 * P + 2)):
        assert run(**bad) == 716, bad
    assert run(B=0) == 0 and run(H=0) == 0


def test_recurrence_gradient_refuses(flib):
    base = dict(T=100, B=3, H=8, gate=P, value=2 * P, grad=3 * P, grad_gate=4 * P, grad_value=5 * P, states=6 * P, grad_last=7 * P, grad_h0=8 * P)
    for name in ("gate", "value", "grad", "grad_gate", "grad_value"):
        base |= {name + "_step": 24, name + "_chunk": 8}
    run = lambda **c: call(flib, "fluke_linear_recurrence_backward_gpu", L.fluke_linear_recurrence_grad_t, base, **c)
    assert flib.fluke_linear_recurrence_backward_gpu(None) == 1
    for bad in (dict(states=0), dict(grad=0), dict(grad_gate=0), dict(grad_value=0), dict(grad_gate=5 * P), dict(grad_value=3 * P), dict(grad_gate_step=10), dict(grad_h0=6 * P), dict(grad_h0=7 * P + 16),
                dict(grad_step=23), dict(grad_gate_step=8)):
        assert run(**bad) == 1, bad
    assert run(grad_h0=8 * P + 4) == 716
    # both gradients as columns of one tensor, one column too near
    wide = dict(grad_gate=4 * P, grad_value=4 * P + 14, grad_gate_step=48, grad_value_step=48, grad_gate_chunk=16, grad_value_chunk=16)
    assert run(**wide) == 1
    assert run(B=0) == 0


def test_norms_refuse_8_bit_outputs_without_scales(flib):
    base = dict(n_tokens=4, hidden_dim=64, x=P, residual=2 * P, pre_weight=3 * P, residual_out=4 * P, out=5 * P, row_scale=6 * P, alpha=1.0, eps=1e-5)
    run = lambda **c: call(flib, "fluke_rmsnorm_block_gpu", L.fluke_rmsnorm_block_t, base, **c)
    for fmt in (4, 5):
        assert run(out_format=fmt, row_scale=0) == 1 and run(out_format=fmt, out=0) == 1
        assert run(out_format=fmt, out=5 * P + 8) == 716 and run(out_format=fmt, row_scale=6 * P + 2) == 716
        assert run(out_format=fmt, out=P) == 1 and run(out_format=fmt, row_scale=P) == 1 and run(out_format=fmt, row_scale=5 * P + 252) == 1
        assert run(out_format=fmt, out=2 * P + 4 * 128 - 32) == 1
    for fmt in (3, 6, -1):
        assert run(out_format=fmt) == 1


@pytest.mark.parametrize("reverse", [False, True])
def test_gradients_of_the_formula_against_differences(reverse):
    rng = np.random.default_rng(1)
    t, b, h = 9, 3, 2
    gate, value, h0 = 2 * rng.standard_normal((t, b, h)), rng.standard_normal((t, b, h)), rng.standard_normal((b, h))
    lengths = np.array([9, 4, 0])
    dy, dl = rng.standard_normal((t, b, h)), rng.standard_normal((b, h))

    def loss(gate, value, h0):
        y, last, _ = ref.forward(gate, value, h0, lengths, reverse)
        return (y * dy).sum() + (last * dl).sum()
    before = ref.forward(gate, value, h0, lengths, reverse)[2]
    grads = ref.backward(dy, gate, value, before, dl, lengths, reverse)[:3]
    for i, args in enumerate((gate, value, h0)):
        for at in np.ndindex(args.shape):
            moved = [gate, value, h0]
            up, down = args.copy(), args.copy()
            up[at] += 1e-5
            down[at] -= 1e-5
            hi, lo = loss(*moved[:i], up, *moved[i + 1:]), loss(*moved[:i], down, *moved[i + 1:])
            # a central difference: its third derivative's part below 1e-9, roundings 2^-53 / 1e-5 of the loss
            assert abs((hi - lo) / 2e-5 - grads[i][at]) < 1e-7
