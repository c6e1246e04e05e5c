"""The gated linear recurrence and its gradients in 64 bits, step by step, for the tests.

    h_t = f_t h_{t-1} + (1 - f_t) v_t,  f = 1 / (1 + exp(-g)),  arrays [T, B, H]"""
import numpy as np


def sigmoid(g):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-g))


def forward(gate, value, h0=None, lengths=None, reverse=False):
    """(out, h_last, the state in front of each step)."""
    gate, value = np.asarray(gate, np.float64), np.asarray(value, np.float64)
    t, b, h = gate.shape
    lengths = np.full(b, t) if lengths is None else np.clip(lengths, 0, t)
    f, i = sigmoid(gate), sigmoid(-gate)
    state = np.zeros((b, h)) if h0 is None else np.array(h0, np.float64)
    out, before = np.zeros((t, b, h)), np.zeros((t, b, h))
    for k in (range(t - 1, -1, -1) if reverse else range(t)):
        live = (k < lengths)[:, None]
        before[k] = state
        state = np.where(live, f[k] * state + i[k] * np.where(live, value[k], 0), state)
        out[k] = np.where(live, state, 0)
    return out, state, before


def backward(grad, gate, value, before, grad_last=None, lengths=None, reverse=False):
    """(gradient of gate, of value, of h0, the largest |e|)."""
    grad, gate, value = (np.asarray(a, np.float64) for a in (grad, gate, value))
    t, b, h = gate.shape
    lengths = np.full(b, t) if lengths is None else np.clip(lengths, 0, t)
    f, i = sigmoid(gate), sigmoid(-gate)
    x = np.zeros((b, h)) if grad_last is None else np.array(grad_last, np.float64)
    dg, dv, most = np.zeros((t, b, h)), np.zeros((t, b, h)), np.abs(x)
    for k in (range(t) if reverse else range(t - 1, -1, -1)):
        live = (k < lengths)[:, None]
        e = np.where(live, grad[k], 0) + x
        dv[k] = np.where(live, i[k] * e, 0)
        dg[k] = np.where(live, e * (before[k] - np.where(live, value[k], 0)) * f[k] * i[k], 0)
        x = np.where(live, f[k] * e, x)
        most = np.maximum(most, np.abs(e))
    return dg, dv, x, most
