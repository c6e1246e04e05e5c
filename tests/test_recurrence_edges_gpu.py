"""Gated linear recurrence on the GPU at the ends of what it takes: calls without steps."""
import ctypes

import pytest
import torch

from fluke_b200 import lib as L, ops

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
