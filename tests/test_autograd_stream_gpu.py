"""The autograd function of the documentation on streams of the caller's own."""
import pytest
import torch

from fluke_b200 import ops
from test_autograd_stream_cpu import documented

pytestmark = pytest.mark.gpu
DEV = "cuda"


def inputs(seed, t=300, b=5, h=96):
    g = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g)
    return [(new(t, b, h) * 1.5 + 2).half().to(DEV), new(t, b, h).half().to(DEV), new(b, h).to(DEV), new(t, b, h).half().to(DEV), new(b, h).to(DEV)]


def wanted(gate, value, h0, wy, wl):
    y, last, states = ops.linear_recurrence(gate, value, h0, save=True)
    return ops.linear_recurrence_backward(wy, gate, value, states, grad_last=wl)


def test_behind_a_slow_producer_on_a_side_stream():
    """The gradient of the outputs is computed on the side stream behind 20 ms of other work; the gradients wait for it."""
    function = documented(ops)
    gate, value, h0, wy, wl = inputs(1)
    want = wanted(gate, value, h0, wy, wl)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        leaves = [t.detach().clone().requires_grad_() for t in (gate, value, h0)]
        # what the allocator hands out again holds NaN
        for _ in range(4):
            torch.full_like(wy, float("nan"))
        y, last = function.apply(*leaves)

        def slow(dy):
            torch.cuda._sleep(40_000_000)
            return dy * 1
        y.register_hook(slow)
        ((y * wy).sum() + (last * wl).sum()).backward()
    stream.synchronize()
    for got, w in zip(leaves, want):
        assert torch.equal(got.grad, w)


def test_captured_on_a_side_stream_and_replayed():
    function = documented(ops)
    gate, value, h0, wy, wl = inputs(2)
    leaves = [t.detach().clone().requires_grad_() for t in (gate, value, h0)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()

    def step():
        y, last = function.apply(*leaves)
        return torch.autograd.grad((y, last), leaves, (wy, wl))
    with torch.cuda.stream(stream):
        step()   # whose graph is gone before the capture
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    new = inputs(3)
    with torch.no_grad():
        for leaf, t in zip(leaves, new):
            leaf.copy_(t)
        wy.copy_(new[3])
        wl.copy_(new[4])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, wanted(*new)):
        assert torch.equal(a, b)


def test_without_a_first_state():
    function = documented(ops)
    gate, value, h0, wy, wl = inputs(4)
    leaves = [t.detach().clone().requires_grad_() for t in (gate, value)]
    y, last = function.apply(*leaves, None)
    torch.autograd.backward((y, last), (wy, wl))
    want = wanted(gate, value, None, wy, wl)
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[1].grad, want[1])
