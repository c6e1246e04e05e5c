"""The autograd function of the documentation, on whatever thread torch runs it: the library launches on torch's current stream there, and the
thread's own setting comes back."""
import os
import re
import threading
import types

import pytest
import torch

from fluke_b200 import lib as L, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def documented(ops):
    """`class Recurrence` as the documentation has it, over these operators."""
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    code = re.search(r"```python\n(class Recurrence\(.*?)```", text, re.S).group(1)
    space = {"torch": torch, "ops": ops}
    exec(code, space)
    return space["Recurrence"]


@pytest.mark.parametrize("own_setting", [None, 0x5000])
def test_both_directions_launch_on_the_current_stream(flib, monkeypatch, own_setting):
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0x1230))
    seen = []

    def record(count, fails=False):
        def call(*args, **kwargs):
            seen.append(flib.fluke_get_stream())
            if fails:
                raise RuntimeError("refused")
            return tuple(torch.zeros(2, 1, 2) for _ in range(count))
        return call

    fake = types.SimpleNamespace(**{n: getattr(ops, n) for n in dir(ops) if not n.startswith("_")})
    fake.linear_recurrence, fake.linear_recurrence_backward = record(3), record(3)
    function = documented(fake)
    x = torch.zeros(2, 1, 2)
    after, bad = [], []

    def work():
        try:
            flib.fluke_set_stream(own_setting or 0)
            ctx = types.SimpleNamespace(save_for_backward=lambda *t: setattr(ctx, "saved_tensors", t), needs_input_grad=(True, True, False))
            function.forward(ctx, x, x, None)
            after.append(flib.fluke_get_stream())
            assert function.backward(ctx, x, x)[2] is None   # no gradient for a first state that there was not
            after.append(flib.fluke_get_stream())
            fake.linear_recurrence_backward = record(0, fails=True)
            with pytest.raises(RuntimeError, match="refused"):
                function.backward(ctx, x, x)
            after.append(flib.fluke_get_stream())
        except BaseException as e:   # shown by the test's own thread
            bad.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not bad, bad
    assert seen == [0x1230] * 3 and after == [own_setting] * 3
    assert flib.fluke_get_stream() is None   # this thread's was not touched
