"""16-bit products called from several host threads at once, each on a stream of its own."""
import threading

import pytest
import torch

from fluke_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("sizes", [((300, 512, 2048), (4000, 1024, 512)), ((1, 4096, 4096), (64, 512, 1024)), ((6000, 1024, 256), (3000, 512, 1024))])
def test_threads_give_what_one_gives(sizes):
    """One thread's product splits K over clusters and the other's runs on pairs of SMs, or both take the same form with other sizes: capacity queries, tensor maps and tensor memory are shared."""
    data, want = [], []
    for i, (m, n, k) in enumerate(sizes):
        g = torch.Generator(device=DEV).manual_seed(m + i)
        t = lambda *s: torch.randn(*s, generator=g, device=DEV).half()
        data.append((t(m, k), t(n, k) / 8, t(n), t(m, n)))
        x, w, bias, res = data[-1]
        want.append([ops.linear(x, w, bias, act, res) for act in (None, "gelu")])
    torch.cuda.synchronize()
    bad, gate = [], threading.Barrier(len(sizes), timeout=60)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            x, w, bias, res = data[i]
            with torch.cuda.stream(stream), ops.on_stream(stream):
                gate.wait()
                for _ in range(40):
                    got = [ops.linear(x, w, bias, act, res) for act in (None, "gelu")]
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        bad.append(i)
        except BaseException as e:   # shown by the test's own thread
            bad.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad, bad
