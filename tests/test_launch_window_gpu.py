"""GPU: the launch window (openvis_amd._lib: a thread waits for its own launches a few windows back) around and inside captured graphs."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _chain(ops, x, gamma, beta, n):
    for _ in range(n):
        x = ops.layernorm(x, gamma, beta)
    return x


def test_a_captured_run_longer_than_the_window():
    """an event recorded into a graph cannot be waited for: calls under capture are not counted against the window, those after it are"""
    from openvis_amd import _lib, ops
    assert _lib.LAUNCH_WINDOW > 0
    g = torch.Generator().manual_seed(0)
    x, gamma, beta = torch.randn(40, 256, generator=g).cuda(), torch.randn(256, generator=g).cuda(), torch.randn(256, generator=g).cuda()
    n = 3 * _lib.LAUNCH_WINDOW + 5
    want = _chain(ops, x, gamma, beta, n)                         # past the window, eager: events are in the queue when the capture begins
    torch.cuda.synchronize()
    queue = list(_lib._tls.q)
    assert len(queue) == 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _chain(ops, x, gamma, beta, n)
    assert _lib._tls.q == queue                                   # none recorded, none waited for
    for k in range(3):
        x.mul_(1.5 if k else 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _chain(ops, x, gamma, beta, n)), k
        if k == 0:
            assert torch.equal(out, want)
    assert _lib._tls.q != queue and len(_lib._tls.q) == 2


def test_threads_have_windows_of_their_own():
    from openvis_amd import _lib, ops
    g = torch.Generator().manual_seed(1)
    x, gamma, beta = torch.randn(40, 256, generator=g).cuda(), torch.randn(256, generator=g).cuda(), torch.randn(256, generator=g).cuda()
    n = 4 * _lib.LAUNCH_WINDOW
    want, got = _chain(ops, x, gamma, beta, n), [None] * 3
    torch.cuda.synchronize()

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got[i] = _chain(ops, x, gamma, beta, n)
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(want, t) for t in got)
