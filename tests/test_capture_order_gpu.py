"""Products on the backend's own stream around a capture on it: a captured product has not run, so a product launched behind the capture
follows the one launched in front of it, whose result it may read."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_a_product_behind_a_capture_waits_for_the_one_in_front():
    import torch
    from honeycrisp_b200 import CUDABackend, _lib
    be = CUDABackend(0)
    kernel = _lib.HC_KERNEL_TENSOR
    n = 2048
    rng = np.random.default_rng(2)
    x0 = rng.integers(-8, 9, (n, n)).astype(np.float16)
    perm = rng.permutation(n)
    P = np.zeros((n, n), np.float16)
    P[np.arange(n), perm] = 1.0
    x, p = be.collection(x0, np.float16), be.collection(P, np.float16)
    first, second = be.allocate(n * n * 2), be.allocate(n * n * 2)
    small, other = be.constant(1.0, 256 * 256, np.float16), be.constant(0.0, 256 * 256, np.float16)
    own = torch.cuda.ExternalStream(be.stream())
    back = np.argsort(perm)
    once, twice = x0[:, back], x0[:, back][:, back]
    graphs = []
    for _ in range(8):
        be.constant(0.0, 1, np.float16)
        be.matmul(x, False, p, False, False, n, n, n, np.float16, kernel=kernel, out=first, mark=False)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(own):
            graph.capture_begin(capture_error_mode="thread_local")
            be.matmul(small, False, small, False, False, 256, 256, 256, np.float16, kernel=kernel, out=other, mark=False)
            graph.capture_end()
        graphs.append(graph)
        be.matmul(first, False, p, False, False, n, n, n, np.float16, kernel=kernel, out=second, mark=False)
        assert np.array_equal(second.onCPU(np.float16).reshape(n, n), twice)
        assert np.array_equal(first.onCPU(np.float16).reshape(n, n), once)
        be.matmul(p, False, p, False, False, n, n, n, np.float16, kernel=kernel, out=first, mark=False)   # other contents for the next round
        be.matmul(p, False, p, False, False, n, n, n, np.float16, kernel=kernel, out=second, mark=False)
    assert not other.onCPU(np.float16).any()
    with torch.cuda.stream(own):
        graphs[0].replay()
    be.sync()
    assert (other.onCPU(np.float16) == 256).all()
    del graphs
    be.checkDeviceStatus()
    be.close()


def test_captured_chain_replays_exactly():
    """A chain of products that read one another's results, captured on the own stream behind a launched product."""
    import torch
    from honeycrisp_b200 import CUDABackend, _lib
    be = CUDABackend(0)
    kernel = _lib.HC_KERNEL_TENSOR
    n, steps = 512, 12
    rng = np.random.default_rng(4)
    x0 = rng.integers(-8, 9, (n, n)).astype(np.float16)
    perm = rng.permutation(n)
    P = np.zeros((n, n), np.float16)
    P[np.arange(n), perm] = 1.0
    x, p = be.collection(x0, np.float16), be.collection(P, np.float16)
    bufs = [be.allocate(n * n * 2) for _ in range(3)]

    def chain():
        cur = bufs[0]
        for i in range(steps):
            out = bufs[1 + i % 2]
            be.matmul(cur, False, p, False, False, n, n, n, np.float16, kernel=kernel, out=out, mark=False)
            cur = out
        return cur

    own = torch.cuda.ExternalStream(be.stream())
    graph = torch.cuda.CUDAGraph()
    be.matmul(x, False, p, False, False, n, n, n, np.float16, kernel=kernel, out=bufs[0], mark=False)
    with torch.cuda.stream(own):
        graph.capture_begin(capture_error_mode="thread_local")
        last = chain()
        graph.capture_end()
    want = x0
    for _ in range(steps + 1):
        want = want[:, np.argsort(perm)]
    for _ in range(3):
        with torch.cuda.stream(own):
            graph.replay()
        be.sync()
        assert np.array_equal(last.onCPU(np.float16).reshape(n, n), want)
    del graph
    be.checkDeviceStatus()
    be.close()
