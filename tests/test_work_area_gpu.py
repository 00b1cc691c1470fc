"""The context's work area around captured graphs: what a graph was captured with stays, what only eager calls used is given back."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
GIB = 1 << 30


def test_only_areas_that_a_graph_has_seen_are_kept():
    import torch
    from honeycrisp_b200 import CUDABackend
    be = CUDABackend(0)
    s = torch.cuda.Stream()
    gen = torch.Generator(device="cuda").manual_seed(3)
    a, b = (torch.randn(256, 256, generator=gen, device="cuda") for _ in range(2))
    out, want = torch.zeros(256, 256, device="cuda"), torch.zeros(256, 256, device="cuda")
    wrap = lambda t: be.wrap(t.data_ptr(), t.numel() * 4, owner=t)  # noqa: E731
    product = lambda to: be.matmul(a, False, b, False, False, 256, 256, 256, np.float32, out=wrap(to), mark=False)  # noqa: E731
    torch.cuda.synchronize()
    be.useStream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        product(out)
    be.useStream(None)
    # float32 products keep the low halves of both operands there: 1, 1.25 and 1.5 GiB of the second one's
    sizes = [GIB // 1024 + i * (GIB // 4096) for i in range(3)]
    wide, result = be.constant(0.0, 256 * sizes[-1], np.float32), be.allocate(256 * 4 * sizes[-1])
    be.sync()
    before = torch.cuda.mem_get_info()[0]
    for cols in sizes:
        be.matmul(a, False, wide, False, False, 256, 256, cols, np.float32, out=result, mark=False)
        be.sync()
    # What the first two growths brought is free again: buffers of those sizes need no more memory.
    held = [be.allocate(256 * 4 * cols - (1 << 20)) for cols in sizes[:2]]
    be.sync()
    assert before - torch.cuda.mem_get_info()[0] <= 4 * GIB   # 3.75 GiB; 6 if the outgrown areas were kept
    del held
    graph.replay()                                             # with the area of its capture
    torch.cuda.synchronize()
    product(want)
    be.sync()
    assert torch.equal(out, want) and bool(out.any())
    del graph
    be.checkDeviceStatus()
    be.close()
