"""Launch tables of grouped kernels (csrc/devtable.h) that another stream, a capture
or an eager call meets before the first one's copy has run (tests/test_devtable.py
has the same on the CPU)."""
import pytest
import torch

from distributed_kfac_pytorch_amd.ops.mixed import BF16Weights

pytestmark = pytest.mark.gpu


class Cast:
    """Casts of one element each, every one a table of its own."""

    def __init__(self, n=64):
        self.src = torch.arange(1, n + 1, device='cuda', dtype=torch.float32)
        self.dst = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
        self.caster = BF16Weights(torch.nn.Module())

    def __call__(self, i):
        self.caster._cast([(self.src[i:i + 1], self.dst[i:i + 1])], 1)

    def done(self, *which):
        torch.cuda.synchronize()
        want = torch.zeros_like(self.dst)
        want[list(which)] = self.src[list(which)].to(torch.bfloat16)
        ok = torch.equal(self.dst, want)
        self.dst.zero_()
        return ok


def test_eager_calls_before_the_graph_runs():
    c = Cast()
    c(0)
    assert c.done(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c(1)
        c(2)
    assert c.done()                      # nothing has run yet
    c(1)
    assert c.done(1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c(2)
    assert c.done(2)
    for _ in range(3):
        g.replay()
        assert c.done(1, 2)
        c(1)
        assert c.done(1)


def test_a_graph_that_never_runs():
    c = Cast()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c(3)
    del g
    c(3)
    assert c.done(3)
    h = torch.cuda.CUDAGraph()
    with torch.cuda.graph(h):
        c(3)
    h.replay()
    assert c.done(3)


def test_two_graphs_share_a_table():
    c = Cast()
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c(4)
        c(5)
    with torch.cuda.graph(h):
        c(5)
    h.replay()
    assert c.done(5)
    g.replay()
    assert c.done(4, 5)


def test_another_stream_waits_for_the_copy():
    """The first stream is busy, so that its copy comes late."""
    c = Cast()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    m = torch.randn(4096, 4096, device='cuda')
    torch.cuda.synchronize()
    for i in range(10, 14):
        with torch.cuda.stream(a):
            for _ in range(20):
                m = m @ m * 1e-3
            c(i)
        with torch.cuda.stream(b):
            c(i)
        assert c.done(i)


def test_a_capture_while_the_eager_copy_waits():
    c = Cast()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    m = torch.randn(4096, 4096, device='cuda')
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(a):
        for _ in range(20):
            m = m @ m * 1e-3
        c(21)
    with torch.cuda.stream(b):
        g.capture_begin()                # without the synchronisation of torch.cuda.graph
        c(21)
        g.capture_end()
        g.replay()
    assert c.done(21)
