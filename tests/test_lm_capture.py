"""Backward passes of the language-model operators in a captured graph, while
eager graphs of some of their leaves live: a gradient that the capture would
hand to another stream is refused, on the host and in front of every launch."""
import pytest
import torch

from dear_pytorch_amd.ops.fused_ln import layer_norm


def leaves():
    gen = torch.Generator().manual_seed(2)
    x, r = torch.randn(2, 6, 64, generator=gen)
    w, b = torch.randn(2, 64, generator=gen)
    return [t.cuda() for t in (x, w, b, r)]


def call(t):
    return layer_norm(t[0], t[1], t[2], 1e-5, residual=t[3])


def captured(fn):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def replayed(graph, got, want):
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(4))
def test_gpu_each_leaf_of_a_live_graph_is_looked_at(i):
    """One leaf asks for a gradient, all others are frozen."""
    t = leaves()
    t[i].requires_grad_(True)
    alive, up = call(t), torch.ones(6, 64, device="cuda")

    def refused():
        with pytest.raises(RuntimeError, match="alive"):
            torch.autograd.grad(call(t), t[i], up)

    captured(refused)
    want = torch.autograd.grad(alive, t[i], up)
    del alive
    graph, got = captured(lambda: torch.autograd.grad(call(t), t[i], up))
    replayed(graph, got, want)


@pytest.mark.gpu
def test_gpu_the_bias_alone_lives_elsewhere():
    t = [v.requires_grad_(True) for v in leaves()]
    other = t[2] * 2.0                    # an eager graph of the bias only
    up = torch.ones(6, 64, device="cuda")

    def refused():
        with pytest.raises(RuntimeError, match="alive"):
            torch.autograd.grad(call(t), t, up)

    captured(refused)
    del other
    want = torch.autograd.grad(call(t), t, up)
    graph, got = captured(lambda: torch.autograd.grad(call(t), t, up))
    replayed(graph, got, want)


@pytest.mark.gpu
def test_gpu_a_leaf_that_nothing_is_asked_of_may_live_elsewhere():
    t = [v.requires_grad_(True) for v in leaves()]
    up = torch.ones(6, 64, device="cuda")
    want = torch.autograd.grad(call(t), t, up)
    other = t[1] * 2.0 + t[2]             # eager graphs of weight and bias
    asked = [t[0], t[3]]
    graph, got = captured(lambda: torch.autograd.grad(call(t), asked, up))
    replayed(graph, got, [want[0], want[3]])
    del other
