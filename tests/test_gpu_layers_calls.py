"""How the layer operators are called: what a gradient call computes and what not, captures beside eager graphs, tensors whose sign is a
flag."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from nrhints_amd import layers, ops  # noqa: E402


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.code = layers.Embedding(20, 16)
        self.l0, self.l1 = layers.Linear(16, 32, activation="silu"), layers.Linear(32, 8, activation="relu")

    def forward(self, view):
        return self.l1(self.l0(self.code(view)))


def net_and_batch(n=100):
    torch.manual_seed(5)
    return Net().cuda(), torch.randint(0, 20, (n,), generator=gen(3), device="cuda"), torch.randn(n, 8, generator=gen(4), device="cuda")


def test_an_inference_is_captured_beside_a_live_eager_graph():
    """Without gradients there is no backward pass to capture: an eager graph of the parameters that is still alive does not matter, and an
    evaluation between two captures leaves no trace."""
    net, view, seed = net_and_batch()
    alive = net(view)
    gr = torch.cuda.CUDAGraph()
    with torch.no_grad():
        net(view)
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            y = net(view)
    for _ in range(3):
        y.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive)
    want = torch.autograd.grad(alive, list(net.parameters()), seed)
    del alive
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        y1 = net(view)
        g1 = torch.autograd.grad(y1, list(net.parameters()), seed)
    with torch.no_grad():
        net(view)
    torch.cuda.synchronize()
    with torch.cuda.graph(second):
        y2 = net(view)
        g2 = torch.autograd.grad(y2, list(net.parameters()), seed)
    for _ in range(3):
        for t in (*g1, *g2):
            t.zero_()
        first.replay()
        second.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, g1, g2))
