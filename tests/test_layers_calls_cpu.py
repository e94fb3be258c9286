"""Which entry of the operators a layer takes, told without a GPU."""

import pytest
import torch

from nrhints_amd import layers, ops


@pytest.fixture
def calls(monkeypatch):
    """The names of the entries that ``layers`` reaches, each replaced by torch operations."""
    seen = []

    def linear(x, weight, bias=None, residual=None, activation="none", beta=100.0):
        seen.append("linear")
        return torch.nn.functional.linear(x, weight, bias)

    def linear_train_forward(x, weight, bias=None, residual=None, activation="none", beta=100.0):
        seen.append("linear_train_forward")
        y = torch.nn.functional.linear(x, weight, bias)
        return y, torch.ones_like(y)

    def embedding(table, index, scale=1.0):
        seen.append("embedding")
        return table[index] * scale

    for f in (linear, linear_train_forward, embedding):
        monkeypatch.setattr(ops, f.__name__, f)
    return seen


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_without_gradients_a_layer_keeps_nothing_for_them(calls, mode):
    lin, emb, x, index = layers.Linear(4, 3, activation="silu"), layers.Embedding(5, 4), torch.randn(6, 4), torch.tensor([1, 2])
    held = torch.autograd.graph.get_gradient_edge(lin.weight), torch.autograd.graph.get_gradient_edge(emb.weight)
    with mode():
        y, e = lin(x), emb(index)
    assert calls == ["linear", "embedding"] and not y.requires_grad and not e.requires_grad
    assert not any(h.node.metadata for h in held)
    y, e = lin(x), emb(index)
    assert calls[2:] == ["linear_train_forward", "embedding"] and y.requires_grad and e.requires_grad
    for p in lin.parameters():
        p.requires_grad_(False)
    assert not lin(x).requires_grad and calls[4:] == ["linear"]
