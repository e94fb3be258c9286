"""What of the layer operators' calls can be told without a GPU: which entry a layer takes, and what the C entries refuse."""
import ctypes

import pytest
import torch

from nrhints_amd import _lib, layers, ops


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


def test_a_derivative_of_no_activation_is_refused():
    """act' of "none" is one and is not written: a buffer for it is a mistake of the caller's, in every form of the product."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buf) + 15) // 16 * 16            # never reached by a launch
    for m in (4, 100):
        assert lib.nrh_linear_forward(0, p, 8, p, 8, None, None, 0, 0, 1.0, m, 4, 8, p, 4, p, None, 0, None) == -1
        assert b"activation" in lib.nrh_last_error_string()
