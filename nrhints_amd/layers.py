"""Layers of any shape under autograd: ``linear`` / ``Linear`` and ``embedding`` / ``Embedding`` over ``ops`` (csrc/nrh_linear.hip,
csrc/nrh_embedding.hip).

The networks of the renderer run on kernels whose shape is compiled in; these are the building blocks for networks that have another
one (the background network at other widths and depths, outside.OutsideNeRF) and for tables looked up per ray (RayGenerator's
per-view deltas).  GPU tensors only, float32 / float16 / bfloat16, one derivative (a second one raises).  Gradients are summed in a
fixed order: the same bits on every run.  Forward and backward may be captured into a graph; a capture is refused while a graph of
the same parameters that was recorded on another stream is alive.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.autograd.graph import get_gradient_edge

from . import ops


_STREAM = "nrhints_amd.layers: stream"


def _same_side_of_capture(*tensors) -> list:
    """A parameter's gradient is accumulated on the stream on which its accumulation node was made, by the first graph that holds the
    parameter, and the node lives as long as any graph does.  A backward pass captured on another stream would accumulate outside the
    capture and end the process: refuse it here, while an exception still can.  -> the nodes, to be held until the graph holds them."""
    held = []
    for t in tensors:
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.requires_grad and t.is_leaf):
            continue
        capturing, here = torch.cuda.is_current_stream_capturing(), torch._C._cuda_getCurrentRawStream(t.device.index)
        node = get_gradient_edge(t).node
        if _STREAM not in node.metadata:
            # Made here and now, it dies with its last reference.  One that stays belongs to another operation's graph: to this capture's own, as far
            # as can be told, or outside a capture to a stream that nobody knows.
            node.metadata[_STREAM] = here if capturing else None
            del node
            node = get_gradient_edge(t).node
            node.metadata.setdefault(_STREAM, here)
        if capturing and node.metadata[_STREAM] != here:
            raise RuntimeError("a graph recorded outside this capture still holds one of these parameters, on another stream: delete its outputs "
                               "(or detach them) before capturing, or record it on the capturing stream (as for a wrapper that keeps its "
                               "parameters' nodes)")
        held.append(node)
    return held


class LinearHip(torch.autograd.Function):
    """(x [..., k], weight [n, k], bias [n] | None, residual [..., n] | None) -> act(x weight^T + bias) + residual."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation: str, beta: float):
        if not any(ctx.needs_input_grad[:3]):
            return ops.linear(x, weight, bias, residual, activation, beta)
        y, dact = ops.linear_train_forward(x, weight, bias, residual, activation, beta)
        ctx.save_for_backward(x, weight, dact)      # relu without residual: dact may be y, an output (saved as such, no copy)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, y_bar):
        need = ctx.needs_input_grad
        g_x = g_w = g_b = None
        if any(need[:3]):
            x, weight, dact = ctx.saved_tensors
            g_x, g_w, g_b = ops.linear_backward(y_bar, x, weight, dact, ctx.activation, need[0], need[1], need[2])
        return g_x, g_w, g_b, (y_bar if need[3] else None), None, None


class EmbeddingHip(torch.autograd.Function):
    """(table [v, d], index) -> scale * table[index]; the table's gradient by sorted tokens."""

    @staticmethod
    def forward(ctx, table, index, scale: float):
        ctx.save_for_backward(index)
        ctx.rows, ctx.scale = table.shape[0], float(scale)
        return ops.embedding(table, index, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, rows_bar):
        (index,) = ctx.saved_tensors
        return ops.embedding_backward(rows_bar, index, ctx.rows, ctx.scale), None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           activation: str = "none", beta: float = 100.0) -> torch.Tensor:
    """``ops.linear`` with gradients for x, weight, bias and residual."""
    if not torch.is_grad_enabled():      # (inside the Function it always is off, and needs_input_grad is requires_grad alone)
        return ops.linear(x, weight, bias, residual, activation, float(beta))
    held = _same_side_of_capture(x, weight, bias, residual)      # noqa: F841 - until the Function's node holds them
    return LinearHip.apply(x, weight, bias, residual, activation, float(beta))


def embedding(table: torch.Tensor, index: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``ops.embedding`` with the table's gradient."""
    if not torch.is_grad_enabled():
        return ops.embedding(table, index, float(scale))
    held = _same_side_of_capture(table)      # noqa: F841 - until the Function's node holds it
    return EmbeddingHip.apply(table, index, float(scale))


class Linear(nn.Module):
    """A layer with its activation: weight [n, k] and bias [n] initialised like nn.Linear (same draws in the same order)."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", beta: float = 100.0):
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError("Linear: in_features and out_features must be positive")
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ops.ACTIVATIONS)}")
        self.in_features, self.out_features, self.activation, self.beta = in_features, out_features, activation, float(beta)
        self.weight = nn.Parameter(torch.empty(out_features, in_features))
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if bias:
            self.bias = nn.Parameter(torch.empty(out_features))
            nn.init.uniform_(self.bias, -1.0 / math.sqrt(in_features), 1.0 / math.sqrt(in_features))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        return linear(x, self.weight, self.bias, residual, self.activation, self.beta)


class Embedding(nn.Module):
    """A table of learned rows, initialised N(0, 1) like nn.Embedding; ``scale`` multiplies every looked-up row."""

    def __init__(self, num_rows: int, dim: int, scale: float = 1.0):
        super().__init__()
        if num_rows < 1 or dim < 1:
            raise ValueError("Embedding: num_rows and dim must be positive")
        self.scale = float(scale)
        self.weight = nn.Parameter(torch.empty(num_rows, dim).normal_())

    def forward(self, index: torch.Tensor) -> torch.Tensor:
        return embedding(self.weight, index, self.scale)
