"""Layer norm over the rows of a node set, on lpg_layer_norm_{fwd,bwd}.

    y = act((x - mean) / sqrt(var + eps) * weight + bias)        per row, act = ReLU or nothing

``layer_norm`` is the function, ``LayerNorm`` the module (parameters ``weight`` / ``bias`` as
torch.nn.LayerNorm names them); ``GCN_FC(..., norm="layer")`` puts one behind every layer of each
side.  x fp32, bf16 or fp16 with any row stride; weight and bias fp32 (the master weights of bf16
training) or x's own type; statistics and sums in fp32, the output rounded once to x's type.  The
backward returns dx in x's type and the weight gradients in theirs, from a deterministic reduction.
There is no CPU path, no forward-mode derivative (a tensor with a tangent raises) and no second derivative
(a backward through gradients raises).  The argument checks and the autograd node are C++ (csrc/host.cpp).
"""
from __future__ import annotations

import torch
from torch import Tensor, nn

from . import _lib
from .timing import TIMER


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
               relu: bool = False) -> Tensor:
    """act((x - mean) / sqrt(var + eps) * weight + bias) over the last dimension of x (weight None = ones,
    bias None = zeros, act = ReLU with ``relu``).  A row that holds a NaN or an infinity comes out as NaN;
    other rows are not touched by it.  The squares are summed in fp32: of a row whose sum of squared deviations passes
    its range (3.4e38) only the bias is left."""
    tok = TIMER.start(("layer_norm", tuple(x.shape), str(x.dtype)[6:])) if TIMER.enabled else None
    y = _lib.host().layer_norm(x, weight, bias, eps, relu)
    TIMER.stop(tok)
    return y


class LayerNorm(nn.Module):
    """Layer norm over the last dimension, ``dim`` wide; ``relu=True`` in the call applies the ReLU that
    follows in the same pass."""

    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))

    def forward(self, x: Tensor, relu: bool = False) -> Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps, relu)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}"
