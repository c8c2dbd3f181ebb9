"""Layer norm over the rows of a node set, on lpg_layer_norm_{fwd,bwd}.

    y = act((x - mean) / sqrt(var + eps) * weight + bias)        per row, act = ReLU or nothing

``layer_norm`` is the function, ``LayerNorm`` the module (parameters ``weight`` / ``bias`` as
torch.nn.LayerNorm names them); ``GCN_FC(..., norm="layer")`` puts one behind every layer of each
side.  x fp32, bf16 or fp16 with any row stride; weight and bias fp32 (the master weights of bf16
training) or x's own type; statistics and sums in fp32, the output rounded once to x's type.  The
backward returns dx in x's type and the weight gradients in theirs, from a deterministic reduction.
There is no CPU path and no second derivative.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import _lib
from .timing import TIMER

_RELU = 1  # LPG_NORM_RELU


def _rows(t: Tensor) -> Tensor:
    """t as [rows, D] with contiguous rows (a copy only where its strides allow no view)."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _check(x: Tensor, weight: Tensor | None, bias: Tensor | None) -> None:
    if x.device.type != "cuda":
        raise RuntimeError("lpgnn layer_norm: runs on a HIP device only (no CPU path)")
    if x.dtype not in _lib.DTYPES:
        raise RuntimeError(f"lpgnn layer_norm: x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"lpgnn layer_norm: x needs a last dimension to normalise, got shape {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (x.shape[-1],) or p.device != x.device:
            raise RuntimeError(f"lpgnn layer_norm: {name} must be [{x.shape[-1]}] on {x.device}, got "
                               f"{tuple(p.shape)} on {p.device}")
        if p.dtype not in (torch.float32, x.dtype):
            raise RuntimeError(f"lpgnn layer_norm: {name} must be float32 or {x.dtype}, got {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"lpgnn layer_norm: weight and bias must share a type, got {weight.dtype} and {bias.dtype}")


def _forward(x: Tensor, w: Tensor | None, b: Tensor | None, eps: float, relu: bool, keep: bool):
    """(y, mean, rstd) of the rows of x [M, D]; the statistics None unless kept for a backward."""
    M, D = x.shape
    y = torch.empty((M, D), dtype=x.dtype, device=x.device)
    stats = torch.empty((2, M), dtype=torch.float32, device=x.device) if keep else (None, None)
    wd = next((t.dtype for t in (w, b) if t is not None), torch.float32)
    with torch.cuda.device(x.device):
        tok = TIMER.start(("layer_norm", M, D, str(x.dtype)[6:]))
        st = _lib.lib().lpg_layer_norm_fwd(_lib.DTYPES[x.dtype], _lib.DTYPES[wd], M, D, x.data_ptr(), x.stride(0),
                                           _lib.ptr(w), _lib.ptr(b), float(eps), _RELU if relu else 0, y.data_ptr(), D,
                                           _lib.ptr(stats[0]), _lib.ptr(stats[1]), _lib.stream_of(x))
        TIMER.stop(tok)
    _lib.check(st, "lpg_layer_norm_fwd")
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, relu):
        xr = _rows(x)
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        y, stats = _forward(xr, w, b, eps, relu, True)
        ctx.save_for_backward(xr, w, b, stats)
        ctx.relu, ctx.shape = relu, x.shape
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, b, stats = ctx.saved_tensors
        M, D = x.shape
        dy = _rows(dy)
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        new = lambda *s, like: torch.empty(s, dtype=like.dtype, device=x.device)
        dx = new(M, D, like=x) if need_x else None
        dw = new(D, like=w) if need_w else None
        db = new(D, like=b) if need_b else None
        wd = next((t.dtype for t in (w, b) if t is not None), torch.float32)
        L = _lib.lib()
        ws = None
        if need_w or need_b:
            ws = torch.empty(L.lpg_layer_norm_bwd_workspace_bytes(M, D) // 4, dtype=torch.float32, device=x.device)
        with torch.cuda.device(x.device):
            tok = TIMER.start(("layer_norm_bwd", M, D, str(x.dtype)[6:]))
            st = L.lpg_layer_norm_bwd(_lib.DTYPES[x.dtype], _lib.DTYPES[wd], M, D, x.data_ptr(), x.stride(0),
                                      dy.data_ptr(), dy.stride(0), _lib.ptr(w), _lib.ptr(b), stats[0].data_ptr(),
                                      stats[1].data_ptr(), _RELU if ctx.relu else 0, _lib.ptr(dx), D, _lib.ptr(dw),
                                      _lib.ptr(db), _lib.ptr(ws), _lib.stream_of(x))
            TIMER.stop(tok)
        _lib.check(st, "lpg_layer_norm_bwd")
        return None if dx is None else dx.view(ctx.shape), dw, db, None, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
               relu: bool = False) -> Tensor:
    """act((x - mean) / sqrt(var + eps) * weight + bias) over the last dimension of x (weight None = ones,
    bias None = zeros, act = ReLU with ``relu``).  A row that holds a NaN or an infinity comes out as NaN;
    other rows are not touched by it."""
    _check(x, weight, bias)
    if not eps >= 0:
        raise RuntimeError(f"lpgnn layer_norm: eps must not be negative, got {eps}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, float(eps), bool(relu))
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    return _forward(_rows(x), w, b, eps, relu, False)[0].view(x.shape)


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
