"""The per-node fully connected layer in 8-bit integers (evaluation), on lpg_quant_i8, lpg_fc_i8 and
lpg_fc_i8_rows.

Both operands are int8 with one scale a row: an activation row's own (found in the call), a weight row's --
an output channel's -- found once, ahead.  With x = [x1 | x2] (GraphConv: the aggregate and the node's own
features) and W = [W_rel | W_root]:

    top_m = max_k |x_mk|,  q_mk = round_half_even(127 x_mk / top_m)
    y_mn  = act((sum_k q_mk wq_nk) (top_m / 127) ws_n + bias_n)

The sum is exact (32-bit integers), the quotient decided exactly, so the result does not depend on how the
work is split.  x fp32, bf16 or fp16, y of its type.  No gradient, backward or forward-mode
(refused where any tensor of the call wants one); no CPU path.  Checks and launches are C++ (csrc/host.cpp).
"""
from __future__ import annotations

from torch import Tensor

from . import _lib
from .timing import TIMER


def quantize_i8(x: Tensor, x2: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """(q, scale): the rows of [x | x2] as int8 [rows, K1 + K2] (a view of rows on 128-byte borders) and their
    fp32 scales, x ~ q * scale[:, None] to half a scale.  Weights for linear_i8: quantize_i8(W_rel, W_root).
    A row of zeros (or below 2^-100) has the scale 0; one with a NaN or an infinity the scale NaN."""
    return _lib.host().quantize_i8(x, x2)


def linear_i8(x: Tensor, wq: Tensor, ws: Tensor, bias: Tensor | None = None, x2: Tensor | None = None,
              relu: bool = False) -> Tensor:
    """act([x | x2] W^T + bias) in 8-bit integers: x [..., K1] (and x2 [..., K2], the same rows) quantised row by
    row, W as (wq int8 [N, K1 + K2], ws float32 [N]) from quantize_i8, bias float32 [N].  A row of x that holds
    a NaN or an infinity comes out as NaN.  wq's rows are used in place where they start on 16-byte borders
    and are readable to the next one (quantize_i8's are), else copied in the call."""
    tok = TIMER.start(("linear_i8", tuple(x.shape), tuple(wq.shape), str(x.dtype)[6:])) if TIMER.enabled else None
    y = _lib.host().linear_i8(x, wq, ws, bias, x2, relu)
    TIMER.stop(tok)
    return y
