"""The 8-bit integer layer, restated on the CPU: codes from the quotient in 64 bits, the sum exact, the
epilogue in the kernel's fp32 operations (and in 64 bits)."""
import torch

U = 2.0 ** -24


def quantize(x):
    """(codes as float64, scale fp32, top) of x [M, K]."""
    top = x.float().abs().amax(1)
    bad = ~torch.isfinite(top)
    live = ~bad & (top >= 2.0 ** -100)
    one = torch.where(live, top, torch.ones_like(top)).double()
    q = torch.where(live[:, None], x.double() * 127.0 / one[:, None], 0.0).round()
    scale = torch.where(live, top / torch.full_like(top, 127.0), 0.0)
    return torch.where(live[:, None], q, 0.0), torch.where(bad, float("nan"), scale), top


def linear(q, scale, wq, ws, bias, relu, dtype):
    """The kernel's bits: (float(acc) * scale) * ws + bias, one rounding each, then to dtype."""
    acc = (q @ wq.double().t()).to(torch.int64).float()  # (products and sums below 2^53: exact)
    y = (acc * scale[:, None]) * ws
    y = y + (torch.zeros(1) if bias is None else bias)
    return (torch.where(y < 0, 0.0, y) if relu else y).to(dtype)


def linear64(q, top, wq, ws, bias, relu):
    y = (q @ wq.double().t()) * (top.double() / 127)[:, None] * ws.double() + (0.0 if bias is None else bias.double())
    return y.clamp(min=0) if relu else y


def bound(q, top, wq, ws, bias, y64, dtype):
    """The sum to fp32 (1 rounding), the scale (1), two products (2), the bias's sum (1), the store."""
    p = ((q @ wq.double().t()) * (top.double() / 127)[:, None] * ws.double()).abs()
    e = 5 * U * (p + (0.0 if bias is None else bias.double().abs()))
    fi = torch.finfo(dtype)
    return e + fi.eps / 2 * (y64.abs() + e) + fi.smallest_normal * fi.eps
