"""Layer norm and its gradients in 64 bits, with the error a 32-bit evaluation may have.

U = 2^-24 is the half step of fp32.  A sum of the kernels takes at most 32 terms a lane, 6 butterfly
levels and 4 wave partials one after another (rows beyond 2048 elements: D / 256 terms a thread), so its
relative error against the sum of magnitudes is below n_sum * U, n_sum = 64 + D / 256."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm64(x, w, b, eps, relu):
    """(y, h, s, mu) in 64 bits of x [M, D]."""
    x = x.double()
    mu = x.mean(1, keepdim=True)
    s = 1 / ((x - mu).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - mu) * s
    z = h * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    return (z.clamp(min=0) if relu else z), h, s, mu


def h_error(x, h, s):
    """|error of h|: the mean's (n_sum U mean|x|), the subtraction's and the scale's (half the variance's, the
    quotient, root and reciprocal: below n_sum U)."""
    n = (64 + x.shape[1] / 256) * U
    x = x.double().abs()
    return n * ((x.mean(1, keepdim=True) + x) * s + h.abs())


def y_error(x, w, b, y, h, s, dtype):
    wa = 1.0 if w is None else w.double().abs()
    ba = 0.0 if b is None else b.double().abs()
    e = h_error(x, h, s) * wa + 2 * U * (h.abs() * wa + ba)
    return e + half_step(dtype) * (y.abs() + e) + torch.finfo(dtype).smallest_normal * half_step(dtype)


def grads64(x, w, b, dy, eps, relu, dtype, wdtype):
    """((dx, dw, db), (their error bounds)) in 64 bits."""
    _, h, s, _ = norm64(x, w, b, eps, relu)
    D, M = x.shape[1], x.shape[0]
    wd = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    z = dy.double()
    if relu:
        z = z * (norm64(x, w, b, eps, False)[0] > 0)
    zw = z * wd
    c1, c2 = zw.mean(1, keepdim=True), (zw * h).mean(1, keepdim=True)
    dx = s * (zw - c1 - h * c2)
    dw, db = (z * h).sum(0), z.sum(0)
    eh = h_error(x, h, s)
    n = (64 + D / 256) * U
    e1 = n * zw.abs().mean(1, keepdim=True)
    e2 = (zw.abs() * eh).mean(1, keepdim=True) + n * (zw * h).abs().mean(1, keepdim=True)
    e = s * (4 * U * (zw.abs() + c1.abs() + (h * c2).abs()) + e1 + h.abs() * e2 + eh * c2.abs()) + n * dx.abs()
    e = e + half_step(dtype) * (dx.abs() + e) + torch.finfo(dtype).smallest_normal * half_step(dtype)
    rows = (96 + M / 64) * U  # a lane's rows, 6 levels, 4 waves, the fold's 64 + 16 terms
    hw, tiny = half_step(wdtype), torch.finfo(wdtype).smallest_normal * half_step(wdtype)
    ew = (z.abs() * eh).sum(0) + rows * (z * h).abs().sum(0)
    eb = rows * z.abs().sum(0)
    return (dx, dw, db), (e, ew + hw * (dw.abs() + ew) + tiny, eb + hw * (db.abs() + eb) + tiny)


def within(got, want, bound):
    """The largest |got - want| / bound (a number at or below 1 passes)."""
    d = (got.double().cpu() - want).abs()
    assert torch.isfinite(d).all()
    return (d / bound.clamp(min=1e-300)).max().item() if d.numel() else 0.0
