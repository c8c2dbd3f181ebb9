"""lpgnn.layer_norm on the CPU: its refusals (before any device work) and the 64-bit reference the GPU
tests use, against differences."""
import pytest
import torch

import norm_ref as R


def test_refuses_host_tensors_and_bad_arguments():
    from lpgnn import layer_norm

    with pytest.raises(RuntimeError, match="no CPU path"):
        layer_norm(torch.ones(2, 4))


def test_c_entry_refusals():
    from lpgnn import _lib

    L = _lib.lib()
    p = 1 << 20  # never dereferenced: each call is refused before any launch

    def fwd(dtype=2, wdtype=2, M=4, D=8, x=p, ldx=8, eps=1e-5, flags=0, y=p, ldy=8, mean=None, rstd=None):
        return L.lpg_layer_norm_fwd(dtype, wdtype, M, D, x, ldx, p, p, eps, flags, y, ldy, mean, rstd, None)

    for kw in (dict(dtype=3), dict(dtype=2, wdtype=0), dict(dtype=0, wdtype=1), dict(M=-1), dict(D=0), dict(ldx=7),
               dict(ldy=7), dict(eps=-1.0), dict(eps=float("nan")), dict(flags=2), dict(x=None), dict(y=None),
               dict(mean=p), dict(D=1 << 31, ldx=1 << 31, ldy=1 << 31)):
        assert fwd(**kw) == 1, kw
        assert b"lpg_layer_norm_fwd" in L.lpg_last_error(), kw
    assert fwd(M=0, x=None, y=None) == 0

    def bwd(dtype=2, wdtype=2, M=4, D=8, x=p, ldx=8, dy=p, lddy=8, mean=p, flags=0, dx=p, lddx=8, dw=p, ws=p):
        return L.lpg_layer_norm_bwd(dtype, wdtype, M, D, x, ldx, dy, lddy, p, p, mean, p, flags, dx, lddx, dw, None, ws,
                                    None)

    for kw in (dict(dtype=7), dict(wdtype=1), dict(M=-1), dict(D=0), dict(ldx=7), dict(lddy=7), dict(lddx=7),
               dict(flags=4), dict(x=None), dict(dy=None), dict(mean=None), dict(ws=None)):
        assert bwd(**kw) == 1, kw
        assert b"lpg_layer_norm_bwd" in L.lpg_last_error(), kw
    assert L.lpg_layer_norm_bwd_workspace_bytes(-1, 8) == -1
    assert L.lpg_layer_norm_bwd_workspace_bytes(0, 8) == 64
    assert L.lpg_layer_norm_bwd_workspace_bytes(10 ** 6, 1024) == 1024 * 2 * 1024 * 4


def test_module_names_and_state():
    from lpgnn import LayerNorm

    n = LayerNorm(16)
    assert list(n.state_dict()) == ["weight", "bias"]
    assert n.weight.eq(1).all() and n.bias.eq(0).all()
    n.load_state_dict(torch.nn.LayerNorm(16).state_dict())


@pytest.mark.parametrize("relu", [False, True])
def test_reference_gradients_against_differences(relu):
    """The oracle's own gradients: central differences of the 64-bit forward (step 1e-5: error below 1e-8 here)."""
    g = torch.Generator().manual_seed(1)
    M, D, eps = 5, 7, 1e-5
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w, b, dy = n(M, D), 1 + 0.3 * n(D), 0.3 * n(D), n(M, D)
    pre = R.norm64(x, w, b, eps, False)[0]
    dy = dy * (pre.abs() > 1e-3)  # no difference across the ReLU's corner
    got = R.grads64(x, w, b, dy, eps, relu, torch.float64, torch.float64)[0]
    f = lambda x, w, b: (R.norm64(x, w, b, eps, relu)[0] * dy).sum()
    for k, t in enumerate((x, w, b)):
        d = n(*t.shape)
        hi, lo = [x, w, b], [x, w, b]
        hi[k], lo[k] = t + 1e-5 * d, t - 1e-5 * d
        diff = (f(*hi) - f(*lo)) / 2e-5
        assert abs(diff - (got[k] * d).sum()) < 1e-7


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_refuses_forward_mode_tangents(which):
    """A dual tensor would come out without its tangent, which reads as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    from lpgnn import layer_norm

    ts = dict(x=torch.ones(2, 4), weight=torch.ones(4), bias=torch.ones(4))
    with fwd.dual_level():
        ts[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                layer_norm(**ts)
