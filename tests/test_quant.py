"""lpgnn.linear_i8 on the CPU: refusals before any device work."""
import pytest
import torch


def test_refuses_host_tensors():
    from lpgnn import linear_i8, quantize_i8

    x = torch.ones(2, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        quantize_i8(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear_i8(x, torch.ones(4, 16, dtype=torch.int8), torch.ones(4))


def test_c_entry_refusals():
    from lpgnn import _lib

    L = _lib.lib()
    p = 1 << 20  # 16-byte aligned, never dereferenced

    def qz(dtype=2, M=4, K1=8, x=p, ldx=8, K2=8, x2=p, ldx2=8, q=p, ldq=128, s=p):
        return L.lpg_quant_i8(dtype, M, K1, x, ldx, K2, x2, ldx2, q, ldq, s, None)

    for kw in (dict(dtype=3), dict(M=-1), dict(K1=0), dict(K2=-1), dict(ldx=7), dict(ldx2=7), dict(ldq=120),
               dict(K1=128, ldx=128), dict(x=None), dict(x2=None), dict(q=None), dict(s=None), dict(q=p + 8),
               dict(K1=131072, ldx=131072, ldq=131072 + 128), dict(K1=1 << 62, ldx=1 << 62)):
        assert qz(**kw) == 1 and b"lpg_quant_i8" in L.lpg_last_error(), kw
    assert qz(M=0, x=None, q=None, s=None, x2=None) == 0

    def fc(dtype=2, M=4, N=4, K=100, q=p, ldq=128, s=p, w=p, ldw=112, ws=p, flags=0, y=p, ldy=4):
        return L.lpg_fc_i8(dtype, M, N, K, q, ldq, s, w, ldw, ws, None, flags, y, ldy, None)

    for kw in (dict(dtype=-1), dict(M=-1), dict(N=0), dict(K=0), dict(K=129), dict(ldq=127), dict(ldw=96), dict(ldw=120),
               dict(flags=2), dict(ldy=3), dict(q=None), dict(s=None), dict(w=None), dict(ws=None), dict(y=None),
               dict(q=p + 1), dict(w=p + 8), dict(K=131073, ldq=131200, ldw=131088), dict(M=1 << 40, N=1 << 30, ldy=1 << 30)):
        assert fc(**kw) == 1 and b"lpg_fc_i8" in L.lpg_last_error(), kw
    assert fc(M=0, q=None, s=None, y=None) == 0

    def rw(dtype=2, M=2, N=4, K1=50, x=p, ldx=50, K2=50, x2=p, ldx2=50, w=p, ldw=112, ws=p, flags=0, y=p, ldy=4):
        return L.lpg_fc_i8_rows(dtype, M, N, K1, x, ldx, K2, x2, ldx2, w, ldw, ws, None, flags, y, ldy, None)

    for kw in (dict(dtype=9), dict(M=-1), dict(N=0), dict(K1=0), dict(K2=-1), dict(ldx=49), dict(ldx2=49),
               dict(ldw=96), dict(ldw=104), dict(flags=4), dict(ldy=3), dict(x=None), dict(x2=None), dict(w=None),
               dict(ws=None), dict(y=None), dict(w=p + 4)):
        assert rw(**kw) == 1 and b"lpg_fc_i8_rows" in L.lpg_last_error(), kw
    assert rw(M=2, K1=6200, ldx=6200, ldw=6256) == 3  # more LDS than the entry takes
    assert rw(M=1, K1=40000, ldx=40000, ldw=40064) == 3
    assert rw(M=1 << 20) == 3  # too many rows for one launch
    assert rw(M=0, x=None, x2=None, y=None) == 0


def test_chunk_rows():
    from lpgnn import _lib

    f = _lib.lib().lpg_i8_chunk_rows
    assert f(-1, 8, 8) == f(8, 0, 8) == f(8, 8, 0) == -1
    assert f(0, 8, 8) == 0 and f(100, 1024, 2048) == 100
    for M, N, K in ((10 ** 5, 1024, 2048), (10 ** 6, 100, 100), (10 ** 6, 2048, 4096), (10 ** 6, 10 ** 6, 131072)):
        rows = f(M, N, K)
        assert 0 < rows <= M and (rows == M or rows % 256 == 0)


@pytest.mark.parametrize("which", ["x", "x2", "ws", "bias"])
def test_refuses_forward_mode_tangents(which):
    """A dual tensor would come out without its tangent, which reads as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    from lpgnn import linear_i8, quantize_i8

    ts = dict(x=torch.ones(2, 16), x2=torch.ones(2, 16), ws=torch.ones(4), bias=torch.ones(4))
    with fwd.dual_level(), torch.no_grad():
        ts[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear_i8(wq=torch.ones(4, 32, dtype=torch.int8), **ts)
        if which in ("x", "x2"):
            with pytest.raises(RuntimeError, match="forward-mode"):
                quantize_i8(ts["x"], ts["x2"])


@pytest.mark.parametrize("which", ["x", "x2", "ws", "bias"])
def test_refuses_whatever_wants_a_gradient(which):
    from lpgnn import linear_i8

    ts = dict(x=torch.ones(2, 16), x2=torch.ones(2, 16), ws=torch.ones(4), bias=torch.ones(4))
    ts[which].requires_grad_(True)
    wq = torch.ones(4, 32, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_i8(wq=wq, **ts)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):  # (what a host tensor is refused for)
        linear_i8(wq=wq, **ts)


def test_c_entry_of_one_row_refuses_more_blocks_than_a_launch_holds():
    """Four columns a block of 256 threads, fewer than 2^32 threads a launch: the two launches take it."""
    from lpgnn import _lib

    p, N = 1 << 20, 1 << 26
    assert _lib.lib().lpg_fc_i8_rows(2, 1, N, 16, p, 16, 0, None, 0, p, 16, p, None, 0, p, N, None) == 3


def test_c_entry_of_few_rows_ends_at_1024_columns():
    from lpgnn import _lib

    p = 1 << 20
    rw = lambda M, K1, K2: _lib.lib().lpg_fc_i8_rows(2, M, 64, K1, p, K1, K2, p, K2, p, 4096, p, None, 0, p, 64, None)
    for M in (2, 16, 64):
        assert rw(M, 1025, 0) == rw(M, 1000, 25) == rw(M, 1, 1024) == 3
