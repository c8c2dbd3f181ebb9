"""lpgnn.layer_norm on the GPU against the 64-bit reference (tests/norm_ref.py derives the bounds)."""
import pytest
import torch

import norm_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# every lane count and vector count, both sides of each border, rows shorter than a vector and past 2048
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 100, 127, 128, 200, 255, 256, 257, 333, 511, 512, 513, 768,
          1000, 1024, 1025, 1280, 1500, 1792, 1793, 2047, 2048, 2049, 5000]


def _inputs(M, D, dtype, wdtype, seed=0, relu=False):
    g = torch.Generator().manual_seed(seed * 7919 + M * 31 + D)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x = (n(M, D) * (0.5 + n(M, 1).abs()) + 2 * n(M, 1)).to(dtype)
    w, b = (1 + 0.3 * n(D)).to(wdtype), (0.3 * n(D)).to(wdtype)
    dy = n(M, D).to(dtype)
    if relu:  # no gradient where the 32-bit sign of the pre-activation may differ
        y, h, s, _ = R.norm64(x, w, b, EPS, False)
        dy = dy * (y.abs() > R.y_error(x, w, b, y, h, s, torch.float32)).to(dtype)
    return x, w, b, dy


def _run(x, w, b, dy, relu, eps=EPS):
    from lpgnn import layer_norm

    ts = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*ts, eps=eps, relu=relu)
    return (y.detach(), *torch.autograd.grad(y, ts, dy.to(DEV)))


def _check(x, w, b, dy, relu, out, eps=EPS):
    y, h, s, _ = R.norm64(x, w, b, eps, relu)
    assert R.within(out[0], y, R.y_error(x, w, b, y, h, s, x.dtype)) <= 1
    want, bound = R.grads64(x, w, b, dy, eps, relu, x.dtype, w.dtype)
    for got, a, e in zip(out[1:], want, bound):
        assert R.within(got, a, e) <= 1


@pytest.mark.parametrize("dtype,wdtype", [("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp32"),
                                          ("fp16", "fp16")])
@pytest.mark.parametrize("D", WIDTHS)
def test_forward_and_gradients(D, dtype, wdtype):
    for M, relu in ((1, False), (3, True), (130, False), (131, True)):
        case = _inputs(M, D, T[dtype], T[wdtype], relu=relu)
        out = _run(*case, relu)
        assert out[0].dtype == T[dtype] and out[1].dtype == T[dtype] and out[2].dtype == T[wdtype]
        _check(*case, relu, out)


@pytest.mark.parametrize("M,D,dtype", [(20011, 128, "fp32"), (20011, 333, "bf16"), (5003, 2048, "bf16")])
def test_many_rows(M, D, dtype):
    """More rows than the persistent grid takes at once: the row loop and the fold of all partial rows."""
    case = _inputs(M, D, T[dtype], torch.float32)
    out = _run(*case, False)
    _check(*case, False, out)
    again = _run(*case, False)
    assert all(torch.equal(a, b) for a, b in zip(out, again))  # deterministic


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_evaluation_gives_the_training_values(dtype):
    from lpgnn import layer_norm

    x, w, b, dy = _inputs(77, 200, T[dtype], torch.float32, relu=True)
    y = _run(x, w, b, dy, True)[0]
    with torch.no_grad():
        assert torch.equal(layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), EPS, True), y)
    with torch.inference_mode():
        assert torch.equal(layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), EPS, True), y)


def test_without_weight_or_bias():
    from lpgnn import layer_norm

    x, w, b, dy = _inputs(9, 40, torch.float32, torch.float32)
    for ww, bb in ((None, None), (w, None), (None, b)):
        ts = [None if t is None else t.to(DEV).requires_grad_(True) for t in (x, ww, bb)]
        y = layer_norm(*ts, eps=EPS)
        g = torch.autograd.grad(y, [t for t in ts if t is not None], dy.to(DEV))
        yr, h, s, _ = R.norm64(x, ww, bb, EPS, False)
        assert R.within(y.detach(), yr, R.y_error(x, ww, bb, yr, h, s, x.dtype)) <= 1
        want, bound = R.grads64(x, ww, bb, dy, EPS, False, x.dtype, torch.float32)
        keep = [0] + ([1] if ww is not None else []) + ([2] if bb is not None else [])
        for got, k in zip(g, keep):
            assert R.within(got, want[k], bound[k]) <= 1


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_only_the_wanted_gradients(need):
    from lpgnn import layer_norm

    for D in (96, 2500):
        x, w, b, dy = _inputs(21, D, torch.float32, torch.float32)
        ts = [t.to(DEV).requires_grad_(k) for t, k in zip((x, w, b), need)]
        y = layer_norm(*ts, eps=EPS)
        g = torch.autograd.grad(y, [t for t, k in zip(ts, need) if k], dy.to(DEV))
        want, bound = R.grads64(x, w, b, dy, EPS, False, x.dtype, w.dtype)
        for got, a, e in zip(g, [a for a, k in zip(want, need) if k], [e for e, k in zip(bound, need) if k]):
            assert R.within(got, a, e) <= 1


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides_offsets_and_shapes(dtype):
    """Rows inside a wider buffer at an odd element offset, a transposed input, an expanded gradient, more
    dimensions, no rows."""
    from lpgnn import layer_norm

    M, D = 37, 75
    x, w, b, dy = _inputs(M, D, T[dtype], torch.float32)
    wide = torch.full((M, D + 9), float("nan"), dtype=T[dtype], device=DEV)
    wide[:, 3:3 + D] = x.to(DEV)
    gw = torch.full((M, D + 5), float("nan"), dtype=T[dtype], device=DEV)
    gw[:, 1:1 + D] = dy.to(DEV)
    wd, bd = w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)
    for xv in (wide[:, 3:3 + D], x.to(DEV).t().contiguous().t()):
        xv = xv.requires_grad_(True)
        y = layer_norm(xv, wd, bd, EPS)
        _check(x, w, b, dy, False, (y.detach(), *torch.autograd.grad(y, (xv, wd, bd), gw[:, 1:1 + D])))
        xv.requires_grad_(False) if xv.is_leaf else None
    one = dy[:1].expand(M, D)
    xv = x.to(DEV).requires_grad_(True)
    y = layer_norm(xv, wd, bd, EPS)
    _check(x, w, b, one, False, (y.detach(), *torch.autograd.grad(y, (xv, wd, bd), dy[:1].to(DEV).expand(M, D))))
    x3 = x[:36].view(4, 9, D).to(DEV)
    assert torch.equal(layer_norm(x3, wd, bd, EPS).view(36, D), layer_norm(x.to(DEV), wd, bd, EPS)[:36])
    empty = torch.empty(0, D, dtype=T[dtype], device=DEV, requires_grad=True)
    y = layer_norm(empty, wd, bd, EPS)
    gx, gww, gbb = torch.autograd.grad(y, (empty, wd, bd), torch.empty_like(y))
    assert y.shape == (0, D) and gx.shape == (0, D) and not gww.any() and not gbb.any()


def test_far_mean_and_constant_rows():
    """|mean| thousands of times the spread (a one-pass variance would have no digits), and rows without
    spread, whose h is 0 and whose gradient is scaled by 1 / sqrt(eps)."""
    M, D = 16, 256
    x, w, b, dy = _inputs(M, D, torch.float32, torch.float32)
    x = (x.double() * 0.1 + 1000).float()
    x[5] = 3.0
    x[6] = 0.0
    _check(x, w, b, dy, False, _run(x, w, b, dy, False))


def test_bad_rows_stay_in_their_rows():
    from lpgnn import layer_norm

    for D in (8, 200, 2048, 3000):
        x, w, b, _ = _inputs(9, D, torch.float32, torch.float32)
        clean = layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), EPS, True)
        x[2, D // 2], x[4, 0], x[7, D - 1] = float("nan"), float("inf"), float("-inf")
        y = layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), EPS, True)
        for r in range(9):
            if r in (2, 4, 7):
                assert torch.isnan(y[r]).all()
            else:
                assert torch.equal(y[r], clean[r])


def test_gradient_against_differences():
    """The kernel's gradients against central differences of the 64-bit definition along random directions:
    its bound along the direction, and 1e-7 for the differences."""
    x, w, b, dy = _inputs(6, 50, torch.float32, torch.float32)
    got = _run(x, w, b, dy, False)[1:]
    _, bound = R.grads64(x, w, b, dy, EPS, False, x.dtype, w.dtype)
    f = lambda *a: (R.norm64(*a, EPS, False)[0] * dy.double()).sum()
    ts = [t.double() for t in (x, w, b)]
    for k in range(3):
        d = torch.randn(ts[k].shape, generator=torch.Generator().manual_seed(k), dtype=torch.float64)
        hi, lo = list(ts), list(ts)
        hi[k], lo[k] = ts[k] + 1e-5 * d, ts[k] - 1e-5 * d
        diff = (f(*hi) - f(*lo)) / 2e-5
        assert abs(diff - (got[k].double().cpu() * d).sum()) <= (bound[k] * d.abs()).sum() + 1e-6


def test_on_another_stream_and_in_a_graph():
    from lpgnn import layer_norm

    x, w, b, dy = (t.to(DEV) for t in _inputs(300, 128, torch.float32, torch.float32))
    ts = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = layer_norm(*ts, eps=EPS)
    want = (want.detach(), *torch.autograd.grad(want, ts, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer_norm(*ts, eps=EPS)
        got = (y.detach(), *torch.autograd.grad(y, ts, dy))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del y, got
    # captured with its backward, replayed on new inputs, eager work between the replays
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(*ts, eps=EPS)
        held = (y.detach(), *torch.autograd.grad(y, ts, dy))
    for k in range(3):
        with torch.no_grad():
            ts[0].copy_(x * (k + 1) + k)
        graph.replay()
        torch.cuda.synchronize()
        e = [t.detach().clone().requires_grad_(True) for t in ts]
        ye = layer_norm(*e, eps=EPS)
        assert all(torch.equal(a, b) for a, b in zip(held, (ye.detach(), *torch.autograd.grad(ye, e, dy))))


def test_refusals():
    from lpgnn import layer_norm

    x = torch.randn(4, 8, device=DEV)
    for bad, msg in ((dict(weight=torch.ones(7, device=DEV)), "weight must be"),
                     (dict(weight=torch.ones(8)), "weight must be"),
                     (dict(bias=torch.ones(8, dtype=torch.float16, device=DEV)), "bias must be"),
                     (dict(eps=-1.0), "eps")):
        with pytest.raises(RuntimeError, match=msg):
            layer_norm(x, **bad)
    with pytest.raises(RuntimeError, match="share a type"):
        layer_norm(x.half(), torch.ones(8, device=DEV), torch.ones(8, dtype=torch.float16, device=DEV))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        layer_norm(x.double())
    with pytest.raises(RuntimeError, match="last dimension"):
        layer_norm(torch.empty(3, 0, device=DEV))
    xr = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(layer_norm(xr).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_capture_beside_an_eager_graph_is_refused():
    """A captured forward whose backward would meet the eager graph's gradient accumulators (of another stream) is
    refused before anything is recorded; after the eager graph is gone it is captured."""
    from lpgnn import layer_norm

    x = torch.randn(8, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    alive = layer_norm(x, w).sum()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(graph):
            layer_norm(x, w)
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(x, w)
        y = layer_norm(y, w)  # the same leaf twice in one capture
        g, = torch.autograd.grad(y.sum(), w)
    graph.replay()
    torch.cuda.synchronize()
    e = layer_norm(layer_norm(x, w), w)
    assert torch.equal(y, e) and torch.equal(g, torch.autograd.grad(e.sum(), w)[0])


def test_gradient_of_a_gradient_raises():
    """Also where it is one term beside others, which have one."""
    from lpgnn import layer_norm

    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y = layer_norm(x, w).square().sum()
    gx, gw = torch.autograd.grad(y, (x, w), create_graph=True)
    plain = torch.autograd.grad(layer_norm(x, w).square().sum(), (x, w))
    assert torch.equal(gx, plain[0]) and torch.equal(gw, plain[1])
    for g in (gx, gw):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y + g.square().sum(), x, retain_graph=True)


def test_more_elements_than_32_bits_count():
    """Offsets past 2^31 elements: the last rows are those of a small call."""
    from lpgnn import layer_norm

    D = 512
    M = 2**31 // D + 501
    x = torch.zeros(M, D, dtype=torch.float16, device=DEV)
    x[-700:].normal_()
    dy = torch.zeros_like(x)
    dy[-700:].normal_()
    w = (torch.rand(D, device=DEV) + 0.5).requires_grad_(True)
    xs = x[-700:].clone().requires_grad_(True)
    small = layer_norm(xs, w)
    gs = torch.autograd.grad(small, xs, dy[-700:])[0]
    x.requires_grad_(True)
    y = layer_norm(x, w)
    g, gw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(y[-700:], small) and torch.equal(g[-700:], gs)
    assert y[:100].count_nonzero() == 0 and g[:100].count_nonzero() == 0 and gw.isfinite().all()


def test_gradients_of_shared_and_broadcast_inputs():
    """x, weight and bias that are expanded, strided, of more dimensions, or one tensor for both: autograd adds up
    what the kernel gives, as with copies."""
    from lpgnn import layer_norm

    M, D = 36, 40
    x, w, _, dy = (t.to(DEV) for t in _inputs(M, D, torch.float32, torch.float32))

    def grads(make, leaves, shape=(M, D)):
        return torch.autograd.grad(make(), leaves, dy.view(shape))

    def copies(xc, wc, bc):
        ts = [t.detach().clone().contiguous().requires_grad_(True) for t in (xc, wc, bc)]
        return torch.autograd.grad(layer_norm(*ts, eps=EPS), ts, dy)

    one = x[:1].clone().requires_grad_(True)  # every row the same one
    base = torch.ones(D, 2, device=DEV).mul_(w[:, None]).requires_grad_(True)  # weight and bias its two columns
    gx, gw, gb = copies(one.expand(M, D), base[:, 0], base[:, 1])
    got = grads(lambda: layer_norm(one.expand(M, D), base[:, 0], base[:, 1], EPS), (one, base))
    assert torch.equal(got[0], gx.sum(0, keepdim=True)) and torch.equal(got[1], torch.stack((gw, gb), 1))

    xs, both = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw, gb = copies(xs, both, both)
    got = grads(lambda: layer_norm(xs, both, both, EPS), (xs, both))
    assert torch.equal(got[0], gx) and torch.equal(got[1], gw + gb)

    scalar = torch.full((1,), 0.7, device=DEV, requires_grad=True)
    x3 = x.view(4, 9, D).transpose(0, 1).detach().requires_grad_(True)  # rows that no view holds
    xp = x.view(4, 9, D).transpose(0, 1).reshape(M, D)
    ts = [xp.clone().requires_grad_(True), scalar.detach().expand(D).clone().requires_grad_(True)]
    want = torch.autograd.grad(layer_norm(ts[0], ts[1], None, EPS), ts, dy)
    got = grads(lambda: layer_norm(x3, scalar.expand(D), None, EPS), (x3, scalar), (9, 4, D))
    assert torch.equal(got[0].reshape(M, D), want[0])
    assert abs(got[1] - want[1].double().sum()) <= D * 2.0**-24 * want[1].abs().double().sum()

    v = x[0].clone().requires_grad_(True)  # one row, one dimension
    y = layer_norm(v, w, None, EPS)
    g, = torch.autograd.grad(y, v, dy[0])
    r = x[:1].clone().requires_grad_(True)
    want, = torch.autograd.grad(layer_norm(r, w, None, EPS), r, dy[:1])
    assert y.shape == (D,) and torch.equal(g, want[0])


def test_capture_beside_an_eager_graph_of_a_view_is_refused():
    """The parameters of the call may be views or casts of the leaves that the eager graph holds; within one capture
    they may be used as often as wanted."""
    from lpgnn import layer_norm

    x = torch.randn(8, 16, device=DEV)
    both = torch.rand(2, 16, device=DEV).add_(0.5).requires_grad_(True)  # weight and bias its two rows

    def norm(x):
        return layer_norm(x, both[0], both[1].clone())

    alive = norm(x).sum()
    for make in (lambda: norm(x), lambda: layer_norm(x + both[0])):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(graph):
                make()
        torch.cuda.synchronize()
    del alive, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = norm(norm(x))
        g, = torch.autograd.grad(y.sum(), both)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        e = norm(norm(x))
        eg, = torch.autograd.grad(e.sum(), both)
        assert torch.equal(y, e) and torch.equal(g, eg)
        del e, eg


@pytest.mark.parametrize("M,D,dtype", [(20011, 128, "fp32"), (20011, 300, "fp32"), (5003, 2048, "fp32"), (20011, 333, "bf16"),
                                       (9001, 1000, "bf16"), (5003, 2048, "bf16"), (30001, 100, "fp16")])
def test_relu_backward_of_many_rows(M, D, dtype):
    """The form a normed GCN_FC trains with, over more rows than the grid takes at once: one and two rows a lane group
    at a time, with and without the next rows loaded ahead."""
    case = _inputs(M, D, T[dtype], torch.float32, relu=True)
    out = _run(*case, True)
    _check(*case, True, out)
    again = _run(*case, True)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("M,D,dtype", [(3001, 2500, "fp32"), (2051, 2049, "bf16"), (70001, 3, "fp32"), (70001, 5, "bf16"),
                                       (70001, 1, "fp16")])
def test_many_rows_of_a_block_each(M, D, dtype, relu):
    """Rows longer than 2048 or shorter than a vector, more of them than blocks: the blocks' second rows, the weight
    gradients' second row a grid row, the fold of all partial rows."""
    case = _inputs(M, D, T[dtype], torch.float32, relu=relu)
    out = _run(*case, relu)
    _check(*case, relu, out)
    again = _run(*case, relu)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_rows_past_the_range_of_their_squares():
    """Finite rows whose sum of squares no fp32 number holds come out as the bias; the ones beside them do not notice."""
    from lpgnn import layer_norm

    for D in (64, 300, 2100):
        x, w, b, _ = (t.to(DEV) for t in _inputs(5, D, torch.float32, torch.float32))
        clean = layer_norm(x, w, b, EPS)
        x[3] = x[3] / x[3].abs().max() * 1e22
        y = layer_norm(x, w, b, EPS)
        assert torch.equal(y[3], b) and torch.equal(y[[0, 1, 2, 4]], clean[[0, 1, 2, 4]])
