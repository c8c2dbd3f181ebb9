"""lpgnn.optim on the GPU.  The kernels' fp32 operations are single roundings in a fixed order, restated in
tests/adamw_ref.py: the results have to be its bits; and the 64-bit formula within derived bounds."""
import math

import pytest
import torch

import adamw_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
SIZES = [0, 1, 3, 4, 5, 255, 256, 257, 1000, 4095, 4096, 4097, 16384, 16385, 70001]
H = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def _lists(sizes, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda k: torch.randn(k, generator=g)
    size = [10.0 ** -(2 + i % 3) for i in range(len(sizes))]
    p = [n(k).to(dtype) for k in sizes]
    gr = [(n(k) * z).to(dtype) for k, z in zip(sizes, size)]
    m = [0.2 * n(k) * z for k, z in zip(sizes, size)]
    v = [((0.3 + n(k).abs()) * z) ** 2 for k, z in zip(sizes, size)]
    return p, gr, m, v


def _dev(ts, offset=0):
    """Copies on the device, each inside a buffer of NaN at this element offset; (tensors, buffers)."""
    bufs = [torch.full((t.numel() + offset + 9,), float("nan"), device=DEV).to(t.dtype) for t in ts]
    for b, t in zip(bufs, ts):
        b[offset:offset + t.numel()] = t.to(DEV)
    return [b[offset:offset + t.numel()] for b, t in zip(bufs, ts)], bufs


def _untouched(bufs, sizes, offset):
    return all(b[:offset].isnan().all() and b[offset + k:].isnan().all() for b, k in zip(bufs, sizes))


def _p_bound(p, g, m, v, t, p64, m64, v64, scale=1.0):
    """m takes 5 roundings (two constants, two products, the sum; the gradient's scale), v 8, its root 4 in
    relative terms, the denominator 7, the quotient and rate 12; p two products and the difference."""
    b1, b2 = H["betas"]
    em = 5 * U * (b1 * m.double().abs() + (1 - b1) * scale * g.double().abs())
    d = v64.sqrt() / math.sqrt(1 - b2 ** t) + H["eps"]
    rate = H["lr"] / (1 - b1 ** t)
    e = 4 * U * (p.double().abs() + p64.abs()) + rate * (em / d + 12 * U * m64.abs() / d)
    return e + (torch.finfo(p.dtype).eps / 2) * (p64.abs() + e), em, 8 * U * v64


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("t", [1, 1000])
def test_step(dtype, offset, t):
    from lpgnn import optim

    host = _lists(SIZES, dtype)
    (p, pb), (g, gb), (m, mb), (v, vb) = (_dev(x, offset) for x in host)
    optim.adamw_step(p, g, m, v, step=t, **H)
    for i in range(len(SIZES)):
        a = [x[i] for x in host]
        want = R.step32(*a, t, **H)
        for got, w in zip((p[i], m[i], v[i]), want):
            assert torch.equal(got.cpu(), w.to(got.dtype)), SIZES[i]
        p64, m64, v64 = R.step64(*a, t, **H)
        bp, bm, bv = _p_bound(*a, t, p64, m64, v64)
        for got, w, b in ((p[i], p64, bp), (m[i], m64, bm), (v[i], v64, bv)):
            assert ((got.cpu().double() - w).abs() <= b).all(), SIZES[i]
        assert torch.equal(g[i].cpu(), host[1][i])
    for bufs in (pb, gb, mb, vb):
        assert _untouched(bufs, SIZES, offset)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_step_8bit(dtype, offset):
    """Three steps from nothing: codes, scales and parameters are the reference's bits; the moments are within
    a step of their format of the 64-bit ones."""
    from lpgnn import optim

    host = _lists(SIZES, dtype, seed=3)
    p, pb = _dev(host[0], offset)
    f8 = torch.float8_e4m3fn
    new8 = lambda: [torch.zeros(k + offset + 9, dtype=torch.uint8, device=DEV) for k in SIZES]
    cut = lambda bs: [b.view(f8)[offset:offset + k] for b, k in zip(bs, SIZES)]
    mb, rb = new8(), new8()
    for b, k in zip(mb + rb, SIZES + SIZES):
        b[:offset], b[offset + k:] = 0x5A, 0x5A
    m8, r8 = cut(mb), cut(rb)
    nb = [-(-k // 256) for k in SIZES]
    ms, rs = ([torch.zeros(k, device=DEV) for k in nb] for _ in range(2))
    ref = [(x.float(), torch.zeros(k), torch.zeros(n), torch.zeros(k), torch.zeros(n))
           for x, k, n in zip(host[0], SIZES, nb)]
    for t in (1, 2, 3):
        grads = _lists(SIZES, dtype, seed=10 + t)[1]
        optim.adamw_step_8bit(p, [x.to(DEV) for x in grads], m8, ms, r8, rs, step=t, seed=(3 << 32) | 77, **H)
        for i, k in enumerate(SIZES):
            old = ref[i]
            out = R.step8(old[0].to(dtype), grads[i], *old[1:], t, R.key(i, t, (3 << 32) | 77), **H)
            ref[i] = (out[0].to(dtype).float(), *out[1:])
            assert torch.equal(p[i].cpu(), out[0].to(dtype)), (t, k)
            for got, w in zip((m8[i], ms[i], r8[i], rs[i]), out[1:]):
                assert torch.equal(got.float().cpu(), w), (t, k)
            m0, r0 = R.decode(old[1], old[2], k), R.decode(old[3], old[4], k)
            _, m64, v64 = R.step64(old[0], grads[i], m0, r0.double() ** 2, t, **H)
            for q, s, want in ((out[1], out[2], m64), (out[3], out[4], v64.sqrt())):
                s = s.double().repeat_interleave(256)[:k]
                x = want.abs() / s.clamp(min=1e-300)
                step = torch.exp2(torch.frexp(x).exponent.sub(1).clamp(min=-6) - 3.0)
                assert ((q.double() * s - want).abs() <= step * s * (1 + 1e-5)).all()
    assert _untouched(pb, SIZES, offset)
    for b, k in zip(mb + rb, SIZES + SIZES):
        assert (b[:offset] == 0x5A).all() and (b[offset + k:] == 0x5A).all()


def test_8bit_format_is_torch_float8():
    """Every code: the kernel's decoding (a step with betas 0 < 1 and no gradient keeps m's sign and order)."""
    from lpgnn import optim

    codes = torch.arange(256, dtype=torch.uint8)
    codes[0x7F], codes[0xFF] = 0, 0  # (NaN)
    m8 = codes.view(torch.float8_e4m3fn).to(DEV)
    ms = torch.ones(1, device=DEV)
    r8, rs = torch.zeros(256, device=DEV).to(torch.float8_e4m3fn), torch.zeros(1, device=DEV)
    p = torch.zeros(256, device=DEV)
    # p = -(m b1 / eps) lr / (1 - b1) with no gradient and no r: b1 = 0.5, eps = 1, lr = 1: p = -m exactly
    optim.adamw_step_8bit([p], [torch.zeros_like(p)], [m8], [ms], [r8], [rs], step=1, lr=1.0, betas=(0.5, 0.5), eps=1.0,
                          weight_decay=0.0)
    assert torch.equal(-p.cpu(), codes.view(torch.float8_e4m3fn).float())
    assert torch.equal(ms.cpu(), torch.full((1,), 224.0) / 448) and not rs.any() and not r8.float().any()


@pytest.mark.parametrize("bits", [8, 32])
def test_many_tensors_and_grad_scale(bits):
    """More tensors than one launch's table, a scale on the device."""
    from lpgnn import optim

    sizes = [1 + (37 * i) % 700 for i in range(300)]
    host = _lists(sizes, seed=5)
    p, g = ([x.to(DEV) for x in ts] for ts in host[:2])
    s = torch.tensor(0.37, device=DEV)
    if bits == 32:
        m, v = ([x.to(DEV) for x in ts] for ts in host[2:])
        optim.adamw_step(p, g, m, v, step=9, grad_scale=s, **H)
        for i in range(300):
            want = R.step32(*(x[i] for x in host), 9, scale=0.37, **H)
            assert all(torch.equal(a.cpu(), b) for a, b in zip((p[i], m[i], v[i]), want))
        return
    nb = [-(-k // 256) for k in sizes]
    f8 = lambda: [torch.zeros(k, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for k in sizes]
    m8, r8 = f8(), f8()
    ms, rs = ([torch.zeros(k, device=DEV) for k in nb] for _ in range(2))
    optim.adamw_step_8bit(p, g, m8, ms, r8, rs, step=9, seed=1, grad_scale=s, **H)
    for i, (k, b) in enumerate(zip(sizes, nb)):
        z = torch.zeros(k)
        want = R.step8(host[0][i], host[1][i], z, torch.zeros(b), z, torch.zeros(b), 9, R.key(i, 9, 1), scale=0.37, **H)
        assert all(torch.equal(a.float().cpu(), w) for a, w in zip((p[i], m8[i], ms[i], r8[i], rs[i]), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clip_scale(dtype):
    """The norm is the fp64 sum's, rounded once (its own error below 2^-40), so within 2^-24."""
    from lpgnn import optim

    for sizes in (SIZES, [5], [1 + i % 300 for i in range(500)]):
        g = _lists(sizes, dtype, seed=len(sizes))[1]
        want = math.sqrt(sum((x.double() ** 2).sum().item() for x in g))
        for most in (0.0, want / 3, want, 1e9):
            norm, scale = optim.clip_scale([x.to(DEV) for x in g], most)
            assert abs(norm.item() - want) <= U * 1.01 * want
            f = min(1.0, most / (want + 1e-6))
            assert abs(scale.item() - f) <= U * 1.01 * f
    for off in (1, 3):  # any alignment
        t, bufs = _dev(_lists([40001], dtype)[1], off)
        assert abs(optim.clip_scale(t, 1.0)[0].item() - t[0].double().norm().item()) <= 2 * U * t[0].double().norm().item()
    x = torch.ones(1000, device=DEV, dtype=dtype)
    for bad in (float("nan"), float("inf")):
        x[500] = bad
        norm, scale = optim.clip_scale([x], 1.0)
        assert not math.isfinite(norm.item()) and not scale.item() > 0
    x.fill_(1e30)  # squares past fp32's range
    assert abs(optim.clip_scale([x], 1.0)[0].item() / (x.double().norm().item()) - 1) < 1e-6


def test_bad_numbers_stay_in_their_block():
    from lpgnn import optim

    p = torch.zeros(1024, device=DEV)
    g = torch.randn(1024, device=DEV)
    g[300], g[600] = float("nan"), float("inf")
    z = lambda n, dt: torch.zeros(n, dtype=torch.uint8 if dt is None else dt, device=DEV)
    m8, r8 = (z(1024, None).view(torch.float8_e4m3fn) for _ in range(2))
    ms, rs = z(4, torch.float32), z(4, torch.float32)
    optim.adamw_step_8bit([p], [g], [m8], [ms], [r8], [rs], step=1, **H)
    for s in (ms, rs):
        assert s.isnan().tolist() == [False, True, True, False]
    assert p[300].isnan() and p[:256].isfinite().all() and p[768:].isfinite().all()
    g.fill_(0.5)
    optim.adamw_step_8bit([p], [g], [m8], [ms], [r8], [rs], step=2, **H)
    assert p[256:768].isnan().all() and p[:256].isfinite().all() and p[768:].isfinite().all()
    # gradients so small that a block's moments are below the format: zeros, and no division by them
    g.fill_(1e-33)
    p2 = torch.zeros(1024, device=DEV)
    a = [z(1024, None).view(torch.float8_e4m3fn) for _ in range(2)] + [z(4, torch.float32) for _ in range(2)]
    optim.adamw_step_8bit([p2], [g], [a[0]], [a[2]], [a[1]], [a[3]], step=1, **H)
    assert not a[2].any() and not a[0].float().any() and p2.isfinite().all()


def _model(seed=0, dtype=torch.float32):
    torch.manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s).to(dtype).to(DEV)) for s in ((64, 33), (64,), (3, 64), (3,), ())]


def test_optimizer_follows_torch_and_its_state_dicts():
    """Five steps with two groups and a schedule beside torch.optim.AdamW in 64 bits, starting from a state dict
    of torch's own AdamW in fp32.  Each step's parameter error is below 2^-18 of lr plus 2^-22 of |p|."""
    from lpgnn import optim

    ps = _model()
    qs = [torch.nn.Parameter(p.detach().double()) for p in ps]
    gs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    groups = lambda x: [dict(params=x[:2]), dict(params=x[2:], lr=3e-3, weight_decay=0.1)]
    a, b = optim.AdamW(groups(ps), lr=1e-3), torch.optim.AdamW(groups(qs), lr=1e-3)
    c = torch.optim.AdamW(groups(gs), lr=1e-3)
    for x in gs:
        x.grad = torch.randn_like(x)
    c.step()
    sd = c.state_dict()
    for p, q, x in zip(ps, qs, gs):
        p.data.copy_(x.data), q.data.copy_(x.data)
    a.load_state_dict(sd), b.load_state_dict(sd)
    sched = [torch.optim.lr_scheduler.StepLR(o, 2, 0.1) for o in (a, b)]
    for k in range(5):
        for p, q in zip(ps, qs):
            p.grad = torch.randn_like(p) if not (k == 2 and p.dim() == 0) else None  # one skips a step
            q.grad = None if p.grad is None else p.grad.double()
        a.step(), b.step()
        for s in sched:
            s.step()
    for p, q in zip(ps, qs):
        assert ((p.double() - q).abs() <= 5 * (3e-3 * 2.0 ** -18 + 2.0 ** -22 * q.abs())).all()
    assert a.state[ps[4]]["step"] == 5 and a.state[ps[0]]["step"] == 6
    d = torch.optim.AdamW(groups(gs), lr=1e-3)
    d.load_state_dict(a.state_dict())  # and back
    assert torch.equal(d.state[gs[0]]["exp_avg"], a.state[ps[0]]["exp_avg"])


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_resumes_bit_for_bit(bits):
    from lpgnn import optim

    def steps(o, ps, n, at):
        for k in range(n):
            g = torch.Generator(device=DEV).manual_seed(100 + at + k)
            for p in ps:
                p.grad = torch.randn(p.shape, generator=g, device=DEV)
            o.step()

    ps = _model()
    o = optim.AdamW(ps, state_bits=bits, max_grad_norm=1.0, seed=4)
    steps(o, ps, 3, 0)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    o2 = optim.AdamW(qs, state_bits=bits, max_grad_norm=1.0, seed=4)
    o2.load_state_dict(o.state_dict())
    steps(o, ps, 3, 3), steps(o2, qs, 3, 3)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and torch.equal(o.last_norm, o2.last_norm)
    with pytest.raises(RuntimeError, match="bit moments"):
        wrong = optim.AdamW(ps, state_bits=40 - bits)
        wrong.load_state_dict(o.state_dict())
        wrong.step()


def test_optimizer_leaves_gradients_and_clips_as_torch():
    from lpgnn import optim

    ps = _model(1)
    qs = [torch.nn.Parameter(p.detach().double()) for p in ps]
    a, b = optim.AdamW(ps, max_grad_norm=0.5), torch.optim.AdamW(qs)
    for k in range(3):
        for p, q in zip(ps, qs):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.double()
        before = [p.grad.clone() for p in ps]
        a.step()
        norm = torch.nn.utils.clip_grad_norm_(qs, 0.5)
        b.step()
        assert abs(a.last_norm.item() - norm.item()) <= 2 * U * norm.item()
        assert all(torch.equal(p.grad, g) for p, g in zip(ps, before))
    for p, q in zip(ps, qs):
        assert ((p.double() - q).abs() <= 3 * (1e-3 * 2.0 ** -18 + 2.0 ** -22 * q.abs())).all()


def test_8bit_training_tracks_32bit_moments():
    """200 steps of noisy gradients with a fixed mean and spread: the stored moments stay unbiased.  r's random
    walk at b2 = 0.9 over 4096 elements: the mean ratio to the 32-bit r is 1 within 5 standard errors, whose one-step
    rounding spread of at most step / 2 (1/16) grows by at most 1 / sqrt(1 - 0.9^2 / ...) < 3: 0.19 / 64 = 0.003."""
    from lpgnn import optim

    n = 4096
    p8, p32 = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    m8, r8 = (torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ms, rs = (torch.zeros(n // 256, device=DEV) for _ in range(2))
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    kw = dict(H, betas=(0.9, 0.9))
    gen = torch.Generator(device=DEV).manual_seed(0)
    for t in range(1, 201):
        g = 0.5 + 0.1 * torch.randn(n, generator=gen, device=DEV)
        optim.adamw_step_8bit([p8], [g], [m8], [ms], [r8], [rs], step=t, seed=2, **kw)
        optim.adamw_step([p32], [g], [m], [v], step=t, **kw)
    r = r8.float() * rs.repeat_interleave(256)
    mm = m8.float() * ms.repeat_interleave(256)
    assert abs((r / v.sqrt()).mean().item() - 1) < 0.015
    assert abs((mm / m).mean().item() - 1) < 0.015


@pytest.mark.parametrize("bits", [8, 32])
def test_other_stream_and_graph(bits):
    """The functions on a side stream, and captured: replays continue from the state they find."""
    from lpgnn import optim

    def make():
        host = _lists([1000, 5, 300], seed=8)
        p, g = ([x.to(DEV) for x in ts] for ts in host[:2])
        if bits == 32:
            return p, g, [[x.to(DEV) for x in ts] for ts in host[2:]]
        f8 = lambda: [torch.zeros_like(x, dtype=torch.uint8).view(torch.float8_e4m3fn) for x in p]
        sc = lambda: [torch.zeros(-(-x.numel() // 256), device=DEV) for x in p]
        return p, g, [f8(), sc(), f8(), sc()]

    def one(p, g, st):
        norm, s = optim.clip_scale(g, 0.1)
        (optim.adamw_step if bits == 32 else optim.adamw_step_8bit)(p, g, *st, step=3, grad_scale=s, **H)
        return norm

    a, b, c = make(), make(), make()
    for _ in range(4):
        na = one(*a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            one(*b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nc = one(*c)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        torch.ones(10, device=DEV).sum().item()
    flat = lambda s: [x.float() for x in s[0]] + [x.float() for ts in s[2] for x in ts]
    for x, y, z in zip(flat(a), flat(b), flat(c)):
        assert torch.equal(x, y) and torch.equal(x, z)
    assert torch.equal(na, nc)


def test_refusals():
    from lpgnn import optim

    t = lambda n=8, dt=torch.float32: torch.ones(n, device=DEV, dtype=dt)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        optim.adamw_step([t(dt=torch.float16)], [t(dt=torch.float16)], [t()], [t()], step=1)
    with pytest.raises(RuntimeError, match="grads must be"):
        optim.adamw_step([t()], [t(dt=torch.bfloat16)], [t()], [t()], step=1)
    with pytest.raises(RuntimeError, match="exp_avgs must be"):
        optim.adamw_step([t()], [t()], [t(dt=torch.bfloat16)], [t()], step=1)
    with pytest.raises(RuntimeError, match="sizes"):
        optim.adamw_step([t()], [t(7)], [t()], [t()], step=1)
    with pytest.raises(RuntimeError, match="1 params and 2 grads"):
        optim.adamw_step([t()], [t(), t()], [t()], [t()], step=1)
    with pytest.raises(RuntimeError, match="contiguous"):
        optim.adamw_step([t(16)[::2]], [t()], [t()], [t()], step=1)
    with pytest.raises(RuntimeError, match="device"):
        optim.adamw_step([t()], [torch.ones(8)], [t()], [t()], step=1)
    with pytest.raises(RuntimeError, match="twice"):
        x = t()
        optim.adamw_step([x, x], [t(), t()], [t(), t()], [t(), t()], step=1)
    with pytest.raises(RuntimeError, match="from 1"):
        optim.adamw_step([t()], [t()], [t()], [t()], step=0)
    for bad in (torch.ones(1), t(2), t(1, torch.float64)):
        with pytest.raises(RuntimeError, match="grad_scale"):
            optim.adamw_step([t()], [t()], [t()], [t()], step=1, grad_scale=bad)
    with pytest.raises(RuntimeError, match="m_scales do not"):
        q = t().to(torch.float8_e4m3fn)
        optim.adamw_step_8bit([t()], [t()], [q], [t(2)], [q.clone()], [t(1)], step=1)
    with pytest.raises(RuntimeError, match="places"):
        optim.adamw_step_8bit([t()], [t()], [q], [t(1)], [q.clone()], [t(1)], step=1, places=[0, 1])
    p = torch.nn.Parameter(t())
    o = optim.AdamW([p])
    p.grad = t()
    o.step()
    torch.cuda.synchronize()
    p.grad = torch.ones(8, device=DEV).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        o.step()
    p.grad = t()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(g):
            o.step()


def test_overlapping_tensors_are_refused():
    from lpgnn import optim

    f = torch.zeros(64, device=DEV)
    t = lambda: torch.zeros(16, device=DEV)
    ok = dict(params=[f[:16], f[16:32]], grads=[t(), t()], exp_avgs=[t(), t()], exp_avg_sqs=[t(), t()])
    optim.adamw_step(**ok, step=1)  # (beside each other)
    g = t()
    optim.adamw_step(**{**ok, "grads": [g, g]}, step=1)  # (read only)
    for bad in (dict(params=[f[:16], f[15:31]]), dict(exp_avgs=[g, g]), dict(exp_avg_sqs=ok["exp_avgs"]),
                dict(grads=[f[4:20], t()]), dict(exp_avgs=[f[40:56], f[32:48]])):
        with pytest.raises(RuntimeError, match="overlap"):
            optim.adamw_step(**{**ok, **bad}, step=1)
    q = [torch.zeros(16, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(4)]
    s = [torch.zeros(1, device=DEV) for _ in range(4)]
    optim.adamw_step_8bit(ok["params"], ok["grads"], q[:2], s[:2], q[2:], s[2:], step=1)
    for m8, ms, r8, rs in ((q[:2], s[:2], q[1:3], s[2:]), (q[:2], s[:2], q[2:], s[1:3]), ([q[0], q[0]], s[:2], q[2:], s[2:])):
        with pytest.raises(RuntimeError, match="overlap"):
            optim.adamw_step_8bit(ok["params"], ok["grads"], m8, ms, r8, rs, step=1)


@pytest.mark.parametrize("bits", [8, 32])
def test_more_elements_than_32_bits_count(bits):
    """One tensor of more than 2^31 numbers: its last blocks are those of a small call with the same hash inputs
    (32 bits: of any call), and the norm sees them."""
    from lpgnn import optim

    n, k = 2**31 + 256 * 5 + 3, 256 * 5 + 3  # (the last k numbers start on a block)
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    p[-k:].normal_()
    g[-k:].normal_()
    p0, g0 = p[-k:].clone(), g[-k:].clone()
    norm, _ = optim.clip_scale([g], 1.0)
    want = g0.double().norm()
    assert abs(norm.double() - want) <= 2.0**-24 * want + 1e-9 * want
    if bits == 32:
        st = [torch.zeros(n, device=DEV) for _ in range(2)]
        s0 = [torch.zeros(k, device=DEV) for _ in range(2)]
        optim.adamw_step([p], [g], [st[0]], [st[1]], step=1)
        optim.adamw_step([p0], [g0], [s0[0]], [s0[1]], step=1)
        assert all(torch.equal(a[-k:], b) for a, b in zip(st, s0))
    else:
        f8 = lambda m: torch.zeros(m, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        sc = lambda m: torch.zeros(-(-m // 256), device=DEV)
        st, s0 = [f8(n), sc(n), f8(n), sc(n)], [f8(k), sc(k), f8(k), sc(k)]
        optim.adamw_step_8bit([p], [g], *[[t] for t in st], step=1)
        optim.adamw_step_8bit([p0], [g0], *[[t] for t in s0], step=1)
        assert torch.equal(st[1][-6:], s0[1]) and torch.equal(st[3][-6:], s0[3])
        # the codes' random bits differ by the element: within a step of the format of each other
        for a, b in ((st[0], s0[0]), (st[2], s0[2])):
            a, b = a[-k:].float(), b.float()
            assert ((a - b).abs() <= torch.maximum(a.abs(), b.abs()) / 8 + 2.0**-9).all() and a.count_nonzero() > k // 2
    assert torch.equal(p[-k:], p0) and p[:1000].count_nonzero() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_split_over_blocks_does_not_show(dtype):
    """More numbers than the small chunks are for, in one call and in pieces of it: the same bits, and the norm of all
    is the pieces' together."""
    from lpgnn import optim

    n = 2**24 + 4099
    gen = torch.Generator(device=DEV).manual_seed(5)
    r = lambda: torch.randn(n, generator=gen, device=DEV)
    p, g, m, v = r().to(dtype), r().to(dtype), r(), r().square()
    pieces = [0, 5, 2**20 + 3, 2**23, n]
    a = [t.clone() for t in (p, g, m, v)]
    optim.adamw_step(*[[t] for t in a], step=7, **H)
    for lo, hi in zip(pieces, pieces[1:]):
        optim.adamw_step(*[[t[lo:hi]] for t in (p, g, m, v)], step=7, **H)
    assert all(torch.equal(x, y) for x, y in zip(a, (p, g, m, v)))
    whole, scale = optim.clip_scale([g], 0.5)
    cut, scale2 = optim.clip_scale([g[lo:hi] for lo, hi in zip(pieces, pieces[1:])], 0.5)
    want = g.double().square().sum().sqrt()
    for x in (whole, cut):
        assert abs(x.double() - want) <= (2.0**-24 + n * 2.0**-53) * want
    assert abs(scale - scale2) <= 2.0**-22 * scale


def test_goes_on_from_a_bf16_state_of_torch():
    """torch keeps bf16 parameters' moments in bf16; the next step here is the kernel's from those numbers."""
    from lpgnn import optim

    ps = _model(2, torch.bfloat16)
    t = torch.optim.AdamW(ps, **H)
    for p in ps:
        p.grad = torch.randn_like(p)
    t.step()
    a = optim.AdamW(ps, **H)
    a.load_state_dict(t.state_dict())
    host = [(p.detach().cpu(), p.grad.cpu(), t.state[p]["exp_avg"].float().cpu(), t.state[p]["exp_avg_sq"].float().cpu())
            for p in ps]
    a.step()
    for p, x in zip(ps, host):
        want = R.step32(*x, 2, **H)
        for got, w in zip((p.detach(), a.state[p]["exp_avg"], a.state[p]["exp_avg_sq"]), want):
            assert torch.equal(got.cpu(), w.to(got.dtype))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_deep_copy_steps_to_the_same_bits(bits):
    import copy

    from lpgnn import optim

    ps = _model(3)
    o = optim.AdamW(ps, state_bits=bits, max_grad_norm=0.7, seed=11)
    for p in ps:
        p.grad = torch.randn_like(p)
    o.step()
    c = copy.deepcopy(o)
    qs = c.param_groups[0]["params"]
    for p, q in zip(ps, qs):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    o.step(), c.step()
    assert all(torch.equal(p, q) and p.data_ptr() != q.data_ptr() for p, q in zip(ps, qs))
    assert torch.equal(o.last_norm, c.last_norm)


def test_a_scale_inside_a_written_tensor_is_refused():
    """grad_scale is read by every block while others write: it may share memory with a gradient only."""
    from lpgnn import optim

    t = lambda: torch.zeros(300, device=DEV)
    p, g, m, v = t(), t(), t(), t()
    for s in (p[:1], p[299:], m[5], v[7:8]):
        with pytest.raises(RuntimeError, match="overlap"):
            optim.adamw_step([p], [g], [m], [v], step=1, grad_scale=s)
    optim.adamw_step([p], [g], [m], [v], step=1, grad_scale=g[3])
    q = [torch.zeros(300, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    s = [torch.zeros(2, device=DEV) for _ in range(2)]
    for scale in (p[1:2], s[0][0], s[1][1]):
        with pytest.raises(RuntimeError, match="overlap"):
            optim.adamw_step_8bit([p], [g], [q[0]], [s[0]], [q[1]], [s[1]], step=1, grad_scale=scale)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_updates_nothing(bits):
    """Two groups, the second with a parameter that its call refuses: the first is as it was, and steps once after."""
    from lpgnn import optim

    a = torch.nn.Parameter(torch.ones(40, device=DEV))
    b = torch.nn.Parameter(torch.ones(8, 6, device=DEV).t())
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    for most in (None, 1.0):
        o = optim.AdamW([dict(params=[a]), dict(params=[b], lr=0.1)], state_bits=bits, max_grad_norm=most)
        with pytest.raises(RuntimeError, match="contiguous"):
            o.step()
        assert torch.equal(a, torch.ones_like(a)) and o.state[a]["step"] == 0 and o.last_norm is None
        assert not any(t.float().any() for t in o.state[a].values() if isinstance(t, torch.Tensor))


def test_8bit_second_moment_at_the_default_beta():
    """b2 = 0.999, where a step changes r by less than half a step of its format and rounding to nearest would keep it
    for good: after 3000 steps of noise v is the 32-bit one's on average.  What random rounding adds: a stored r lies on
    the format's grid, so a step of the grid (at most r / 8) and the distance d to a grid point give it the variance of
    at most d r / 8, d at most r's change plus that of the block's scale, each (1 - b2) / 2 E|g^2 / v - 1| r, the
    expectation 0.97 of a normal g: v gains 0.121 (1 - b2) v a step and forgets 1 - b2 of it, so its mean ratio is
    between 1 and 1.121.  An element's ratio spreads by less than 0.5 (v itself by 0.03): 5 standard errors are 0.04."""
    from lpgnn import optim

    n = 4096
    gen = torch.Generator(device=DEV).manual_seed(0)
    spread = 2.0 ** (-4 * torch.rand(n, generator=gen, device=DEV))  # (all of a block within the format's normal range)
    p8, p32, m, v = (torch.zeros(n, device=DEV) for _ in range(4))
    m8, r8 = (torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ms, rs = (torch.zeros(n // 256, device=DEV) for _ in range(2))
    for t in range(1, 3001):
        g = torch.randn(n, generator=gen, device=DEV) * spread
        optim.adamw_step_8bit([p8], [g], [m8], [ms], [r8], [rs], step=t, seed=2, **H)
        optim.adamw_step([p32], [g], [m], [v], step=t, **H)
    ratio = (r8.float() * rs.repeat_interleave(256)).square() / v
    assert 0.96 < ratio.mean().item() < 1.17 and ratio.std().item() < 0.5


def test_the_clip_under_other_splits_is_at_most_a_neighbour():
    """The 64-bit sums of other splits differ by n 2^-53 of themselves at most, far below a step of fp32: the rounded
    norm and factor are equal or neighbours, and the same list gives the same bits."""
    from lpgnn import optim

    g = torch.randn(3 * 2**20 + 77, generator=torch.Generator(device=DEV).manual_seed(9), device=DEV)
    near = lambda a, b: abs(a.view(torch.int32).item() - b.view(torch.int32).item()) <= 1
    whole = optim.clip_scale([g], 0.37)
    assert all(torch.equal(a, b) for a, b in zip(whole, optim.clip_scale([g], 0.37)))
    for k in (1, 5, 4096, 100003, 2**20):
        for pieces in ([g[:k], g[k:]], list(g.split(max(k, 50021)))):
            assert all(near(a, b) for a, b in zip(whole, optim.clip_scale(pieces, 0.37)))
