"""lpgnn.linear_i8 and quantize_i8 on the GPU: the codes and the sums are exact and the epilogue is a fixed
chain of fp32 roundings, so results have to be the restatement's bits (tests/i8_ref.py); and within the
derived bound of the 64-bit formula."""
import pytest
import torch

import i8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _case(M, N, K1, K2, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 101 + M * 7 + N * 3 + K1)
    n = lambda *s: torch.randn(*s, generator=g)
    x = (n(M, K1) * torch.exp(n(M, 1))).to(dtype)
    x2 = n(M, K2).to(dtype) if K2 else None
    W, bias = n(N, K1 + K2) * 0.1, n(N)
    return x, x2, W, bias


def _dev(t):
    return None if t is None else t.to(DEV)


def _check(x, x2, W, bias, relu, w=None):
    from lpgnn import linear_i8, quantize_i8

    wq, ws = quantize_i8(_dev(W)) if w is None else w
    y = linear_i8(_dev(x), wq, ws, _dev(bias), x2=_dev(x2), relu=relu)
    xx = x if x2 is None else torch.cat((x, x2), 1)
    q, s, top = R.quantize(xx)
    a, sw = wq.cpu(), ws.cpu()
    assert y.dtype == x.dtype and y.shape == (x.shape[0], a.shape[0])
    assert torch.equal(y.cpu(), R.linear(q, s, a, sw, bias, relu, x.dtype))
    y64 = R.linear64(q, top, a, sw, bias, relu)
    assert ((y.cpu().double() - y64).abs() <= R.bound(q, top, a, sw, bias, y64, x.dtype)).all()
    return y


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("K1,K2", [(1, 0), (3, 4), (8, 8), (15, 1), (16, 0), (100, 27), (128, 0), (64, 64), (129, 0),
                                   (200, 200), (1000, 25), (1024, 1024), (5000, 0)])
def test_codes(K1, K2, dtype):
    from lpgnn import quantize_i8

    for M in (1, 5, 130):
        x, x2, _, _ = _case(M, 1, K1, K2, T[dtype])
        x[0, 0] = x.abs().max() * 2  # 63.5 of 127: an exact border, decided to the even code
        if K1 > 1:
            x[0, 1], x[0, K1 - 1] = x[0, 0] / 2, -x[0, 0] / 2
        q, s = quantize_i8(_dev(x), _dev(x2))
        want, sw, _ = R.quantize(x if x2 is None else torch.cat((x, x2), 1))
        assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), sw)
        assert q.stride(0) % 128 == 0 and not q.as_strided((M, q.stride(0)), (q.stride(0), 1))[:, K1 + K2:].any()


def test_codes_next_to_borders():
    """fp32 numbers on both sides of every border between two codes, one unit in the last place apart: an fp32
    quotient would put some on the wrong side."""
    from lpgnn import quantize_i8

    for top in (1.0, 1.7, 3.1415927, 0.1, 127.0, 253.99998):
        top = torch.tensor(top)
        b = ((torch.arange(127).double() + 0.5) / 127 * top.double()).float()
        lo, hi = torch.nextafter(b, torch.tensor(0.0)), torch.nextafter(b, torch.tensor(1e9))
        row = torch.cat((top[None], lo, b, hi, -lo, -b, -hi))
        x = row.repeat(70, 1)
        x[1:] *= (1 + torch.rand(69, 1, generator=torch.Generator().manual_seed(1)))
        q, s = quantize_i8(_dev(x))
        want, sw, _ = R.quantize(x)
        assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), sw)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 63, 64, 65, 130, 300])
def test_linear(M, dtype):
    for k, (N, K1, K2) in enumerate(((1, 40, 0), (17, 16, 16), (64, 128, 0), (65, 100, 29), (128, 127, 130), (333, 200, 200),
                                     (200, 1024, 1024), (20, 4500, 100))):
        _check(*_case(M, N, K1, K2, T[dtype]), relu=k % 2 == 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(128 * 63 + 1, 384, 300), (128 * 64, 383, 128), (256 * 95 + 3, 512, 260),
                                   (256 * 96, 511, 385), (256 * 96, 264, 512)])
def test_linear_large_tiles(M, N, K, dtype):
    """Shapes of the 128 and 256 tiles, with rows, columns and k that end inside one."""
    _check(*_case(M, N, K, 0, T[dtype]), relu=False)


def test_longest_sum_and_largest_codes():
    """K at its limit with every product 127 * 127: 2114060288, below 2^31."""
    K = 131072
    from lpgnn import linear_i8

    wq = torch.full((16, K), 127, dtype=torch.int8, device=DEV)
    wq[1] = -127
    for M in (1, 9):
        y = linear_i8(torch.ones(M, K, device=DEV), wq, torch.ones(16, device=DEV))
        want = torch.full((M, 16), float(K * 127 * 127)) * (torch.ones(1) / torch.full((1,), 127.0))
        want[:, 1] *= -1
        assert torch.equal(y.cpu(), want)
    with pytest.raises(RuntimeError, match="131072"):
        linear_i8(torch.ones(9, K + 16, device=DEV), torch.zeros(16, K + 16, dtype=torch.int8, device=DEV),
                  torch.ones(16, device=DEV))


@pytest.mark.parametrize("M", [3, 40])
def test_bad_and_empty_rows(M):
    from lpgnn import linear_i8, quantize_i8

    x, x2, W, bias = _case(M, 50, 70, 30, torch.float32)
    wq, ws = quantize_i8(_dev(W))
    clean = linear_i8(_dev(x), wq, ws, _dev(bias), x2=_dev(x2), relu=True)
    x[0], x2[0] = 0.0, 0.0
    x[1, 5] = float("nan")
    x2[2, 29] = float("-inf")
    y = linear_i8(_dev(x), wq, ws, _dev(bias), x2=_dev(x2), relu=True)
    assert torch.equal(y[0].cpu(), bias.clamp(min=0)) and y[1].isnan().all() and y[2].isnan().all()
    assert torch.equal(y[3:], clean[3:])
    x[0] = 2.0 ** -101  # below what the format of the scale holds: zeros
    assert torch.equal(linear_i8(_dev(x), wq, ws, _dev(bias), x2=_dev(x2))[0].cpu(), bias)
    x[0] = 2.0 ** -99
    _check(x[:1], x2[:1], W, None, False)
    assert linear_i8(_dev(x)[:0], wq, ws, x2=_dev(x2)[:0]).shape == (0, 50)


@pytest.mark.parametrize("M", [2, 50])
def test_strides_and_layouts(M):
    """Rows inside wider buffers at odd offsets, transposed inputs, weights off 16-byte borders, weights at the
    very end of their storage, more dimensions."""
    from lpgnn import linear_i8, quantize_i8

    x, x2, W, bias = _case(M, 37, 75, 33, torch.bfloat16)
    wq, ws = quantize_i8(_dev(W))
    want = linear_i8(_dev(x), wq, ws, _dev(bias), x2=_dev(x2))
    wide = torch.full((M, 200), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, 3:78], wide[:, 101:134] = _dev(x), _dev(x2)
    assert torch.equal(linear_i8(wide[:, 3:78], wq, ws, _dev(bias), x2=wide[:, 101:134]), want)
    assert torch.equal(linear_i8(_dev(x).t().contiguous().t(), wq, ws, _dev(bias), x2=_dev(x2)), want)
    tight = torch.empty(37 * 108 + 1, dtype=torch.int8, device=DEV)
    odd = tight[1:].view(37, 108)
    odd.copy_(wq)
    end = torch.zeros(36 * 112 + 108, dtype=torch.int8, device=DEV).as_strided((37, 108), (112, 1))
    end.copy_(wq)
    for w in (wq.contiguous(), odd, wq.t().contiguous().t(), end):
        assert torch.equal(linear_i8(_dev(x), w, ws, _dev(bias), x2=_dev(x2)), want)
    a, b = _dev(x).view(M // 2, 2, 75), _dev(x2).view(M // 2, 2, 33)
    assert torch.equal(linear_i8(a, wq, ws, _dev(bias), x2=b).view(M, 37), want)
    one = _dev(x[:1]).t().contiguous().t()  # a single row whose stride is 1
    assert torch.equal(linear_i8(one, wq, ws, _dev(bias), x2=_dev(x2[:1])), want[:1])


def test_other_stream_and_graph():
    from lpgnn import linear_i8, quantize_i8

    for M in (4, 100):
        x, x2, W, bias = (_dev(t) for t in _case(M, 64, 80, 40, torch.float16))
        wq, ws = quantize_i8(W)
        want = linear_i8(x, wq, ws, bias, x2=x2)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = linear_i8(x, wq, ws, bias, x2=x2)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = linear_i8(x, wq, ws, bias, x2=x2)
        for k in range(3):
            x.mul_(-0.5)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, linear_i8(x, wq, ws, bias, x2=x2))


def test_refusals():
    from lpgnn import linear_i8, quantize_i8

    x = torch.randn(4, 32, device=DEV)
    wq, ws = quantize_i8(torch.randn(8, 32, device=DEV))
    for args, kw, msg in (((x.double(), wq, ws), {}, "float32, bfloat16 or float16"),
                          ((x, wq[:, :31], ws), {}, "wq must be"),
                          ((x, wq.short(), ws), {}, "wq must be"),
                          ((x, wq.cpu(), ws), {}, "wq must be"),
                          ((x, wq, ws[:7]), {}, "ws must be"),
                          ((x, wq, ws, torch.ones(8, device=DEV).half()), {}, "bias must be"),
                          ((x, wq, ws), dict(x2=x), "wq must be"),
                          ((x[:, :16], wq, ws), dict(x2=x[:3, :16]), "x2 must have"),
                          ((x[:, :16], wq, ws), dict(x2=x[:, :16].half()), "x2 must have"),
                          ((x.clone().requires_grad_(True), wq, ws), {}, "no gradient")):
        with pytest.raises(RuntimeError, match=msg):
            linear_i8(*args, **kw)
    with torch.no_grad():
        linear_i8(x.clone().requires_grad_(True), wq, ws)


@pytest.mark.parametrize("K1,K2", [(96, 32), (131, 0)])
def test_more_rows_than_a_chunk(K1, K2):
    """Rows taken through in several chunks, the last one short: the same bits as chunk by chunk."""
    from lpgnn import _lib, linear_i8, quantize_i8

    N = 8
    rows = _lib.lib().lpg_i8_chunk_rows(1 << 40, N, K1 + K2)
    M = 2 * rows + 777
    g = torch.Generator(device=DEV).manual_seed(0)
    wide = torch.randn(M, K1 + K2 + 3, generator=g, device=DEV).half()
    x, x2 = wide[:, :K1], wide[:, K1 + 1:K1 + 1 + K2] if K2 else None
    wq, ws = quantize_i8(torch.randn(N, K1 + K2, generator=g, device=DEV))
    y = linear_i8(x, wq, ws, x2=x2)
    for a, b in ((0, 100), (rows - 50, rows + 50), (2 * rows - 3, 2 * rows + 60), (M - 30, M)):
        part = linear_i8(x[a:b], wq, ws, x2=None if x2 is None else x2[a:b])
        assert torch.equal(y[a:b], part)


def test_more_elements_than_32_bits_count():
    """Offsets past 2^31 elements in x and in y, and a weight whose rows are far apart (copied): the bits of small
    calls."""
    from lpgnn import linear_i8, quantize_i8

    K = N = 512
    M = 2**31 // K + 501
    x = torch.zeros(M, K, dtype=torch.float16, device=DEV)
    x[-300:].normal_()
    wq, ws = quantize_i8(torch.randn(N, K, device=DEV))
    y = linear_i8(x, wq, ws)
    assert torch.equal(y[-300:], linear_i8(x[-300:].contiguous(), wq, ws)) and y[:1000].count_nonzero() == 0
    q, s = quantize_i8(x)
    q0, s0 = quantize_i8(x[-300:].contiguous())
    assert torch.equal(q[-300:], q0) and torch.equal(s[-300:], s0)
    far = torch.zeros(3, (1 << 22) + 16, dtype=torch.int8, device=DEV)[:, :K]
    far.copy_(wq[:3])
    assert torch.equal(linear_i8(x[-300:], far, ws[:3]), y[-300:, :3])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,N,K", [(256 * 150 + 5, 512, 100), (256 * 150, 512, 129), (256 * 280, 512, 260),
                                   (300 * 128 + 1, 1100, 40), (256 * 131, 1024, 384),
                                   (256 * 132, 1024, 600)])
def test_blocks_that_go_on_to_further_tiles(M, N, K, dtype):
    """More tiles than blocks, of one k tile and of several, whole ones and cut ones, outputs on lines and off: the
    codes' product by the C entry is that of few rows at a time."""
    from lpgnn import _lib, linear_i8, quantize_i8

    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    x = (torch.randn(M, K, generator=g, device=DEV) * torch.rand(M, 1, generator=g, device=DEV)).to(T[dtype])
    wq, ws = quantize_i8(torch.randn(N, K, generator=g, device=DEV))
    bias = torch.randn(N, generator=g, device=DEV)
    q, s = quantize_i8(x)
    L, code = _lib.lib(), {"bf16": 0, "fp16": 1, "fp32": 2}[dtype]
    for pad, b in ((0, bias), (3, None)):
        y = torch.full((M, N + pad), 7.0, dtype=x.dtype, device=DEV)
        for _ in range(2):
            _lib.check(L.lpg_fc_i8(code, M, N, K, q.data_ptr(), q.stride(0), s.data_ptr(), wq.data_ptr(), wq.stride(0),
                                   ws.data_ptr(), None if b is None else b.data_ptr(), 1, y.data_ptr(), N + pad,
                                   torch.cuda.current_stream().cuda_stream), "lpg_fc_i8")
        assert pad == 0 or bool((y[:, N:] == 7.0).all())
        for a in (0, 256 * 64 + 100, M - 512):
            assert torch.equal(y[a:a + 512, :N], linear_i8(x[a:a + 512], wq, ws, b, relu=True))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("K1,K2", [(65, 0), (70, 3), (90, 45), (97, 7), (150, 150), (200, 8), (300, 0), (301, 299),
                                   (5, 700), (760, 2), (1030, 0), (777, 778), (1537, 0), (2500, 33), (3, 2050),
                                   (4097, 0), (8000, 193)])
def test_codes_of_every_row_length(K1, K2, dtype):
    """The rows' codes where the last vectors overlap, parts are shorter than a vector and lanes run out; the
    padding is zero, rows beside each other are left alone."""
    from lpgnn import quantize_i8

    M = 67
    x, x2, _, _ = _case(M, 1, K1, K2, T[dtype], seed=3)
    wide = torch.full((M, K1 + 3), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, 1:1 + K1] = x.to(DEV)
    q, s = quantize_i8(wide[:, 1:1 + K1], _dev(x2))
    want, ws, _ = R.quantize(x if x2 is None else torch.cat((x, x2), 1))
    assert torch.equal(q.cpu().to(want.dtype), want) and torch.equal(s.cpu(), ws.view(-1).to(s.dtype))
    pitch = q.stride(0)
    assert not q.as_strided((M, pitch), (pitch, 1))[:, K1 + K2:].any()


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 3, 5000), (3, 1, 40), (700, 1, 1281), (9000, 1, 33), (9000, 2, 200),
                                   (33000, 17, 64), (50, 129, 1280), (50, 129, 1281), (20000, 255, 129)])
def test_smallest_sides(M, N, K):
    """One column, one row, one number; both sides of the longest row that few rows take in one launch."""
    for dtype in (torch.float16, torch.float32):
        x, _, W, bias = _case(M, N, K, 0, dtype, seed=5)
        _check(x, None, W, bias, True)


def test_one_tensor_as_both_parts():
    from lpgnn import linear_i8, quantize_i8

    x, _, W, bias = _case(70, 40, 24, 0, torch.bfloat16)
    xd, wq, ws = _dev(x), *quantize_i8(_dev(torch.cat((W, W), 1)))
    assert torch.equal(linear_i8(xd, wq, ws, _dev(bias), x2=xd), linear_i8(xd.repeat(1, 2), wq, ws, _dev(bias)))
    rows = xd[:1].expand(70, 24)  # a broadcast input
    assert torch.equal(linear_i8(rows, wq, ws, x2=rows), linear_i8(rows.contiguous(), wq, ws, x2=rows.contiguous()))


def test_more_rows_than_a_launch_holds():
    """Four rows a block of 256 threads, fewer than 2^32 threads a launch: rows past 2^26 have their codes too."""
    from lpgnn import quantize_i8

    M, K = 2**26 + 77, 72
    x = torch.zeros(M, 1, dtype=torch.float16, device=DEV)
    x2 = torch.zeros(M, K, dtype=torch.float16, device=DEV)
    for t in (x, x2):
        t[:100].normal_()
        t[-200:].normal_()
    q, s = quantize_i8(x, x2)
    for a, b in ((0, 300), (M - 300, M)):
        q0, s0 = quantize_i8(x[a:b].clone(), x2[a:b].clone())
        assert torch.equal(q[a:b], q0) and torch.equal(s[a:b], s0)
    assert s.count_nonzero() == 300


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("K1,K2", [(1024, 0), (1025, 0), (512, 512), (1000, 24), (1000, 25), (3, 1021), (769, 0), (768, 0), (257, 0),
                                   (500, 13)])
def test_few_rows_of_every_vector_count(K1, K2, dtype):
    """Both sides of the longest row that few rows take in one launch, and of the rows that a lane's vectors reach."""
    for M in (2, 17):
        _check(*_case(M, 130, K1, K2, T[dtype], seed=6), relu=False)
