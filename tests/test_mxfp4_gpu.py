"""The MXFP4 kernels against float64 at the edges of their tiles: every pattern of the 16-bit types, rows and columns that end
inside a tile, k that ends inside a stage, strided rows, non-finite rows, graphs and streams."""
import math

import pytest
import torch

import _ref_mxfp4 as ref
import lumen.ops.mxfp4 as mx
from lumen.ops.mxfp4 import MXFP4, mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(seed, *shape):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def weight(seed, N, K, spread=1.0):
    """A weight [N, K] whose blocks differ in size, in MXFP4, and its values in float64."""
    w = randn(seed, N, K) * 0.05 * torch.exp(spread * randn(seed + 1, N, K // 8)).repeat_interleave(8, 1)
    q = mxfp4_quantize(w.bfloat16())
    return q, ref.values(q)


# ---- the format -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", HALF)
def test_every_pattern(dtype):
    """Each of the 65536 values in a block whose largest is 2^0 ... 2^3 times as large: all codes, ties and denormals."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    v = bits.view(dtype)
    v = v[torch.isfinite(v.float())]
    v = v[:len(v) // 16 * 16].view(-1, 16)
    v = v[torch.randperm(len(v), generator=torch.Generator().manual_seed(0))]
    block = torch.cat((v, v.flip(0)), 1)                  # two runs of neighbouring values of different size
    same = torch.cat((v, v), 1)
    x = torch.cat((block, same)).contiguous()
    q = mxfp4_quantize(x.cuda())
    code, byte = ref.encode(x)
    got = ref.unpack(q)
    assert torch.equal(got[1], byte) and torch.equal(got[0], code)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("R,K", [(1, 8), (1, 32), (1, 4096), (3, 96), (5, 416), (9, 424), (70, 2048), (257, 160), (4, 11008)])
def test_quantize(R, K, dtype):
    x = (randn(R + K, R, K + 24) * torch.exp(3 * randn(K, R, 1))).clamp(-6e4, 6e4).to(dtype)[:, 8:8 + K]
    code, byte = ref.encode(x)
    for rows in (x, x.contiguous(), x.t().contiguous().t()):
        q = mxfp4_quantize(rows)
        got = ref.unpack(q)
        assert torch.equal(got[1], byte) and torch.equal(got[0], code)
        assert q._codes.shape[0] == q._scales.shape[0] == -(-K // 128)    # (padded with zeros)
        assert int(q._codes.long().sum()) == int(q.codes.long().sum()) and int(q._scales.long().sum()) == int(q.scales.long().sum())
    want = ref.decode(code, byte)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(mxfp4_dequantize(q, dt).cpu(), want.to(dt))


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
def test_non_finite_blocks(dtype):
    x = randn(1, 4, 128).to(dtype)
    x[0, 33], x[1, 0], x[2, 127] = float("inf"), float("nan"), -float("inf")
    x[3, :32] = 0
    q = mxfp4_quantize(x)
    code, byte = ref.encode(x)
    assert torch.equal(ref.unpack(q)[0], code) and torch.equal(ref.unpack(q)[1], byte)
    y = mxfp4_dequantize(q, dtype)
    assert torch.isnan(y[0, 32:64]).all() and torch.isnan(y).sum() == 96
    y = mxfp4_matmul(q, mxfp4_quantize(randn(2, 20, 128)), out_dtype=torch.float32)
    assert torch.isnan(y[:3]).all() and torch.isfinite(y[3]).all()


def test_all_codes_and_scales_dequantize():
    code = torch.arange(256, dtype=torch.uint8).view(16, 16).repeat(256, 1)           # 32 codes a row
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat_interleave(16, 0)
    q = MXFP4(code.cuda(), scale.cuda())
    want = ref.values(q)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        got = mxfp4_dequantize(q, dt).cpu()
        assert torch.equal(torch.nan_to_num(got, nan=1234.0), torch.nan_to_num(want.to(dt), nan=1234.0))


# ---- products -------------------------------------------------------------------------------------
ROWS = [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 300, 513]
SIZES = [(1, 32), (3, 8), (40, 184), (4, 64), (15, 96), (16, 128), (20, 160), (33, 224), (66, 416), (130, 512), (257, 704), (520, 1056)]


def check_linear(M, N, K, dtype, bias, seed=0, wide=True):
    x = randn(M * 7 + N + K + seed, M, K + (16 if wide else 0)).to(dtype)[:, (8 if wide else 0):][:, :K]
    q, _ = weight(N + K, N, K)
    W = mxfp4_dequantize(q, dtype).double().cpu()
    b = randn(N, N).to(dtype) if bias else None
    xd = x.double().cpu()
    want, mag = xd @ W.t(), xd.abs() @ W.abs().t()
    if bias:
        want, mag = want + b.double().cpu(), mag + b.double().cpu().abs()
    y = mxfp4_linear(x, q, b)
    assert y.dtype == dtype and y.shape == (M, N) and y.is_contiguous()
    ref.close(y, want, mag, K + 1, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M", ROWS)
def test_linear_rows(M, dtype):
    for i, (N, K) in enumerate(SIZES):
        check_linear(M, N, K, dtype, bias=i % 2 == 0, wide=i % 3 == 0)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (5, 1000, 5632), (17, 2048, 2048), (64, 4100, 1024), (96, 1028, 4128), (509, 1000, 2080),
                                   (1021, 2048, 544), (2050, 516, 1024), (1030, 4097, 288)])
def test_linear_sizes(M, N, K, dtype):
    check_linear(M, N, K, dtype, bias=True)


def check_grad(M, N, K, dtype, wide=False):
    dy = randn(M * 3 + N + K, M, N + (16 if wide else 0)).to(dtype)[:, (8 if wide else 0):][:, :N]
    q, _ = weight(N + K, N, K)
    W = mxfp4_dequantize(q, dtype).double().cpu()
    x = randn(1, M, K).to(dtype).requires_grad_()
    y = mxfp4_linear(x, q)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx.dtype == dtype and dx.shape == (M, K)
    d = dy.double().cpu()
    ref.close(dx, d @ W, d.abs() @ W.abs(), N, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M", ROWS)
def test_grad_rows(M, dtype):
    for i, (N, K) in enumerate(SIZES):
        check_grad(M, N, K, dtype, wide=i % 3 == 0)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [(1, 2048, 4096), (509, 1000, 2080), (300, 1001, 1024), (1021, 544, 2048), (2050, 1030, 544), (64, 4096, 1024)])
def test_grad_sizes(M, N, K, dtype):
    check_grad(M, N, K, dtype)


def check_matmul(M, N, K, dtype, bias):
    a = mxfp4_quantize((randn(M + K, M, K) * torch.exp(randn(K, M, 1))).bfloat16())
    b, B = weight(N + K, N, K)
    A = ref.values(a)
    c = randn(N, N).to(dtype) if bias else None
    want, mag = A @ B.t(), A.abs() @ B.abs().t()
    if bias:
        want, mag = want + c.double().cpu(), mag + c.double().cpu().abs()
    y = mxfp4_matmul(a, b, bias=c, out_dtype=dtype)
    assert y.dtype == dtype and y.shape == (M, N)
    ref.close(y, want, mag, K + 1, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("M", ROWS)
def test_matmul_rows(M, dtype):
    for i, (N, K) in enumerate(SIZES):
        check_matmul(M, N, K, dtype, bias=i % 2 == 0)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M,N,K", [(1, 2048, 4096), (48, 4100, 5632), (509, 1000, 2080), (1021, 2048, 544), (2050, 516, 1024), (1030, 4097, 288)])
def test_matmul_sizes(M, N, K, dtype):
    check_matmul(M, N, K, dtype, bias=True)


# every form of the kernels, at sizes that end inside its tiles and with fewer stages than its rings hold
EDGES = [(1, 1, 32), (33, 100, 96), (40, 24, 264), (70, 257, 192), (300, 515, 416), (129, 384, 2080)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("form", sorted({f[2] for f in mx._ROWS + mx._TILES}))
def test_linear_forms(form, dtype, monkeypatch):
    monkeypatch.setattr(mx, "_linear_form", lambda M, N, K: form)
    for M, N, K in EDGES:
        check_linear(M, N, K, dtype, bias=True)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("form", sorted({f[2] for f in mx._GRAD}))
def test_grad_forms(form, dtype, monkeypatch):
    monkeypatch.setattr(mx, "_grad_form", lambda M, N, K: form)
    for M, K, N in EDGES:
        check_grad(M, N, -(-K // 8) * 8, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
@pytest.mark.parametrize("form", sorted({f[2] for f in mx._MATMUL}))
def test_matmul_forms(form, dtype, monkeypatch):
    monkeypatch.setattr(mx, "_matmul_form", lambda M, N, K: form)
    for M, N, K in EDGES:
        check_matmul(M, N, K, dtype, bias=True)


@pytest.mark.parametrize("M", [3, 64, 300])
def test_scales_from_the_smallest_to_the_largest(M):
    """Products whose scales cancel: rows of 2^100 against weights of 2^-100, blocks far below their neighbours."""
    x = randn(1, M, 256).bfloat16()
    big = (x.float() * 2.0 ** 100).bfloat16()
    w = randn(2, 80, 256)
    q = mxfp4_quantize((w * 2.0 ** -100).bfloat16())
    W = ref.values(q)
    ref.close(mxfp4_linear(big, q), big.double().cpu() @ W.t(), big.double().cpu().abs() @ W.abs().t(), 256, torch.bfloat16)
    a = mxfp4_quantize(big)
    A = ref.values(a)
    ref.close(mxfp4_matmul(a, q, out_dtype=torch.float32), A @ W.t(), A.abs() @ W.abs().t(), 256, torch.float32)


@pytest.mark.parametrize("M", [2, 33, 140, 300])
@pytest.mark.parametrize("K", [128, 160, 200])
def test_non_finite_rows_stay_theirs(M, K):
    """An infinite or missing value of a row reaches that row alone; an infinite one keeps its sign where no other meets it."""
    x = randn(3, M, K).bfloat16()
    q, _ = weight(5, 70, K)
    clean = mxfp4_linear(x, q)
    x[0, K - 1], x[1, 3] = float("inf"), float("nan")
    y = mxfp4_linear(x, q)
    assert torch.equal(y[2:], clean[2:])
    W = mxfp4_dequantize(q, torch.float32)
    want = x.float() @ W.t()
    assert torch.equal(torch.isnan(y[:2]), torch.isnan(want[:2]))
    inf = torch.isinf(want[0])
    assert torch.equal(y[0][inf].float(), want[0][inf])


@pytest.mark.parametrize("M", [5, 300])
def test_memory_around_the_rows_is_left_alone(M):
    """Rows in a buffer of NaN: nothing beside them is read into a result."""
    for K in (160, 128, 72):
        buf = torch.full((M + 2, K + 64), float("nan"), device="cuda", dtype=torch.bfloat16)
        x = buf[1:M + 1, 32:32 + K]
        x.copy_(randn(1, M, K))
        q, _ = weight(7, 50, K)
        assert torch.equal(mxfp4_linear(x, q), mxfp4_linear(x.contiguous(), q))
        assert torch.isfinite(mxfp4_dequantize(mxfp4_quantize(x))).all()


def test_leading_dimensions_and_odd_strides():
    q, _ = weight(3, 40, 96)
    x = randn(1, 2, 5, 96).bfloat16()
    y = mxfp4_linear(x, q)
    assert y.shape == (2, 5, 40)
    assert torch.equal(y.view(10, 40), mxfp4_linear(x.view(10, 96), q))
    odd = torch.zeros(10, 97, device="cuda", dtype=torch.bfloat16)[:, 1:]
    odd.copy_(x.view(10, 96))
    assert torch.equal(mxfp4_linear(odd, q), y.view(10, 40))
    t = x.view(10, 96).t().contiguous().t()
    assert torch.equal(mxfp4_linear(t, q), y.view(10, 40))
    one = x.view(10, 96)[:1].expand(10, 96)               # a row read ten times
    assert torch.equal(mxfp4_linear(one, q), y.view(10, 40)[:1].expand(10, 40))


def test_a_run_as_a_layer_makes_it():
    """Quantised base, rows through it, the gradient back, against the same in float64; then with 4-bit rows."""
    w = randn(1, 300, 256) * 0.05
    x = randn(2, 70, 256).bfloat16()
    q = mxfp4_quantize(w.bfloat16())
    leaf = x.clone().requires_grad_()
    y = mxfp4_linear(leaf, q)
    (y.float() ** 2).sum().backward()
    W = ref.values(q)
    dy = 2 * y.detach().double().cpu()
    rounded = dy.to(torch.bfloat16).double()
    ref.close(leaf.grad, rounded @ W, rounded.abs() @ W.abs(), 300, torch.bfloat16)
    a = mxfp4_quantize(x)
    z = mxfp4_matmul(a, q)
    ref.close(z, ref.values(a) @ W.t(), ref.values(a).abs() @ W.abs().t(), 256, torch.bfloat16)


@pytest.mark.parametrize("M", [1, 40, 400])
def test_captured_calls_replay_on_new_rows(M):
    q, _ = weight(1, 500, 288)
    x = randn(1, M, 288).bfloat16()
    dy = randn(2, M, 500).bfloat16()
    from lumen.ops.mxfp4 import input_grad

    def step():
        return mxfp4_linear(x, q), mxfp4_matmul(mxfp4_quantize(x), q), input_grad(dy, q)

    step()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    with torch.cuda.graph(other):
        z = step()
    for i in range(4):
        x.copy_(randn(10 + i, M, 288))
        dy.copy_(randn(20 + i, M, 500))
        want = step()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(want, y, z):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_another_stream():
    q, _ = weight(1, 260, 512)
    x = randn(1, 90, 512).bfloat16()
    want = mxfp4_linear(x, q), mxfp4_matmul(mxfp4_quantize(x), q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = mxfp4_linear(x, q), mxfp4_matmul(mxfp4_quantize(x), q)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_the_same_call_gives_the_same_bits():
    q, _ = weight(1, 1000, 2048)
    for M in (1, 30, 300):
        x = randn(M, M, 2048).bfloat16()
        assert torch.equal(mxfp4_linear(x, q), mxfp4_linear(x, q))


def test_refused_on_the_gpu():
    q, _ = weight(1, 16, 64)
    x = randn(1, 3, 64)
    for f in (lambda: mxfp4_linear(x, q), lambda: mxfp4_linear(x.cpu().bfloat16(), q), lambda: mxfp4_linear(x.bfloat16(), q, torch.zeros(16).bfloat16()),
              lambda: mxfp4_matmul(mxfp4_quantize(x.cpu()), q)):
        with pytest.raises(ValueError):
            f()


def test_empty_on_the_gpu():
    q, _ = weight(1, 16, 64)
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = mxfp4_linear(x, q)
    assert y.shape == (0, 16)
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert dx.shape == (0, 64)
    e = mxfp4_quantize(x)
    assert e.shape == (0, 64) and mxfp4_matmul(e, q).shape == (0, 16) and mxfp4_dequantize(e).shape == (0, 64)
    x = randn(1, 3, 64).bfloat16().requires_grad_()
    (dx,) = torch.autograd.grad(mxfp4_linear(x, e).sum(), x)
    assert mxfp4_matmul(q, e).shape == (16, 0) and int(dx.abs().sum()) == 0


def test_results_past_32_bits():
    """36000 x 65536 values and results: the last rows equal those of a call that has only them."""
    M, N, K = 36000, 65536, 64
    q, _ = weight(3, N, K)
    x = randn(1, M, K).bfloat16()
    W, X = ref.values(q), x[-40:].double().cpu()
    y = mxfp4_linear(x, q)
    ref.close(y[-40:], X @ W.t(), X.abs() @ W.abs().t(), K, torch.bfloat16)
    a = mxfp4_quantize(y)
    assert torch.equal(a.codes[-40:], mxfp4_quantize(y[-40:]).codes) and torch.equal(a.scales[-40:], mxfp4_quantize(y[-40:]).scales)
    back = mxfp4_dequantize(a)
    assert torch.equal(back[-40:], mxfp4_dequantize(mxfp4_quantize(y[-40:])))
    del back
    t, _ = weight(5, K, N)                                # rows of y against 64 rows, and their gradient as large as y
    dx = mx.input_grad(x, t)
    V = ref.values(t)
    ref.close(dx[-40:], X @ V, X.abs() @ V.abs(), K, torch.bfloat16)
    del dx
    z = mxfp4_matmul(mxfp4_quantize(x), q)
    A = ref.values(mxfp4_quantize(x[-40:]))
    ref.close(z[-40:], A @ W.t(), A.abs() @ W.abs().t(), K, torch.bfloat16)


@pytest.mark.parametrize("M", [1, 20, 70])
def test_the_longest_rows(M):
    """2^22 values a row, 65 of them not zero."""
    K = mx.MAX_LD
    at = torch.cat((torch.randint(0, K, (64,), generator=torch.Generator().manual_seed(M)), torch.tensor([K - 1]))).unique().cuda()
    x = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16)
    x[:, at] = randn(M, M, len(at)).bfloat16()
    w = torch.zeros(24, K, device="cuda", dtype=torch.bfloat16)
    w[:, at] = randn(7, 24, len(at)).bfloat16()
    q = mxfp4_quantize(w)
    W = mxfp4_dequantize(q)[:, at].double().cpu()
    X = x[:, at].double().cpu()
    ref.close(mxfp4_linear(x, q), X @ W.t(), X.abs() @ W.abs().t(), 65, torch.bfloat16)
    a = mxfp4_quantize(x)
    A = mxfp4_dequantize(a)[:, at].double().cpu()
    ref.close(mxfp4_matmul(a, q), A @ W.t(), A.abs() @ W.abs().t(), 65, torch.bfloat16)
    g = mx.input_grad(randn(3, M, 24).bfloat16(), q)
    G = randn(3, M, 24).bfloat16().double().cpu()
    ref.close(g[:, at], G @ W, G.abs() @ W.abs(), 24, torch.bfloat16)


def test_the_gradient_can_be_differentiated_on_the_gpu():
    q, W = weight(1, 52, 96)
    x = randn(1, 20, 96).bfloat16().requires_grad_()
    dy = randn(2, 20, 52).bfloat16().requires_grad_()
    (dx,) = torch.autograd.grad(mxfp4_linear(x, q), x, dy, create_graph=True)
    g = randn(3, 20, 96).bfloat16()
    (ddy,) = torch.autograd.grad(dx, dy, g)
    G = g.double().cpu()
    ref.close(ddy, G @ W.t(), G.abs() @ W.abs().t(), 96, torch.bfloat16)


def test_a_bias_between_other_values():
    """A bias that is every second value of a buffer, another that starts at an odd address."""
    q, W = weight(2, 50, 96)
    x = randn(1, 5, 96).bfloat16()
    X = x.double().cpu()
    buf = randn(4, 101).bfloat16()
    for b in (buf[::2][:50], buf[1:51]):
        B = b.double().cpu()
        ref.close(mxfp4_linear(x, q, b), X @ W.t() + B, X.abs() @ W.abs().t() + B.abs(), 97, torch.bfloat16)
        a = mxfp4_quantize(x)
        A = ref.values(a)
        ref.close(mxfp4_matmul(a, q, b), A @ W.t() + B, A.abs() @ W.abs().t() + B.abs(), 97, torch.bfloat16)


def test_the_graph_of_a_call():
    """What autograd promises of any node: a second pass only if kept, saved tensors through hooks and guarded against changes, no
    forward mode."""
    import torch.autograd.forward_ad as fwad

    q, W = weight(1, 60, 96)
    x = randn(1, 7, 96).bfloat16().requires_grad_()
    dy = randn(2, 7, 60).bfloat16()
    D = dy.double().cpu()
    y = mxfp4_linear(x, q)
    (a,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    (b,) = torch.autograd.grad(y, x, dy)
    ref.close(a, D @ W, D.abs() @ W.abs(), 60, torch.bfloat16)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, dy)
    with torch.autograd.graph.save_on_cpu():
        y = mxfp4_linear(x, q)
    (c,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(a, c)
    other = MXFP4(q.codes, q.scales)
    y = mxfp4_linear(x, other)
    other.data.zero_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, dy)
    with fwad.dual_level():
        with pytest.raises(ValueError):
            mxfp4_linear(fwad.make_dual(x.detach(), torch.ones_like(x)), q)
    with torch.no_grad():
        assert mxfp4_linear(x, q).grad_fn is None
    z = mxfp4_linear(x.view(7, 1, 96), q).sum()          # (a gradient whose rows all lie at one address)
    z.backward()
    one = torch.ones(7, 60, dtype=torch.float64)
    ref.close(x.grad, one @ W, one @ W.abs(), 60, torch.bfloat16)


def test_a_captured_forward_and_backward():
    q, _ = weight(1, 500, 288)
    x = randn(1, 70, 288).bfloat16().requires_grad_()
    dy = randn(2, 70, 500).bfloat16()

    def step():
        y = mxfp4_linear(x, q)
        (dx,) = torch.autograd.grad(y, x, dy)
        return y.detach(), dx

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(randn(10 + i, 70, 288))
            dy.copy_(randn(20 + i, 70, 500))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_threads():
    """Calls of two host threads, each on its stream."""
    import threading

    q, _ = weight(1, 1000, 512)
    xs = [randn(i, 40 + 60 * i, 512).bfloat16() for i in range(2)]
    want = [(mxfp4_linear(x, q), mxfp4_matmul(mxfp4_quantize(x), q)) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y, z = mxfp4_linear(xs[i], q), mxfp4_matmul(mxfp4_quantize(xs[i]), q)
            torch.cuda.current_stream().synchronize()
            if not (torch.equal(y, want[i][0]) and torch.equal(z, want[i][1])):
                bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("K", [256, 248])
def test_rows_of_another_width_are_refused(K):
    """Rows whose last panel is the weight's own last one too: their bytes alone fit."""
    q, _ = weight(1, 40, K)
    for other in (K - 8, K + 8, K - 128):
        x = randn(1, 5, other).bfloat16()
        for f in (lambda: mx.linear_rows(x, q), lambda: mxfp4_linear(x, q), lambda: mxfp4_linear(x.requires_grad_(), q)):
            with pytest.raises(ValueError):
                f()
    for n in (32, 39, 41, 48):
        with pytest.raises(ValueError):
            mx.input_grad(randn(1, 5, n).bfloat16(), q)


def test_rows_and_weights_the_extension_refuses():
    """What the calls under autograd functions hand over unchecked: rows of 32 bits, a weight on the host, a bias of other size."""
    q, _ = weight(1, 40, 256)
    x = randn(1, 5, 256).bfloat16()
    for f in (lambda: mx.linear_rows(x.float(), q), lambda: mx.input_grad(randn(1, 5, 40), q), lambda: mx.linear_rows(x, q.to("cpu")),
              lambda: mx.input_grad(randn(1, 5, 40).bfloat16(), q.to("cpu")), lambda: mx.linear_rows(x, q, randn(1, 41).bfloat16()),
              lambda: mx.linear_rows(x, q, randn(1, 40)), lambda: mx.linear_rows(x, q, torch.zeros(40, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            f()


def test_a_negated_bias_of_one_value():
    """A view whose sign torch keeps beside its memory: the imaginary part of a conjugate."""
    q, W = weight(3, 1, 64)
    x = randn(1, 4, 64).bfloat16()
    a = mxfp4_quantize(x)
    A = ref.values(a)
    b = torch.complex(torch.zeros(1), torch.full((1,), 3.0)).cuda().conj().imag
    assert b.is_neg() and float(b) == -3
    ref.close(mxfp4_matmul(a, q, b, out_dtype=torch.float32), A @ W.t() - 3, A.abs() @ W.abs().t() + 3, 65, torch.float32)


def test_two_threads_every_result():
    """As above, each of 50 results compared, and a thread that raises is seen."""
    import threading

    q, _ = weight(1, 1000, 512)
    xs = [randn(i, 40 + 60 * i, 512).bfloat16() for i in range(2)]
    want = [(mxfp4_linear(x, q), mxfp4_matmul(mxfp4_quantize(x), q)) for x in xs]
    torch.cuda.synchronize()
    equal = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [(mxfp4_linear(xs[i], q), mxfp4_matmul(mxfp4_quantize(xs[i]), q)) for _ in range(50)]
            torch.cuda.current_stream().synchronize()
            equal[i] = [torch.equal(a, b) for pair in got for a, b in zip(pair, want[i])]

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(e is not None and len(e) == 100 and all(e) for e in equal)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
def test_blocks_of_the_smallest_numbers(dtype):
    """Blocks whose largest value is denormal or nearly so: codes and scales as for any other."""
    fi = torch.finfo(dtype)
    x = randn(4, 40, 64)
    x = (x / x.abs().amax(1, keepdim=True)).double().cpu()
    top = torch.pow(2.0, torch.linspace(math.log2(fi.smallest_normal) - 12, math.log2(fi.smallest_normal) + 5, 40, dtype=torch.float64))
    x = (x * top.unsqueeze(1)).to(dtype)
    q = mxfp4_quantize(x.cuda())
    code, byte = ref.encode(x)
    assert torch.equal(ref.unpack(q)[1], byte) and torch.equal(ref.unpack(q)[0], code)


@pytest.mark.parametrize("M", [3, 64, 300])
def test_products_with_the_smallest_weights(M):
    """Weights of 2^-128 to 2^-118, below bf16's normal numbers in part, against rows of 2^100; both in 4 bits with the smallest scales on
    one side and the largest on the other."""
    g = torch.Generator().manual_seed(M)
    N, K = 80, 256
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    q = MXFP4(codes.cuda(), torch.randint(0, 8, (N, K // 32), generator=g, dtype=torch.uint8).cuda())
    W = ref.values(q)
    x = (randn(1, M, K) * 2.0 ** 100).bfloat16()
    X = x.double().cpu()
    ref.close(mxfp4_linear(x, q), X @ W.t(), X.abs() @ W.abs().t(), K, torch.bfloat16)
    dy = (randn(2, M, N) * 2.0 ** 100).bfloat16()
    D = dy.double().cpu()
    ref.close(mx.input_grad(dy, q), D @ W, D.abs() @ W.abs(), N, torch.bfloat16)
    a = MXFP4(torch.randint(0, 256, (M, K // 2), generator=g, dtype=torch.uint8).cuda(),
              torch.randint(235, 247, (M, K // 32), generator=g, dtype=torch.uint8).cuda())
    A = ref.values(a)
    ref.close(mxfp4_matmul(a, q, out_dtype=torch.float32), A @ W.t(), A.abs() @ W.abs().t(), K, torch.float32)


@pytest.mark.parametrize("M", [3, 64, 300])
@pytest.mark.parametrize("K", [128, 256])
def test_zeros_under_the_largest_scales(M, K):
    """Codes of zero times any finite scales are zero, also where the two scales' product has no fp32."""
    q, W = weight(1, 300, K)
    q = MXFP4(q.codes, torch.full_like(q.scales, 254))
    a = MXFP4(torch.zeros(M, K // 2, dtype=torch.uint8).cuda(), torch.full((M, K // 32), 254, dtype=torch.uint8).cuda())
    assert int(mxfp4_matmul(a, q, out_dtype=torch.float32).abs().max()) == 0


@pytest.mark.parametrize("shape", [(70, 288), (2, 35, 288)])
def test_a_captured_backward_at_a_leaf_of_a_live_graph(shape):
    """The leaf's accumulation belongs to the eager stream while a graph from before the capture is alive: refused, and possible as
    soon as that graph is gone."""
    q, _ = weight(1, 500, 288)
    x = randn(1, *shape).bfloat16().requires_grad_()
    dy = randn(2, *shape[:-1], 500).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        (want,) = torch.autograd.grad(mxfp4_linear(x, q), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    live = mxfp4_linear(x, q)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="drop that graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(mxfp4_linear(x, q), x, dy)
    (dx,) = torch.autograd.grad(live, x, dy)
    assert torch.equal(dx, want)
    del live
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(mxfp4_linear(x, q), x, dy)
    for _ in range(3):
        got.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
