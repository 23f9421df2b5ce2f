"""MXFP4 on CPU tensors: the format against the oracle, the products' torch path, every refusal."""
import pytest
import torch

import _ref_mxfp4 as ref
from lumen.ops.mxfp4 import MXFP4, mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize


def spread(R, K, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(4 * torch.randn(R, K // 8, generator=g)).repeat_interleave(8, 1)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,K", [(1, 32), (3, 96), (7, 256), (2, 8), (3, 104)])
def test_format(R, K, dtype):
    x = spread(R, K, R + K, dtype).clamp(-60000, 60000)
    x[0, :32] = 0
    x[R - 1, 5] = -0.0
    q = mxfp4_quantize(x)
    code, byte = ref.encode(x)
    assert torch.equal(ref.unpack(q)[0], code) and torch.equal(ref.unpack(q)[1], byte)
    assert torch.equal(mxfp4_dequantize(q, torch.float32).double(), ref.decode(code, byte))


def test_ties_and_every_magnitude():
    x = (torch.arange(-64, 64) / 8.0).view(4, 32).clone()
    x[:, 0] = 6.0                                         # all blocks of unit 1
    q = mxfp4_quantize(x)
    assert (q.scales == 127).all()
    code, _ = ref.encode(x)
    assert torch.equal(ref.unpack(q)[0], code)


def test_extremes():
    x = torch.zeros(6, 32)
    x[0, 3] = 2.0 ** -149
    x[1, 3] = torch.finfo(torch.float32).max
    x[2, 3] = float("inf")
    x[3, 3] = float("nan")
    x[4, 3] = 2.0 ** -126
    x[5, 3] = 7.99
    q = mxfp4_quantize(x)
    assert q.scales.view(-1).tolist() == [0, 252, 255, 255, 0, 127]
    y = mxfp4_dequantize(q, torch.float32)
    assert torch.isnan(y[2:4]).all() and torch.isfinite(y[[0, 1, 4, 5]]).all()
    assert y[1, 3] == 6 * 2.0 ** 125 and y[4, 3] == 2.0 ** -126 and y[5, 3] == 6


@pytest.mark.parametrize("K", [8, 32, 96, 120, 128, 416])
def test_rows_are_padded_and_given_back(K):
    q = mxfp4_quantize(spread(5, K, K))
    assert q.codes.shape == (5, K // 2) and q.scales.shape == (5, -(-K // 32))
    again = MXFP4(q.codes.clone(), q.scales.clone())
    assert again.shape == q.shape
    assert torch.equal(mxfp4_dequantize(again), mxfp4_dequantize(q))
    assert torch.equal(again.to("cpu").codes, q.codes)


def test_products():
    x, w = torch.randn(2, 3, 160), mxfp4_quantize(spread(12, 160, 1).clamp(-9, 9))
    b = torch.randn(12)
    W = ref.values(w)
    y = mxfp4_linear(x, w, b)
    assert y.shape == (2, 3, 12)
    want = x.double() @ W.t() + b.double()
    ref.close(y, want, x.double().abs() @ W.abs().t() + b.abs(), 161, torch.float32)
    a = mxfp4_quantize(x.view(6, 160))
    ref.close(mxfp4_matmul(a, w, out_dtype=torch.float32), ref.values(a) @ W.t(), ref.values(a).abs() @ W.abs().t(), 160, torch.float32)


def test_gradient_of_the_rows():
    w = mxfp4_quantize(torch.randn(9, 64))
    x = torch.randn(4, 64, requires_grad=True)
    dy = torch.randn(4, 9)
    (dx,) = torch.autograd.grad(mxfp4_linear(x, w), x, dy)
    W = ref.values(w)
    ref.close(dx, dy.double() @ W, dy.double().abs() @ W.abs(), 9, torch.float32)
    d = torch.randn(4, 64)                                # linear in x: a difference is exact but for the roundings of its sums
    with torch.no_grad():
        fd = ((mxfp4_linear(x + d, w) - mxfp4_linear(x - d, w)).double() / 2 * dy.double()).sum()
    size = (dy.double().abs() * ((x.detach().abs() + d.abs()).double() @ W.abs().t())).sum()
    assert abs(float(fd - (dx.double() * d.double()).sum())) <= float(size) * (64 + 9) * 2.0 ** -23


def test_the_gradient_can_be_differentiated():
    w = mxfp4_quantize(torch.randn(9, 64))
    W = ref.values(w)
    x = torch.randn(4, 64, requires_grad=True)
    dy = torch.randn(4, 9, requires_grad=True)
    (dx,) = torch.autograd.grad(mxfp4_linear(x, w), x, dy, create_graph=True)
    g = torch.randn(4, 64)
    (ddy,) = torch.autograd.grad(dx, dy, g)
    ref.close(ddy, g.double() @ W.t(), g.double().abs() @ W.abs().t(), 64, torch.float32)


def test_empty():
    w = mxfp4_quantize(torch.randn(4, 64))
    assert mxfp4_linear(torch.randn(0, 64), w).shape == (0, 4)
    none = mxfp4_quantize(torch.randn(0, 64))
    assert mxfp4_dequantize(none).shape == (0, 64)
    assert mxfp4_linear(torch.randn(3, 64), none).shape == (3, 0)
    assert mxfp4_matmul(none, w).shape == (0, 4)
    x = torch.randn(3, 64, requires_grad=True)
    (dx,) = torch.autograd.grad(mxfp4_linear(x, none).sum(), x)
    assert torch.equal(dx, torch.zeros(3, 64))


def refused(f, *a, **k):
    with pytest.raises(ValueError):
        f(*a, **k)


def test_refusals():
    x, w = torch.randn(3, 64), mxfp4_quantize(torch.randn(4, 64))
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)    # noqa: E731
    refused(MXFP4, u8(4, 32).int(), u8(4, 2))
    refused(MXFP4, u8(4, 32), u8(4, 3))
    refused(MXFP4, u8(4, 32), u8(3, 2))
    refused(MXFP4, u8(4, 32).view(-1), u8(4, 2))
    refused(MXFP4, u8(4, 0), u8(4, 0))
    refused(MXFP4, u8(4, 24), u8(4, 3))
    refused(MXFP4, u8(4, 18), u8(4, 2))
    refused(mxfp4_quantize, torch.randn(3, 60))
    refused(mxfp4_quantize, torch.randn(64))
    refused(mxfp4_quantize, torch.randn(3, 0))
    refused(mxfp4_quantize, torch.randn(3, 64).double())
    refused(mxfp4_dequantize, w, torch.float64)
    refused(mxfp4_linear, x.double(), w)
    refused(mxfp4_linear, torch.randn(3, 96), w)
    refused(mxfp4_linear, x, torch.randn(4, 64))
    refused(mxfp4_linear, x, w, torch.randn(5))
    refused(mxfp4_linear, x, w, torch.randn(4).bfloat16())
    refused(mxfp4_linear, x, w, torch.randn(4, requires_grad=True))
    refused(mxfp4_linear, torch.tensor(1.0), w)
    refused(mxfp4_matmul, x, w)
    refused(mxfp4_matmul, w, x)
    refused(mxfp4_matmul, w, w, out_dtype=torch.float64)
    refused(mxfp4_matmul, w, w, bias=torch.zeros(4))      # fp32 bias, bf16 result
    refused(mxfp4_matmul, w, mxfp4_quantize(torch.randn(4, 96)))
    long = MXFP4(u8(1, 1 << 22), u8(1, 1 << 18))          # 2^23 values a row: to quantise and back, not to multiply
    assert long.dequantize().shape == (1, 1 << 23)
    refused(mxfp4_linear, torch.zeros(1, 1 << 23), long)
    refused(mxfp4_matmul, long, long)
    refused(MXFP4, u8(1, (1 << 22) + 4), u8(1, (1 << 18) + 1))
    with pytest.raises(TypeError):
        w.to(torch.float16)                               # (a device: its type is the format)


def test_matrices_pickle_and_copy():
    import copy
    import pickle

    q = mxfp4_quantize(torch.randn(5, 72))
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), q.to("cpu")):
        assert c.shape == q.shape and torch.equal(c.data, q.data)


def test_quantising_leaves_the_graph():
    """Rows that want a gradient quantise as their values do, and what comes of them wants none."""
    x = torch.randn(3, 64, requires_grad=True)
    w = mxfp4_quantize(torch.randn(4, 64))
    q = mxfp4_quantize(x)
    assert torch.equal(q.data, mxfp4_quantize(x.detach()).data)
    assert not q.dequantize(torch.float32).requires_grad and not mxfp4_matmul(q, w).requires_grad
    assert mxfp4_linear(x, w).requires_grad
