"""The operators of 4-bit weights that lumen is timed on: microscaled 4-bit floating point (MXFP4) and its products.

A row is cut into blocks of 32 values.  A block holds one power of two, 2^e with e = floor(log2(largest magnitude)) - 2
(its byte: e + 127), and 32 four-bit numbers: a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, the nearest to value / 2^e (of two
equally near ones the one with an even code; 6 where it passes 6).

A case is a plain dict: ``op``, ``rows`` of activations, ``n`` x ``k`` of the weight (``quantize``: rows x k), ``dtype`` of the
activations, ``bias``, ``wide`` (the rows lie in a wider buffer, as the operand of the folded adapters does).

  quantize  x -> MXFP4 -> the values it stands for, in x's type: what a weight becomes when it is loaded, and what a merge
            or a check of it reads back
  matmul    activations are quantised and multiplied with a quantised weight
  linear    activations stay in 16 bits, the weight is MXFP4 (its values rounded to the activations' type)
  grad      linear and the gradient of its input: a frozen weight under adapters

``prepare`` makes activations, output gradients and the quantised weight from the seed; ``run`` is one call (``grad``: forward and
backward); ``exact`` recomputes it in float64.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 32
F64 = torch.float64


def case(name, op, rows, n, k, dtype="bf16", bias=False, wide=False):
    c = dict(op=op, rows=rows, n=n, k=k, dtype=dtype, bias=bias, wide=wide)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the rows of a few decoded tokens before a product with 4-bit operands: latency alone
        case("quantize_8", "quantize", 8, 0, 4096),
        # a merged gate|up projection is quantised when a model is loaded
        case("quantize_gate_up", "quantize", 22016, 0, 4096),
        # rows of unequal prompts, in the buffer of the folded adapters, half precision
        case("quantize_ragged", "quantize", 509, 0, 5632, "fp16", wide=True),
        # a full decode batch against q|k|v
        case("matmul_48_qkv", "matmul", 48, 12288, 4096),
        # unequal prompts through the down projection of a grouped-query model
        case("matmul_1021_fp16", "matmul", 1021, 2048, 5632, "fp16", wide=True),
        # a scheduler's budget of prompt rows against gate|up: the largest product
        case("matmul_4096_gate_up", "matmul", 4096, 22016, 4096),
        # one chat user: the output projection of one token
        case("linear_1_o", "linear", 1, 4096, 4096),
        # a full server: 64 streams against gate|up
        case("linear_64_gate_up", "linear", 64, 22016, 4096),
        # logits of 17 sampled rows, half precision, a head with a bias
        case("linear_17_head_fp16", "linear", 17, 32000, 2048, "fp16", bias=True),
        # prompt rows against q|k|v
        case("linear_4096_qkv", "linear", 4096, 12288, 4096),
        # one packed micro-batch of unequal sequences through the output projection
        case("grad_509_fp16", "grad", 509, 4096, 4096, "fp16", wide=True),
        # the headline training step's rows (8 x 512) through the down projection
        case("grad_4096_down", "grad", 4096, 4096, 11008),
    ]


LARGEST = 4096 * 22016 * 4096          # multiply-adds of the largest listed product
LARGEST_GRAD = 4096 * 4096 * 11008
LARGEST_QUANTIZE = 22016 * 4096


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "matmul", "linear", "linear", "grad"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    wide = rng.random() < 0.3
    k = BLOCK * _log(rng, 2, 352)                        # 64 ... 11264: every multiple of a block
    if op == "quantize":
        return case(None, op, _log(rng, 1, min(32000, LARGEST_QUANTIZE // k)), 0, k, dtype, wide=wide)
    n = rng.choice((_log(rng, 16, 32000), 16 * _log(rng, 1, 1376), 4096, 11008))
    most = LARGEST_GRAD if op == "grad" else LARGEST
    rows = _log(rng, 1, max(1, min(4096, most // (n * k))))
    return case(None, op, rows, n, k, dtype, rng.random() < 0.3, wide)


# ---- the format in plain torch --------------------------------------------------------------------
def encode(x):
    """Codes [R, K / 2] (two to a byte, the first in its low half) and scales [R, K / 32] of x [R, K]."""
    R, K = x.shape
    b = x.float().view(R, K // BLOCK, BLOCK)
    amax = b.abs().amax(-1)
    e = torch.clamp(torch.frexp(amax)[1] - 3, -127, 127)           # frexp: amax = f 2^p with f in [0.5, 1)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    v = torch.ldexp(b, -e.unsqueeze(-1))
    m = v.abs()
    half = (m < 2).to(torch.float32) * 0.5 + (m >= 2).to(torch.float32) + (m >= 4).to(torch.float32)
    r = torch.clamp(torch.round(m / half) * half, max=6.0)         # the step between neighbours: 0.5, 1, 2
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.view(R, K // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def decode(codes, scales):
    """The values [R, K] in fp32 that codes and scales stand for."""
    R = codes.shape[0]
    lut = torch.tensor(VALUES, dtype=torch.float32, device=codes.device)
    v = torch.stack((lut[(codes & 15).int()], lut[(codes >> 4).int()]), -1).view(R, -1, BLOCK)
    return torch.ldexp(v, scales.int().unsqueeze(-1) - 127).view(R, -1)


# ---- inputs ----------------------------------------------------------------------------------------
def tensors(c, seed):
    """x, dy, bias, codes and scales of the weight (None where the case has none)."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    M, N, K, dt = c["rows"], c["n"], c["k"], DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if c["op"] == "quantize" and M > 4096:               # a weight
        x = normal(M, K).mul_(0.02)
    else:                                                # activations: a few channels stand out
        x = normal(M, K)
        x *= torch.where(torch.rand(K, generator=g, device=dev) < 0.01, 20.0, 1.0)
    if c["wide"]:
        buf = torch.zeros(M, K + 64, dtype=dt, device=dev)
        buf[:, :K] = x
        x = buf[:, :K]
    else:
        x = x.to(dt)
    out = dict(x=x, dy=None, bias=None, codes=None, scales=None)
    if c["op"] != "quantize":
        w = normal(N, K).mul_(0.02).mul_(torch.exp(0.3 * normal(N, 1)))
        out["codes"], out["scales"] = encode(w)
        if c["bias"]:
            out["bias"] = normal(N).mul_(0.1).to(dt)
        if c["op"] == "grad":
            out["dy"] = normal(M, N).mul_(0.01).to(dt)
    return out


def prepare(case, seed):
    st = tensors(case, seed)
    st["op"] = case["op"]
    if own and st["codes"] is not None:
        from lumen.ops.mxfp4 import MXFP4

        st["w"] = MXFP4(st.pop("codes"), st.pop("scales"))
    if case["op"] == "grad":
        st["x"].requires_grad_(own)
    return st


# ---- one pass --------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from lumen.ops.mxfp4 import mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize

    op, x = s["op"], s["x"]
    if op == "quantize":
        return mxfp4_dequantize(mxfp4_quantize(x), x.dtype)
    if op == "matmul":
        return mxfp4_matmul(mxfp4_quantize(x), s["w"], bias=s["bias"], out_dtype=x.dtype)
    y = mxfp4_linear(x, s["w"], s["bias"])
    if op == "linear":
        return y
    (dx,) = torch.autograd.grad(y, x, s["dy"])
    return y.detach(), dx


def _plain(s):
    op, x, dt = s["op"], s["x"], s["x"].dtype
    if op == "quantize":
        return decode(*encode(x)).to(dt)
    w = decode(s["codes"], s["scales"])
    if op == "matmul":
        a = decode(*encode(x))
    else:
        a, w = x.float(), w.to(dt).float()
    y = torch.matmul(a, w.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if op != "grad":
        return y.to(dt)
    return y.to(dt), torch.matmul(s["dy"].float(), w).to(dt)


def work(case):
    M, N, K, op = case["rows"], case["n"], case["k"], case["op"]
    packed = K // 2 + K // BLOCK                         # bytes of a quantised row
    if op == "quantize":                                 # x read, codes written, read again, values written
        return {"bytes": M * (4 * K + 2 * packed), "flops": 0}
    b = 2 * M * K + N * packed + 2 * M * N + (2 * N if case["bias"] else 0)
    if op != "grad":
        return {"bytes": b, "flops": 2 * M * N * K}
    return {"bytes": b + 2 * M * N + N * packed + 2 * M * K, "flops": 4 * M * N * K}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def _nearest(x):
    """x [R, K] in float64 -> the values of its MXFP4 form: nearest of the eight magnitudes, by their midpoints."""
    R, K = x.shape
    b = x.to(F64).view(R, -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))
    e = torch.where(torch.pow(2.0, e) > top, e - 1, e)             # (the logarithm may round across a power of two)
    e = torch.where(torch.pow(2.0, e + 1) <= top, e + 1, e)
    unit = torch.pow(2.0, (e - 2).clamp(-127, 127))
    m = b.abs() / unit
    out = torch.zeros_like(m)
    # midpoint, value above it, whether the midpoint itself goes up (to the even code)
    for mid, val, up in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True),
                         (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
        over = m >= mid if up else m > mid
        out = torch.where(over, torch.full_like(out, val), out)
    return (torch.copysign(out, b) * unit).view(R, K)


def _stands_for(codes, scales):
    """Codes and scales -> float64 values, from the bits: sign, two of exponent, one of fraction."""
    R = codes.shape[0]
    c = torch.stack((codes.long() & 15, codes.long() >> 4), -1).view(R, -1)
    ex, fr = (c >> 1) & 3, (c & 1).to(F64)
    mag = torch.where(ex == 0, fr * 0.5, (1 + 0.5 * fr) * torch.pow(2.0, (ex - 1).to(F64)))
    unit = torch.pow(2.0, scales.to(F64) - 127).repeat_interleave(BLOCK, 1)
    return torch.where(c >= 8, -mag, mag) * unit


def _times_nt(a, b):
    """a [M, K] times b [N, K]^T in float64."""
    return torch.matmul(a, b.t())


def exact(case, seed):
    t = tensors(case, seed)
    op, x, dt = case["op"], t["x"], t["x"].dtype
    if op == "quantize":
        return _nearest(x)
    w = _stands_for(t["codes"], t["scales"])
    if op == "matmul":
        a = _nearest(x)
    else:
        a, w = x.to(F64), w.to(dt).to(F64)
    y = _times_nt(a, w)
    if t["bias"] is not None:
        y = y + t["bias"].to(F64)
    if op != "grad":
        return y
    return y, torch.matmul(t["dy"].to(F64), w)
