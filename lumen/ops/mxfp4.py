"""Microscaled 4-bit floating point (MXFP4): quantisation, and products with quantised operands.

A row is cut into blocks of 32 values; a block holds one power of two, 2^e with e = floor(log2(largest magnitude)) - 2 (its
byte is e + 127), and 32 four-bit numbers: +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, the nearest to value / 2^e (ties to the even
code, 6 beyond it).  Two share a byte, the first in its low half.  A block with an infinity or a NaN becomes NaN (byte 255).

    w = mxfp4_quantize(weight)                 # [N, K] -> MXFP4: 4.25 bits a value
    y = mxfp4_linear(x, w, bias)               # 16-bit rows, 4-bit weight; differentiable in x
    y = mxfp4_matmul(mxfp4_quantize(x), w)     # both operands in 4 bits, on the scaled matrix instructions
    mxfp4_dequantize(w, torch.bfloat16)

On the GPU these are HIP kernels (``csrc/seqmix/mxfp4.hip``, ``mx_*.hip``); CPU tensors take the torch path below.  The
weight holds no gradient: it is the frozen base of adapters, or served.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
import torch.nn.functional as F

from ._seqmix import DT, call, use_seqmix

BLOCK = 32                # values that share a scale
PANEL = 128               # values of a row that lie together (csrc/seqmix/mxfp4.hip)
MAX_K, MAX_ROWS = 1 << 23, 1 << 24
HALF = (torch.bfloat16, torch.float16)


class MXFP4:
    """A matrix [rows, K] in MXFP4: ``codes`` uint8 [rows, K / 2], ``scales`` uint8 [rows, K / 32].

    Built from such tensors (of another program's checkpoint, say) or by ``mxfp4_quantize``.  It holds them in panels of 128
    values, [panel, row, 64] and [panel, row, 4] bytes, zeros behind a row's end, as the kernels read them; ``codes`` and
    ``scales`` give copies in rows."""

    __slots__ = ("shape", "_codes", "_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("MXFP4: codes [rows, K / 2] and scales [rows, K / 32], both uint8")
        R, K = codes.shape[0], 2 * codes.shape[1]
        if scales.shape[0] != R or scales.shape[1] * BLOCK != K:
            raise ValueError(f"MXFP4: scales {list(scales.shape)} do not fit codes {list(codes.shape)}")
        if not 0 < K <= MAX_K or R > MAX_ROWS:
            raise ValueError(f"MXFP4: {R} rows of {K} values (at most {MAX_ROWS}, and 32 to {MAX_K})")
        if codes.device != scales.device:
            raise ValueError(f"MXFP4: codes on {codes.device}, scales on {scales.device}")
        self.shape = (R, K)
        self._codes = _panels(codes.detach(), PANEL // 2)
        self._scales = _panels(scales.detach(), PANEL // BLOCK)

    @property
    def codes(self) -> torch.Tensor:
        return _rows_of(self._codes)[:, :self.shape[1] // 2]

    @property
    def scales(self) -> torch.Tensor:
        return _rows_of(self._scales)[:, :self.shape[1] // BLOCK]

    @property
    def device(self) -> torch.device:
        return self._codes.device

    @property
    def nbytes(self) -> int:
        return self._codes.numel() + self._scales.numel()

    def to(self, device) -> "MXFP4":
        return _of(self._codes.to(device), self._scales.to(device), self.shape[1])

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return mxfp4_dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MXFP4({self.shape[0]} x {self.shape[1]}, {self.device})"


def _panels(t: torch.Tensor, unit: int) -> torch.Tensor:
    """[rows, n] bytes -> [panels, rows, unit], zeros behind a row's last one."""
    R, n = t.shape
    P = -(-n // unit)
    out = torch.zeros(P, R, unit, dtype=t.dtype, device=t.device)
    whole = n // unit
    out[:whole].copy_(t[:, :whole * unit].reshape(R, whole, unit).transpose(0, 1))
    if whole < P:
        out[whole, :, :n - whole * unit].copy_(t[:, whole * unit:])
    return out


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[panels, rows, unit] bytes -> [rows, panels * unit], a copy."""
    P, R, unit = t.shape
    return t.transpose(0, 1).reshape(R, P * unit)


def _of(codes: torch.Tensor, scales: torch.Tensor, K: int) -> MXFP4:
    q = MXFP4.__new__(MXFP4)
    q.shape, q._codes, q._scales = (codes.shape[1], K), codes, scales
    return q


def _rows(x: torch.Tensor, unit: int = 8) -> torch.Tensor:
    """``x`` [rows, K] itself where its rows are contiguous and at 16-byte addresses, else a copy."""
    if x.is_neg():
        x = x.resolve_neg()
    if x.stride(1) == 1 and x.data_ptr() % 16 == 0 and (x.shape[0] < 2 or x.stride(0) % unit == 0 and x.stride(0) >= x.shape[1]):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _on(device: torch.device):
    """The device's context (its current stream) where it is not the current one already."""
    return torch.cuda.device(device)


# ---- the format -------------------------------------------------------------------------------------
def mxfp4_quantize(x: torch.Tensor) -> MXFP4:
    """The MXFP4 form of x [rows, K] (fp32, bf16 or fp16; K a multiple of 32)."""
    if x.dim() != 2 or x.dtype not in DT:
        raise ValueError("mxfp4_quantize: a matrix [rows, K] of fp32, bf16 or fp16")
    R, K = x.shape
    if K % BLOCK or not 0 < K <= MAX_K or R > MAX_ROWS:
        raise ValueError(f"mxfp4_quantize: {R} rows of {K} values (at most {MAX_ROWS}; a multiple of {BLOCK}, at most {MAX_K})")
    x = x.detach()
    if not use_seqmix(x):
        return MXFP4(*_encode(x))
    P = -(-K // PANEL)
    codes = torch.empty(P, R, PANEL // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(P, R, PANEL // BLOCK, dtype=torch.uint8, device=x.device)
    if R:
        with _on(x.device):
            x = _rows(x, 16 // x.element_size())
            call("sm_mx_quantize", DT[x.dtype], x, _ld(x), codes, scales, R, K)
    return _of(codes, scales, K)


def mxfp4_dequantize(q: MXFP4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, K] that ``q`` stands for: exact in fp32 and bf16, in fp16 rounded to it (exact between 2^-24 and
    its largest number).  What lies beyond ``dtype``'s largest number becomes infinite."""
    if dtype not in DT:
        raise ValueError("mxfp4_dequantize: fp32, bf16 or fp16")
    R, K = q.shape
    if not use_seqmix(q._codes):
        return _decode(q.codes, q.scales).to(dtype)
    y = torch.empty(R, K, dtype=dtype, device=q.device)
    if R:
        with _on(q.device):
            call("sm_mx_dequantize", DT[dtype], q._codes, q._scales, y, R, K)
    return y


_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _power(s: torch.Tensor) -> torch.Tensor:
    """2^(s - 127) of scale bytes as fp32, 255: NaN."""
    bits = s.int() << 23
    bits = torch.where(s == 0, torch.full_like(bits, 1 << 22), torch.where(s == 255, torch.full_like(bits, 0x7fc00000), bits))
    return bits.view(torch.float32)


def _encode(x: torch.Tensor):
    R, K = x.shape
    b = x.float().reshape(R, K // BLOCK, BLOCK)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = (top.contiguous().view(torch.int32) >> 23) - 2             # (exponent field: 0 of zero and denormals)
    s = torch.where(bad, torch.full_like(e, 255), e.clamp(min=0))
    m = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b).double() / _power(s.where(~bad, torch.zeros_like(s))).double().unsqueeze(-1)
    a = m.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8) | (torch.signbit(m).to(torch.uint8) << 3)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).reshape(R, K // 2, 2)
    return code[..., 0] | code[..., 1] << 4, s.to(torch.uint8)


def _decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    lut = torch.tensor(_VALUES, dtype=torch.float32, device=codes.device)
    R, n = scales.shape
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).reshape(R, n, BLOCK)
    return (v * _power(scales).unsqueeze(-1)).reshape(R, n * BLOCK)


def _best(M: int, N: int, tiles, cost) -> tuple:
    """The tile of ``tiles`` (rows, columns, ...) whose rounds of 256 workgroups take the least time, ``cost`` a stage."""
    return min(tiles, key=lambda t: -(-(-(-M // t[0]) * -(-N // t[1])) // 256) * cost(t))


_LINEAR = [(32 * mj, 32 * ni, mj, ni) for mj, ni in ((8, 8), (8, 6), (8, 4), (8, 2), (4, 8), (4, 4), (4, 2), (2, 8), (2, 4), (2, 2), (2, 1), (1, 8),
                                                    (1, 4), (1, 2), (1, 1))]
_MATMUL = [t for t in _LINEAR if t[2:] not in ((8, 6), (8, 2))]
_GRAD = [(64 * mj // wn, 128 * wn, mj, wn) for mj, wn in ((8, 2), (4, 2), (2, 2), (1, 2), (4, 1), (2, 1), (1, 1))]


@functools.lru_cache(4096)
def _linear_tile(M: int, N: int) -> tuple:
    return _best(M, N, _LINEAR, lambda t: max(t[0] * t[1] / 32, (t[0] * 128 + t[1] * 36) / 48) + 200)[2:]


@functools.lru_cache(4096)
def _grad_tile(M: int, K: int) -> tuple:
    return _best(M, K, _GRAD, lambda t: max(t[0] * t[1] / 32, (t[0] * 128 + t[1] * 36) / 48) + 400)[2:]


@functools.lru_cache(4096)
def _matmul_tile(M: int, N: int) -> tuple:
    return _best(M, N, _MATMUL, lambda t: max(t[0] * t[1] / 64, (t[0] + t[1]) * 68 / 48) + 200)[2:]


# ---- products ---------------------------------------------------------------------------------------
def _check(name: str, K: int, device, w, bias: Optional[torch.Tensor], dtype: torch.dtype) -> None:
    if not isinstance(w, MXFP4):
        raise ValueError(f"{name}: the weight is no MXFP4 matrix (mxfp4_quantize makes one)")
    if w.shape[1] != K:
        raise ValueError(f"{name}: rows of {K} values against a weight of {w.shape[1]}")
    if w.device != device:
        raise ValueError(f"{name}: rows on {device}, weight on {w.device}")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != w.shape[0] or bias.dtype != dtype or bias.device != device):
        raise ValueError(f"{name}: the bias is not [{w.shape[0]}] values of {dtype} on {device}")


def _linear(x: torch.Tensor, w: MXFP4, bias: Optional[torch.Tensor]) -> torch.Tensor:
    """``mxfp4_linear`` of checked rows [M, K], without autograd."""
    (M, K), N = x.shape, w.shape[0]
    if not use_seqmix(x):
        y = x.float() @ _decode(w.codes, w.scales).to(x.dtype).float().t()
        return (y if bias is None else y + bias.float()).to(x.dtype)
    y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    if M and N:
        with _on(x.device):
            x = _rows(x)
            call("sm_mx_linear", DT[x.dtype], x, _ld(x), w._codes, w._scales, None if bias is None else bias.contiguous(), y, M, N, K, *_linear_tile(M, N))
    return y


def _input_grad(dy: torch.Tensor, w: MXFP4) -> torch.Tensor:
    """dx [M, K] = dy [M, N] times the weight's values in dy's type."""
    (M, N), K = dy.shape, w.shape[1]
    if not use_seqmix(dy):
        return (dy.float() @ _decode(w.codes, w.scales).to(dy.dtype).float()).to(dy.dtype)
    if not (M and N):
        return torch.zeros(M, K, dtype=dy.dtype, device=dy.device)
    dx = torch.empty(M, K, dtype=dy.dtype, device=dy.device)
    with _on(dy.device):
        dy = F.pad(dy, (0, -N % 8)) if N % 8 else _rows(dy)          # (rows at 16-byte addresses, zeros behind them)
        call("sm_mx_grad", DT[dy.dtype], dy, _ld(dy), w._codes, w._scales, dx, M, N, K, *_grad_tile(M, K))
    return dx


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias):
        ctx.save_for_backward(w._codes, w._scales)
        ctx.K = w.shape[1]
        return _linear(x, w, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        return _input_grad(dy, _of(codes, scales, ctx.K)), None, None


def mxfp4_linear(x: torch.Tensor, w: MXFP4, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] @ W^T (+ ``bias`` [N]) for a weight [N, K] in MXFP4: W's values in x's type (``mxfp4_dequantize``), fp32
    sums, one rounding to x's type (bf16 or fp16; on the CPU fp32 too).  Differentiable in x, not in the weight or the bias."""
    if x.dim() < 1 or x.dtype not in (DT if not x.is_cuda else HALF):
        raise ValueError("mxfp4_linear: rows [..., K] of bf16 or fp16")
    K = x.shape[-1]
    _check("mxfp4_linear", K, x.device, w, bias, x.dtype)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("mxfp4_linear: the bias has no gradient here (freeze it, or add it to the result)")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if torch.is_grad_enabled() and x.requires_grad:
        y = _Linear.apply(x2, w, bias)
    else:
        y = _linear(x2, w, bias)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.shape[0])


def mxfp4_matmul(a: MXFP4, b: MXFP4, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] @ b [N, K]^T (+ ``bias`` [N] of ``out_dtype``) of two MXFP4 matrices: fp32 sums of their exact products, one
    rounding to ``out_dtype`` (bf16, fp16 or fp32).  No gradient: activations that need one stay in 16 bits (``mxfp4_linear``)."""
    if not isinstance(a, MXFP4):
        raise ValueError("mxfp4_matmul: the rows are no MXFP4 matrix (mxfp4_quantize makes one)")
    if out_dtype not in DT:
        raise ValueError("mxfp4_matmul: results in bf16, fp16 or fp32")
    (M, K) = a.shape
    _check("mxfp4_matmul", K, a.device, b, bias, out_dtype)
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("mxfp4_matmul: the bias has no gradient here")
    N = b.shape[0]
    if not use_seqmix(a._codes):
        y = _decode(a.codes, a.scales) @ _decode(b.codes, b.scales).t()
        return (y if bias is None else y + bias.float()).to(out_dtype)
    y = torch.empty(M, N, dtype=out_dtype, device=a.device)
    if M and N:
        with _on(a.device):
            call("sm_mx_matmul", DT[out_dtype], a._codes, a._scales, b._codes, b._scales,
                 None if bias is None else bias.contiguous(), y, M, N, K, *_matmul_tile(M, N))
    return y
