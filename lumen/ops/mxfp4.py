"""Microscaled 4-bit floating point (MXFP4): quantisation, and products with quantised operands.

A row is cut into blocks of 32 values (the last one holds what is left); a block holds one power of two, 2^e with e = floor(log2(largest magnitude)) - 2 (its
byte is e + 127), and 32 four-bit numbers: +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, the nearest to value / 2^e (ties to the even
code, 6 beyond it).  Two share a byte, the first in its low half.  A block with an infinity or a NaN becomes NaN (byte 255).

    w = mxfp4_quantize(weight)                 # [N, K] -> MXFP4: 4.25 bits a value
    y = mxfp4_linear(x, w, bias)               # 16-bit rows, 4-bit weight; differentiable in x
    y = mxfp4_matmul(mxfp4_quantize(x), w)     # both operands in 4 bits, on the scaled matrix instructions
    mxfp4_dequantize(w, torch.bfloat16)

On the GPU these are HIP kernels (``csrc/seqmix/mxfp4.hip``, ``mx_*.hip``; ``csrc/mx_calls.cpp`` calls them); CPU tensors take the torch path below.  The
weight holds no gradient: it is the frozen base of adapters, or served.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch
import torch.nn.functional as F

from . import _seqmix
from ._native import native, native_error
from ._seqmix import DT

BLOCK = 32                # values that share a scale
PANEL = 128               # values of a row that lie together (csrc/seqmix/mxfp4.hip)
MAX_K, MAX_ROWS = 1 << 23, 1 << 24
MAX_LD = 1 << 22          # values from row to row that the products take
HALF = (torch.bfloat16, torch.float16)


class MXFP4:
    """A matrix [rows, K] in MXFP4, K a multiple of 8: ``codes`` uint8 [rows, K / 2], ``scales`` uint8 [rows, K / 32 rounded up].

    Built from such tensors (of another program's checkpoint, say) or by ``mxfp4_quantize``.  It holds them as the kernels read
    them, in panels of 128 values of all rows: [panel, row, 64] bytes of codes, then [panel, row, 4] of scales, zeros behind a
    row's end; ``codes`` and ``scales`` give copies in rows."""

    __slots__ = ("shape", "data")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("MXFP4: codes [rows, K / 2] and scales [rows, K / 32 rounded up], both uint8")
        R, K = codes.shape[0], 2 * codes.shape[1]
        if scales.shape[0] != R or scales.shape[1] != -(-K // BLOCK):
            raise ValueError(f"MXFP4: scales {list(scales.shape)} do not fit codes {list(codes.shape)}")
        if K % 8 or not 0 < K <= MAX_K or R > MAX_ROWS:
            raise ValueError(f"MXFP4: {R} rows of {K} values (at most {MAX_ROWS}; a multiple of 8, at most {MAX_K})")
        if codes.device != scales.device:
            raise ValueError(f"MXFP4: codes on {codes.device}, scales on {scales.device}")
        self.shape = (R, K)
        self.data = torch.zeros(_nbytes(R, K), dtype=torch.uint8, device=codes.device)
        _fill(self._codes, codes.detach())
        _fill(self._scales, scales.detach())

    @property
    def _codes(self) -> torch.Tensor:
        R, K = self.shape
        P = -(-K // PANEL)
        return self.data[:P * R * 64].view(P, R, 64)

    @property
    def _scales(self) -> torch.Tensor:
        R, K = self.shape
        P = -(-K // PANEL)
        return self.data[P * R * 64:].view(P, R, 4)

    @property
    def codes(self) -> torch.Tensor:
        return _rows_of(self._codes)[:, :self.shape[1] // 2]

    @property
    def scales(self) -> torch.Tensor:
        return _rows_of(self._scales)[:, :-(-self.shape[1] // BLOCK)]

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def to(self, device) -> "MXFP4":
        return of_data(self.data.to(device=device), self.shape)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return mxfp4_dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MXFP4({self.shape[0]} x {self.shape[1]}, {self.device})"


def _nbytes(R: int, K: int) -> int:
    return -(-K // PANEL) * R * 68


def _fill(panels: torch.Tensor, t: torch.Tensor) -> None:
    """[rows, n] bytes into [panels, rows, unit] ones."""
    unit, n = panels.shape[2], t.shape[1]
    whole = n // unit
    panels[:whole].copy_(t[:, :whole * unit].reshape(t.shape[0], whole, unit).transpose(0, 1))
    if n % unit:
        panels[whole, :, :n % unit].copy_(t[:, whole * unit:])


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[panels, rows, unit] bytes -> [rows, panels * unit], a copy."""
    P, R, unit = t.shape
    return t.transpose(0, 1).reshape(R, P * unit)


def of_data(data: torch.Tensor, shape: tuple) -> MXFP4:
    """The [rows, K] matrix whose ``data`` this is."""
    q = MXFP4.__new__(MXFP4)
    q.data, q.shape = data, shape
    return q


# what csrc/mx_calls.cpp launches, in its order
_LAUNCHERS = ("sm_mx_quantize", "sm_mx_dequantize", "sm_mx_linear", "sm_mx_rows", "sm_mx_grad", "sm_mx_rows_grad", "sm_mx_matmul",
              "sm_mx_rows_matmul")
_calls = None


def _native_calls():
    """The extension's calls, with the kernel library's launchers handed to them once."""
    global _calls
    if _calls is None:
        lib, C = _seqmix._load(), native()
        if lib is None or C is None:
            raise RuntimeError(f"lumen kernels are not available ({_seqmix.seqmix_error() or native_error()!r}); build them with "
                               "`python -m lumen.csrc.build`")
        C.mx_launchers([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _LAUNCHERS])
        _calls = C
    return _calls


# ---- the format -------------------------------------------------------------------------------------
def mxfp4_quantize(x: torch.Tensor) -> MXFP4:
    """The MXFP4 form of x [rows, K] (fp32, bf16 or fp16; K a multiple of 8).  No gradient passes: the result stands outside the
    graph as that of ``x.detach()`` does, and so does what is multiplied with it (``mxfp4_linear`` has the gradient of 16-bit rows)."""
    if x.dim() != 2 or x.dtype not in DT:
        raise ValueError("mxfp4_quantize: a matrix [rows, K] of fp32, bf16 or fp16")
    R, K = x.shape
    if K % 8 or not 0 < K <= MAX_K or R > MAX_ROWS:
        raise ValueError(f"mxfp4_quantize: {R} rows of {K} values (at most {MAX_ROWS}; a multiple of 8, at most {MAX_K})")
    if not x.is_cuda:
        return MXFP4(*_encode(x.detach()))
    return of_data((_calls or _native_calls()).mx_quantize(x), (R, K))


def mxfp4_dequantize(q: MXFP4, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, K] that ``q`` stands for: exact in fp32 and bf16, in fp16 rounded to it (exact between 2^-24 and
    its largest number).  What lies beyond ``dtype``'s largest number becomes infinite."""
    if dtype not in DT:
        raise ValueError("mxfp4_dequantize: fp32, bf16 or fp16")
    if not q.data.is_cuda:
        return _decode(q.codes, q.scales).to(dtype)
    return (_calls or _native_calls()).mx_dequantize(q.data, *q.shape, dtype)


_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _power(s: torch.Tensor) -> torch.Tensor:
    """2^(s - 127) of scale bytes as fp32, 255: NaN."""
    bits = s.int() << 23
    bits = torch.where(s == 0, torch.full_like(bits, 1 << 22), torch.where(s == 255, torch.full_like(bits, 0x7fc00000), bits))
    return bits.view(torch.float32)


def _encode(x: torch.Tensor):
    R, K = x.shape
    n = -(-K // BLOCK)
    b = F.pad(x.float(), (0, n * BLOCK - K)).reshape(R, n, BLOCK)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = (top.contiguous().view(torch.int32) >> 23) - 2             # (exponent field: 0 of zero and denormals)
    s = torch.where(bad, torch.full_like(e, 255), e.clamp(min=0))
    m = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b).double() / _power(s.where(~bad, torch.zeros_like(s))).double().unsqueeze(-1)
    a = m.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = (torch.round(a / step) * step).clamp(max=6.0)
    code = torch.where(r < 2, r * 2, torch.where(r < 4, r + 2, r / 2 + 4)).to(torch.uint8) | (torch.signbit(m).to(torch.uint8) << 3)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).reshape(R, n * BLOCK)[:, :K].reshape(R, K // 2, 2)
    return code[..., 0] | code[..., 1] << 4, s.to(torch.uint8)


def _decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    lut = torch.tensor(_VALUES, dtype=torch.float32, device=codes.device)
    (R, n), K = scales.shape, 2 * codes.shape[1]
    v = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).reshape(R, K)
    v = F.pad(v, (0, n * BLOCK - K)).reshape(R, n, BLOCK)
    return (v * _power(scales).unsqueeze(-1)).reshape(R, n * BLOCK)[:, :K]


# What a round of 256 workgroups takes, us (bf16, weights from HBM), as a time a stage of 64 k and one beside them: a + b rt and f + g rt on the
# few-row kernel's xr x 16 rt results, c and e on tiles of 32 mj x 32 ni (the kernels say what either form takes).  Over 222 sizes of 1 to
# 4096 rows, all three products, the form chosen takes 0.5 % more than the best of the seven that this predicts to be fastest, 12 % at worst.
_ROWS = [(xr, 16 * rt, (0, xr, rt), a + b * rt, f + g * rt)
         for xr, a, b, f, g, rts in ((16, 0.03, 0.0075, 1.8, 0.4, (1, 2, 3, 4, 6, 8)), (32, 0.065, 0.012, 1.9, 0.5, (1, 2, 3, 4, 6)),
                                     (32, 0.21, 0.0, 5.0, 0.0, (8,)), (64, 0.09, 0.017, 2.3, 0.5, (2, 3, 4, 6, 8)))
         for rt in rts]
_TILES = [(32 * mj, 32 * ni, (1, mj, ni), c, e)
          for mj, ni, c, e in ((4, 4, 0.48, 9.0), (4, 6, 0.63, 7.5), (6, 4, 0.6, 8.5), (8, 4, 0.77, 8.0), (8, 6, 1.04, 9.5), (8, 8, 1.29, 12.0))]


def _best(M: int, N: int, K: int, forms) -> tuple:
    """The form of ``forms`` (rows, columns, form, us a stage, us beside) whose rounds of workgroups take the least time."""
    return min(forms, key=lambda f: -(-(-(-M // f[0]) * -(-N // f[1])) // 256) * (f[3] * (K / 64) + f[4]))[2]


@functools.lru_cache(4096)
def _linear_form(M: int, N: int, K: int) -> tuple:
    """(0, rows, 16 columns) of the few-row kernel or (1, mj, ni) of the tiles for x [M, K] against a weight [N, K]."""
    return _best(M, N, K, _ROWS + _TILES)


# both operands in 4 bits
_MATMUL = ([(xr, 16 * rt, (0, xr, rt), (a + b * rt) / 2, f + g * rt)
            for xr, a, b, f, g, rts in ((16, 0.05, 0.0125, 2.9, 0.1, (1, 2, 4, 6, 8)), (32, 0.05, 0.015, 3.3, 0.1, (1, 2, 4, 6, 8)),
                                        (64, 0.087, 0.013, 2.8, 0.4, (1, 2, 3, 4, 6, 8)), (128, 0.0, 0.048, 0.0, 1.4, (4,)))
            for rt in rts]
           + [(32 * mj, 32 * ni, (1, mj, ni), c, e)
              for mj, ni, c, e in ((4, 4, 0.173, 7.0), (4, 6, 0.25, 6.3), (6, 4, 0.24, 6.6), (8, 4, 0.3, 7.3), (8, 6, 0.355, 9.0), (8, 8, 0.44, 9.0))])


@functools.lru_cache(4096)
def _matmul_form(M: int, N: int, K: int) -> tuple:
    """(0, rows, 16 columns) of the few-row kernel or (1, mj, ni) of the tiles."""
    return _best(M, N, K, _MATMUL)


# the gradient likewise, a stage 64 of the weight's rows
_GRAD = ([(xr, 128, (0, xr, 0), c, e) for xr, c, e in ((16, 0.15, 4.5), (32, 0.2, 4.6), (64, 0.25, 5.2))]
         + [(32 * mj, 256, (1, mj, 0), c, e) for mj, c, e in ((4, 0.85, 11.5), (6, 1.13, 12.2), (8, 1.42, 13.3))])


@functools.lru_cache(4096)
def _grad_form(M: int, N: int, K: int) -> tuple:
    """(0, rows, 0) of the few-row kernel or (1, mj, 0) of the tiles for dy [M, N] against a weight [N, K]."""
    return _best(M, K, N, _GRAD)


# ---- products ---------------------------------------------------------------------------------------
def _check(name: str, K: int, device, w, bias: Optional[torch.Tensor], dtype: torch.dtype) -> None:
    if type(w) is not MXFP4:
        raise ValueError(f"{name}: the weight is no MXFP4 matrix (mxfp4_quantize makes one)")
    if w.shape[1] != K:
        raise ValueError(f"{name}: rows of {K} values against a weight of {w.shape[1]}")
    if w.data.device != device:
        raise ValueError(f"{name}: rows on {device}, weight on {w.device}")
    if K > MAX_LD:
        raise ValueError(f"{name}: rows of {K} values (at most {MAX_LD})")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != w.shape[0] or bias.dtype != dtype or bias.device != device:
            raise ValueError(f"{name}: the bias is not [{w.shape[0]}] values of {dtype} on {device}")
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name}: the bias has no gradient here (freeze it, or add it to the result)")


def linear_rows(x: torch.Tensor, w: MXFP4, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mxfp4_linear`` of rows [M, K], on the GPU without autograd (and checked there by the extension alone)."""
    M, (N, K) = x.shape[0], w.shape
    if not x.is_cuda:
        y = x.float() @ _decode(w.codes, w.scales).to(x.dtype).float().t()
        return (y if bias is None else y + bias.float()).to(x.dtype)
    return (_calls or _native_calls()).mx_linear(x, w.data, N, K, bias, *_linear_form(M, N, K))


def input_grad(dy: torch.Tensor, w: MXFP4) -> torch.Tensor:
    """dx [M, K] = dy [M, N] times the weight's values in dy's type."""
    M, (N, K) = dy.shape[0], w.shape
    if not dy.is_cuda:
        return (dy.float() @ _decode(w.codes, w.scales).to(dy.dtype).float()).to(dy.dtype)
    return (_calls or _native_calls()).mx_grad(dy, w.data, N, K, *_grad_form(M, N, K))


def mxfp4_linear(x: torch.Tensor, w: MXFP4, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] @ W^T (+ ``bias`` [N]) for a weight [N, K] in MXFP4: W's values in x's type (``mxfp4_dequantize``), fp32
    sums, one rounding to x's type (bf16 or fp16; on the CPU fp32 too).  Differentiable in x, not in the weight or the bias."""
    if x.dim() < 1 or x.dtype not in (HALF if x.is_cuda else DT):
        raise ValueError("mxfp4_linear: rows [..., K] of bf16 or fp16")
    sh = x.shape
    _check("mxfp4_linear", sh[-1], x.device, w, bias, x.dtype)
    x2 = x if len(sh) == 2 else x.reshape(-1, sh[-1])
    if x2.shape[0] > MAX_ROWS:
        raise ValueError(f"mxfp4_linear: {x2.shape[0]} rows (at most {MAX_ROWS})")
    if x.requires_grad and torch.is_grad_enabled() and x.is_cuda:
        (M, K), N = x2.shape, w.shape[0]
        if N > MAX_LD:
            raise ValueError(f"mxfp4_linear: {N} columns with a gradient (at most {MAX_LD})")
        y = (_calls or _native_calls()).mx_linear_tracked(x2, w.data, N, K, bias, *_linear_form(M, N, K), *_grad_form(M, N, K))
    else:
        y = linear_rows(x2, w, bias)
    return y if len(sh) == 2 else y.view(*sh[:-1], w.shape[0])


def mxfp4_matmul(a: MXFP4, b: MXFP4, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K] @ b [N, K]^T (+ ``bias`` [N] of ``out_dtype``) of two MXFP4 matrices: fp32 sums of their exact products, one
    rounding to ``out_dtype`` (bf16, fp16 or fp32).  No gradient: activations that need one stay in 16 bits (``mxfp4_linear``)."""
    if type(a) is not MXFP4:
        raise ValueError("mxfp4_matmul: the rows are no MXFP4 matrix (mxfp4_quantize makes one)")
    if out_dtype not in DT:
        raise ValueError("mxfp4_matmul: results in bf16, fp16 or fp32")
    (M, K), dev = a.shape, a.data.device
    _check("mxfp4_matmul", K, dev, b, bias, out_dtype)
    N = b.shape[0]
    if not a.data.is_cuda:
        y = _decode(a.codes, a.scales) @ _decode(b.codes, b.scales).t()
        return (y if bias is None else y + bias.float()).to(out_dtype)
    return (_calls or _native_calls()).mx_matmul(a.data, b.data, M, N, K, bias, out_dtype, *_matmul_form(M, N, K))
