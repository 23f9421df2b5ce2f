"""Oracle of the MXFP4 format and its products in float64, by search: shares no code with lumen."""
import math

import torch

MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def encode(x):
    """(codes [R, K], scale bytes [R, K / 32 rounded up]) of x [R, K] as integers: for every value the nearest magnitude, of two the even code."""
    R, K0 = x.shape
    K = -(-K0 // 32) * 32
    b = torch.zeros(R, K, dtype=torch.float64)            # (a last block of fewer values: as if zeros followed)
    b[:, :K0] = x.double().cpu()
    b = b.reshape(R, K // 32, 32)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    byte = torch.zeros_like(top, dtype=torch.long)
    for i in range(R):
        for j in range(K // 32):
            t = float(top[i, j])
            if bad[i, j]:
                byte[i, j] = 255
            elif t > 0:
                byte[i, j] = max(math.frexp(t)[1] - 1 - 2 + 127, 0)
    m = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b) / torch.pow(2.0, (byte.where(~bad, torch.full_like(byte, 127)) - 127).double()).unsqueeze(-1)
    dist = (m.abs().unsqueeze(-1) - torch.tensor(MAGS, dtype=torch.float64)).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best                                   # one or two neighbours
    idx = torch.arange(8)
    even = (near & (idx % 2 == 0)).any(-1)
    first = near.double().argmax(-1)
    pick = torch.where(even, (near & (idx % 2 == 0)).double().argmax(-1), first)
    code = pick + 8 * torch.signbit(m).long()
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code)
    return code.reshape(R, K)[:, :K0], byte


def decode(code, byte):
    """float64 values of integer codes and scale bytes."""
    mag = torch.tensor(MAGS, dtype=torch.float64)[code & 7]
    v = torch.where(code >= 8, -mag, mag)
    unit = torch.pow(2.0, (byte - 127).double())
    unit = torch.where(byte == 255, torch.full_like(unit, float("nan")), unit)
    return v * unit.repeat_interleave(32, 1)[:, :v.shape[1]]


def unpack(q):
    """Integer codes and bytes of a lumen MXFP4."""
    c = q.codes.cpu().long()
    return torch.stack((c & 15, c >> 4), -1).reshape(c.shape[0], -1), q.scales.cpu().long()


def values(q):
    return decode(*unpack(q))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, mag, terms, dtype):
    """got against float64 ``want``: ``terms`` roundings of fp32 sums of ``mag`` = sum of the products' magnitudes (a sum in any order is off
    by at most (terms - 1) half steps of it, twice that where the matrix core truncates), then half a step of ``dtype``; below
    its normal numbers half of the smallest one's step."""
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
    acc = mag * terms * 2.0 ** -23
    tol = acc + (want.abs() + acc) * half_step(dtype) + tiny
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), f"off by {float((err / tol).max()):.3g} of the tolerance"
