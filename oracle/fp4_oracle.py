"""CPU restatement of the 4-bit floating point formats in 64 bits (test infrastructure).

quantize(x, scheme) -> (codes uint8 [M, Kp], scale bytes uint8 [M, Kp / g], row scale fp32 [M] or None), from the
definitions alone: every quotient is formed in fp64, where the borders between two codes of 16-bit inputs are exact
(a quotient of an 11-bit and a 4-bit number that is no border is at least 2^-17 of itself away from one).
"""
from __future__ import annotations

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def e2m1(v: torch.Tensor) -> torch.Tensor:
    """Nearest code of v (fp64): ties to the even code, 6 beyond, the sign bit kept."""
    mid = (MAGNITUDES[1:] + MAGNITUDES[:-1]) / 2
    a = v.abs()
    code = torch.zeros(v.shape, dtype=torch.uint8)
    for i, m in enumerate(mid):  # from code i to i + 1; a tie goes up to an even code
        code += ((a > m) | ((a == m) & (i % 2 == 1))).to(torch.uint8)
    return code + 8 * torch.signbit(v).to(torch.uint8)


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 byte of v >= 0 (fp64, at most 448): 3 mantissa bits, exponents -6..8, denormals of 2^-9."""
    e = torch.frexp(v)[1].to(torch.float64) - 1
    step = torch.exp2(e.clamp(-6, 8) - 3)
    q = torch.round(v / step) * step
    return q.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)  # exact: q is representable


def pow2(e: torch.Tensor) -> torch.Tensor:
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantize(x: torch.Tensor, scheme: str):
    g = BLOCK[scheme]
    M, K = x.shape
    xp = torch.zeros(M, (K + 31) // 32 * 32, dtype=torch.float64)
    xp[:, :K] = x.double()
    b = xp.view(M, -1, g)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b)
    top = b.abs().amax(-1)
    if scheme == "mxfp4":
        e = torch.frexp(top)[1].to(torch.int64) - 1 - 2
        e = torch.where(top > 0, e.clamp(-127, 127), torch.full_like(e, -127))
        sf = (e + 127).to(torch.uint8)
        codes = e2m1(b * pow2(-e).unsqueeze(-1))
        row = None
    else:
        m, ex = torch.frexp(top.amax(-1) / 2688)  # exact enough: 2688 has 7 bits, a tie only at m == 0.5
        er = torch.where(m == 0.5, ex - 1, ex).to(torch.int64)
        er = torch.where(m > 0, er.clamp(min=-126), torch.full_like(er, -126))
        unit = pow2(-er).view(-1, 1)
        sf = e4m3(top * unit / 6)
        d = sf.view(torch.float8_e4m3fn).double().unsqueeze(-1)
        v = b * unit.unsqueeze(-1)
        codes = e2m1(torch.where(d > 0, v / d.clamp_min(2.0 ** -20), torch.copysign(torch.zeros_like(v), v)))
        row = pow2(er).float()
    sf = torch.where(bad, torch.full_like(sf, 0xFF if scheme == "mxfp4" else 0x7F), sf)
    return codes.view(M, -1), sf, row


def values(codes: torch.Tensor, sf: torch.Tensor, row: torch.Tensor | None, scheme: str) -> torch.Tensor:
    """What codes and scales stand for, in fp64 [M, Kp]."""
    M, Kp = codes.shape
    v = MAGNITUDES[(codes & 7).long()]
    v = torch.where(codes >= 8, -v, v)
    if scheme == "mxfp4":
        s = pow2(sf.to(torch.int64) - 127)
        s = torch.where(sf == 0xFF, torch.full_like(s, float("nan")), s)
    else:
        s = sf.view(torch.float8_e4m3fn).double()
    v = (v.view(M, -1, BLOCK[scheme]) * s.unsqueeze(-1)).view(M, Kp)
    return v if row is None else v * row.double().unsqueeze(-1)


def pack(codes: torch.Tensor) -> torch.Tensor:
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()


def unpack(data: torch.Tensor) -> torch.Tensor:
    return torch.stack((data & 15, data >> 4), -1).view(data.shape[0], -1)
