"""Microscaled formats in 64 bits, on torch tensors of any device: what codes
and scales stand for, and what a value may be quantised to.

Written from the definition (blocks of 32, scale ``2 ** (floor(log2 max|x|) -
emax)``, nearest element with ties to the even code, saturating), as searches
in the table of element values; nothing of the package is used.
"""

from __future__ import annotations

import torch

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8}
SIGN = {"mxfp4": 8, "mxfp8": 128}  # the code's sign bit


def pow2(e):
    """2 ** e as float64, from the exponent's bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def elements(fmt, device="cpu"):
    """Non-negative element values in the order of their codes."""
    if fmt == "mxfp4":
        v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        v = [m * 2.0 ** -9 for m in range(8)]
        v += [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
        v = v[:127]  # the code after 448 is NaN
    return torch.tensor(v, dtype=torch.float64, device=device)


def unpack(codes, fmt):
    if fmt == "mxfp8":
        return codes.long()
    return torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1).long()


def pack(codes, fmt):
    if fmt == "mxfp8":
        return codes.to(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def decode(codes, scales, fmt):
    """float64 values of packed codes ``[..., bytes]`` and scales ``[..., n / 32]``."""
    c = unpack(codes, fmt)
    grid = torch.cat((elements(fmt, c.device), torch.full((SIGN[fmt] - len(elements(fmt)),),
                                                          float("nan"), dtype=torch.float64,
                                                          device=c.device)))
    mag = grid[c & (SIGN[fmt] - 1)]
    s = pow2(scales.long() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return torch.where(c >= SIGN[fmt], -mag, mag) * s.repeat_interleave(BLOCK, -1)


def scale_bytes(amax, fmt):
    """Bytes of blocks with these largest magnitudes (float64; 255 where not finite)."""
    ok = torch.isfinite(amax) & (amax > 0)
    e = (torch.where(ok, amax, torch.ones_like(amax)).view(torch.int64) >> 52) - 1023
    b = torch.where(ok, (e - EMAX[fmt] + 127).clamp(0, 254), torch.zeros_like(e))
    return torch.where(torch.isfinite(amax), b, torch.full_like(b, 255))


def element_codes(v, fmt):
    """Codes (without sign) of magnitudes ``v``: the nearest element, ties to the even code."""
    grid = elements(fmt, v.device)
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.bucketize(v.contiguous(), mid), torch.bucketize(v.contiguous(), mid, right=True)
    return torch.where(lo % 2 == 0, lo, hi)


def quantize(x, fmt):
    """(codes not packed, scale bytes) of ``x [..., n]``, float64 values."""
    g = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    amax = torch.where(torch.isnan(g), torch.full_like(g, float("inf")), g.abs()).amax(-1)
    b = scale_bytes(amax.contiguous(), fmt)
    bad = (b == 255)[..., None]
    v = torch.where(bad, torch.zeros_like(g), g)
    v = v * pow2(127 - b[..., None])
    c = element_codes(v.abs(), fmt) + SIGN[fmt] * torch.signbit(v).long()
    c = torch.where(bad, torch.zeros_like(c), c)
    return c.reshape(x.shape), b


def check_quantized(codes, scales, fmt, x, delta):
    """Asserts that packed codes and scales are a quantisation of values within
    ``delta`` of ``x`` (float64 tensors, finite): the scale that of a largest
    magnitude within reach, each element between those of x - delta and x +
    delta at that scale."""
    g, d = x.reshape(*x.shape[:-1], -1, BLOCK), delta.reshape(*x.shape[:-1], -1, BLOCK)
    low = (g.abs() - d).clamp(min=0).amax(-1).contiguous()
    high = (g.abs() + d).amax(-1).contiguous()
    b = scales.long()
    wrong = (b < scale_bytes(low, fmt)) | (b > scale_bytes(high, fmt))
    assert not wrong.any(), f"{int(wrong.sum())} scales out of reach"
    got = decode(codes, torch.full_like(scales, 127), fmt).reshape(g.shape)
    grid = elements(fmt, x.device)

    def element(v):
        v = v * pow2(127 - b[..., None])
        return torch.copysign(grid[element_codes(v.abs(), fmt)], v)

    lo, hi = element(g - d), element(g + d)
    off = ~((got >= lo) & (got <= hi))
    assert not off.any(), f"{int(off.sum())} elements out of reach of {off.numel()}"
