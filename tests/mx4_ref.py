"""Microscaled 4-bit floating point in 64 bits on the CPU, from the definition: 32 values of a row share a scale
2^(byte - 127), a code is a sign and one of GRID; byte 255 is no number."""
import math

import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
MOST = {torch.float16: 13, torch.bfloat16: 125, torch.float32: 125}  # largest exponent of a scale that the type takes


def quantize(x, most=125):
    """(codes, scales) of x [..., n] as float64: the nearest value, of two as near the one with an even code."""
    y = x.double().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1)
    fine = torch.isfinite(top) & ~torch.isnan(y).any(-1)
    safe = torch.where(fine & (top > 0), top, torch.ones_like(top))
    e = torch.where(fine & (top > 0), torch.frexp(safe)[1].long() - 1 - 2, torch.full_like(top, -127).long())
    e = e.clamp(-127, most)
    t = torch.where(fine[..., None], y, torch.zeros_like(y)) * torch.pow(2.0, -e.double())[..., None]
    off = (t.abs()[..., None] - GRID).abs()
    best = off.amin(-1, keepdim=True)
    odd = torch.arange(8) % 2
    code = (off + torch.where(off == best, 0.0, math.inf) + odd * 1e-300).argmin(-1)  # ties: adding 1e-300 is lost where off > 0
    tie = (off == best).sum(-1) > 1
    both = torch.where(off == best, torch.arange(8), 99).amin(-1)  # the lower of two
    code = torch.where(tie, torch.where(both % 2 == 0, both, both + 1), code)
    code = code + 8 * torch.signbit(t).long()
    code = torch.where(fine[..., None], code, torch.zeros_like(code)).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(fine, e + 127, 255).to(torch.uint8)


def values(codes, scales, dtype=None):
    """float64 values; with a dtype those that it has of them (rounded; past it infinite)."""
    grid = torch.cat([GRID, -GRID])
    v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2).unflatten(-1, (-1, 32))
    v = v * torch.where(scales == 255, math.nan, torch.pow(2.0, scales.double() - 127))[..., None]
    v = v.flatten(-2)
    return v if dtype is None else v.to(dtype).double()


def cached(codes, scales, dtype):
    """What attention takes of a cache in that type: blocks whose scale passes it are no numbers."""
    return values(codes, torch.where(scales.long() - 127 > MOST[dtype], 255, scales.long()).to(torch.uint8), dtype)
