"""Tensors in 4 bits (e2m1 values, a power of two a group of 32) in 64 bits, value by value (test infrastructure)."""
import math

import torch

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pack(x):
    """(codes, scales) of a CPU tensor (rows, C) in plain order, two codes to a byte: the nearest level, of two as near the even code."""
    rows, C = x.shape
    groups = -(-C // 32)
    v = torch.zeros(rows, groups * 32, dtype=torch.float64)
    v[:, :C] = x.double()
    v = v.view(rows, groups, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad[..., None], torch.zeros_like(v), v)
    top = v.abs().amax(-1)
    # (frexp: top = m 2^k with m from 0.5 to 1, so floor(log2(top)) = k - 1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.tensor(-127)).clamp(min=-127)
    share = torch.ldexp(v.abs(), -e[..., None])
    far = (share[..., None] - torch.tensor(LEVELS, dtype=torch.float64)).abs()
    far = torch.where(torch.arange(8) % 2 == 1, far * (1 + 1e-12) + 1e-300, far)      # ties to the even code
    code = far.argmin(-1) | torch.where(torch.signbit(v), 8, 0)
    code = torch.where(bad[..., None], torch.zeros_like(code), code).view(rows, groups * 32)
    code[:, C:] = 0
    codes = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)[:, :(C + 1) // 2]
    return codes, torch.where(bad, torch.tensor(255), e + 127).to(torch.uint8)


def values(codes, scales, C):
    """The values in 64 bits."""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(1)[:, :C]
    e = scales.long().repeat_interleave(32, dim=1)[:, :C]
    return torch.where(e == 255, torch.tensor(math.nan, dtype=torch.float64), torch.ldexp(v, e - 127))
