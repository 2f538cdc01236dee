"""Linear layers, their gradients and activations in 8 bits in 64 bits, with bounds on what fp32 sums and one rounding may be off by
(test infrastructure)."""
import math

import torch

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
TYPES = (torch.float32, torch.float16, torch.bfloat16)
SUM = 2.0 ** -24        # half a step of fp32: what one addition of a sum rounds by
# activations and their derivatives by the hardware's 2^v and reciprocal (2 ulp each), a polynomial within 5e-7 and a handful of
# roundings, each 2^-24 of a value of at most 1 + |z|: 16 of them
SLOPE = 2.0 ** -20


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    """Half a step of the subnormal numbers."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        th = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * a * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def forward(x, w, b, r, name, after):
    """(y, z, bound of y, bound of z) of 2-D CPU tensors of one type."""
    t = x.dtype
    X, W = x.double(), w.double()
    z, mass = X @ W.t(), X.abs() @ W.abs().t()
    for v in (b, None if after else r):
        if v is not None:
            z, mass = z + v.double(), mass + v.double().abs()
    off = (x.shape[1] + 8) * SUM * mass
    y = act(z, name)
    # no activation is steeper than 1.13
    off_y = 1.13 * off + (SLOPE * (1 + z.abs()) if name not in ("none", "relu") else 0)
    if after and r is not None:
        y = y + r.double()
        off_y = off_y + 2 * SUM * (y.abs() + r.double().abs())
    u = half_step(t)
    return y, z, off_y * (1 + u) + u * y.abs() + least(t), off * (1 + u) + u * z.abs() + least(t)


def backward(dy, x, w, z, name, w_type=None, b_type=None):
    """{name: (value, bound)} of dx, dw, db, dz; x and z the values that the layer kept."""
    t = dy.dtype
    u = half_step(t) if name != "none" else 0.0             # dz is rounded before the products
    DY, X, W = dy.double(), x.double(), w.double()
    dz = DY * slope(z.double(), name) if name != "none" else DY
    off = SLOPE * DY.abs() * (1 + z.double().abs()) if name not in ("none", "relu") else torch.zeros_like(DY)
    off_r = off * (1 + u) + u * dz.abs() + (least(t) if name != "none" else 0)
    out = {"dz": (dz, off_r)}

    def rounded(v, bound, t):
        return v, bound * (1 + half_step(t)) + half_step(t) * v.abs() + least(t)
    K, rows = W.shape[0], DY.shape[0]
    out["dx"] = rounded(dz @ W, off_r @ W.abs() + (K + 8) * SUM * (dz.abs() @ W.abs()), t)
    out["dw"] = rounded(dz.t() @ X, off_r.t() @ X.abs() + (rows + 8) * SUM * (dz.abs().t() @ X.abs()), w_type or t)
    out["db"] = rounded(dz.sum(0), off.sum(0) + (rows + 8) * SUM * dz.abs().sum(0), b_type or t)
    return out


def within(got, want, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), "%s: %g over a bound of %g at %r" % (what, float(over.max()), float(bound.flatten()[over.argmax()]), int(over.argmax()))


def pack(x, keep_sign=False):
    """(codes, exponents) of a CPU tensor (rows, C), group by group in 64 bits."""
    rows, C = x.shape
    codes, exps = torch.zeros(rows, C, dtype=torch.int8), torch.zeros(rows, (C + 31) // 32, dtype=torch.int8)
    for g in range(exps.shape[1]):
        v = x[:, 32 * g:32 * g + 32].double()
        top = v.abs().amax(1)
        bad = ~torch.isfinite(v).all(1)
        e = torch.where((top > 0) & ~bad, torch.frexp(torch.where(bad, torch.zeros_like(top), top)).exponent - 7, torch.tensor(-126)).clamp(min=-126)
        q = torch.ldexp(torch.where(bad[:, None], torch.zeros_like(v), v), -e[:, None]).round().clamp(-127, 127)
        if keep_sign:
            q = torch.where((q == 0) & (v != 0) & ~bad[:, None], v.sign(), q)
        codes[:, 32 * g:32 * g + 32] = q.to(torch.int8)
        exps[:, g] = torch.where(bad, torch.tensor(127), e).to(torch.int8)
    return codes, exps


def unpack(codes, exps):
    """The values in 64 bits."""
    e = exps.to(torch.int64).repeat_interleave(32, dim=1)[:, :codes.shape[1]]
    return torch.where(e == 127, torch.tensor(math.nan, dtype=torch.float64), torch.ldexp(codes.double(), e))
