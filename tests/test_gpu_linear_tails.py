"""Activations and their slopes where they are small: relative to the value, down to what fp32 holds, against 64 bits.

A layer of one channel with a weight of one, so that z is the input to the last bit.  e: half a step of fp32, 2^-24.  2^v and 1 / v are off by at
most 4 e (2 ulp), every other operation and constant by e.
  e^-u, u off by n e: (n + 2) u e for u and the product with log2(e) and its constant, and 4 e
  gelu: u = z^2 / 2 by the square of |z| / sqrt 2 (a product and a constant, twice; the square): n = 5; the polynomial 5e-7, a dozen operations with it
  gelu by tanh: u = k (z + c z^3): three products, a sum, a product, two constants: n = 7; silu: n = 0
  logistic function g = 1 / (1 + e^-u): what e^-u is off by counts by its share 1 - g; the sum e, 1 / v 4 e
The hardware's 2^v and 1 / v may give 0 for what is below the smallest normal number, 2^-126: of the density, and of g, which then is missing in every
place it has in the formula - |z| g in the value, g + g |q| in the slope, |q| up to 390 at z = -12."""
import math

import pytest
import torch

from pytorch_winoconv_amd import matrix_linear

import linear_oracle as lo

pytestmark = pytest.mark.gpu

e = lo.SUM
LEAST = 2.0 ** -126
K, C3 = 2 * math.sqrt(2 / math.pi), 0.044715


def _logistic(u, n):
    """(g, what it is off by)"""
    g = torch.sigmoid(u)
    return g, g * ((1 - g) * ((n + 2) * u.abs() + 4) * e + 6 * e)


def _normal(z):
    """(density, what it is off by, distribution, what it is off by)"""
    off = (7 * z * z / 2 + 4) * e
    d = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    # (torch.special.ndtr has no digits left below z = -8)
    below, tail = (0.5 * torch.special.erfc(v / math.sqrt(2)) for v in (-z, z.abs()))
    return d, d * off, below, tail * (off + 5e-7 + 12 * e) + torch.where(z < 0, 0, e)


def _value(z, act):
    if act == "gelu":
        _, _, g, off = _normal(z)
    else:
        g, off = _logistic(K * (z + C3 * z ** 3), 7) if act == "gelu_tanh" else _logistic(z, 0)
    return z * g, z.abs() * (off + 2 * e * g + LEAST)


def _slope(z, act):
    if act == "gelu":
        d, off_d, g, off = _normal(z)
        return g + z * d, off + z.abs() * (off_d + 4 * e * d) + (1 + z.abs()) * LEAST
    g, off = _logistic(K * (z + C3 * z ** 3), 7) if act == "gelu_tanh" else _logistic(z, 0)
    # h q, h = g (1 - g): 1 - g is off by what g is and its rounding; q by seven operations and constants
    q = K * z * (1 + 3 * C3 * z * z) if act == "gelu_tanh" else z
    h = g * (1 - g)
    return g + h * q, off + q.abs() * (off * (1 - g) + g * (off + e) + 9 * e * h) + (1 + q.abs()) * LEAST


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_small_values(dev, act, t):
    x = torch.linspace(-12, 12, 4801).to(t)[:, None]
    z, u = x.double()[:, 0], lo.half_step(t)
    y = matrix_linear.linear_forward(x.cuda(), torch.ones(1, 1, dtype=t, device=dev), activation=act)[:, 0]
    dz = matrix_linear.linear_backward(torch.ones_like(x, device=dev), None, None, x.cuda(), act, need_dx=False, need_dw=False, need_db=False, need_dz=True)[3][:, 0]
    for got, (want, off), what in ((y, _value(z, act), "y"), (dz, _slope(z, act), "slope")):
        lo.within(got, want, off + 2 * u * want.abs(), what)
