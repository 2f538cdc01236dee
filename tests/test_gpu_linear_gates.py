"""relu's gate from z in 8 bits is z's own: beside infinities and NaN too, whose group of 32 channels has no step."""
import pytest
import torch

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import checkpoint8

import linear_oracle as lo

pytestmark = pytest.mark.gpu

inf, nan = float("inf"), float("nan")


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("K", [96, 77])
@pytest.mark.parametrize("after", [False, True])
@pytest.mark.parametrize("third", [inf, nan])
def test_gates_beside_infinities(dev, host_layer, t, K, after, third):
    torch.manual_seed(K)
    x, r, dy = (torch.randn(40, n, device=dev).to(t) for n in (24, K, K))
    layers = [pkg.MatrixLinear(24, K, activation="relu", residual_after=after, checkpoint=c).to(dev, t) for c in (None, "int8")]
    layers[1].load_state_dict(layers[0].state_dict())
    grads = []
    for layer in layers:
        with torch.no_grad():
            layer.bias[5], layer.bias[40], layer.bias[70] = inf, -inf, third
        X, R = x.clone().requires_grad_(), r.clone().requires_grad_()
        y = layer(X, R)
        assert bool(torch.isinf(y[:, 5]).all()) and bool((torch.isnan if third != third else torch.isinf)(y[:, 70]).all())
        y.backward(dy)
        grads.append((X.grad, R.grad, layer.bias.grad))
    for a, b in zip(*grads):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))
    dx, _, db = grads[1]
    assert bool(torch.isnan(dx).all()) == bool(torch.isnan(db[70])) == (third != third)
    assert third != third or bool(torch.isfinite(dx).all())
    assert bool(torch.isfinite(db[:70]).all()) and bool(torch.isfinite(db[71:]).all())
    assert float(db[5]) != 0 and float(db[40]) == 0


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("K", [64, 50])
def test_codes_of_gates(dev, host_layer, t, K):
    """As with keep_sign where all are numbers; signs, with -1 for zero, beside one that is not, and such a group reads as NaN."""
    z = torch.randn(33, K, generator=torch.Generator().manual_seed(K)).to(t)
    z[:, 3], z[4] = 0, 1e-3
    p, q = checkpoint8.pack_gates(z.to(dev)), checkpoint8.pack8(z.to(dev), True)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.exponents, q.exponents)
    z[7, 1], z[8, 2], z[9, 40] = inf, -inf, nan
    p, q = checkpoint8.pack_gates(z.to(dev)), checkpoint8.pack8(z.to(dev), True)
    assert torch.equal(p.exponents, q.exponents)
    codes = lo.pack(z, True)[0]
    for row, group in ((7, slice(0, 32)), (8, slice(0, 32)), (9, slice(32, K))):
        v = z[row, group].double()
        codes[row, group] = torch.where(v > 0, 1, torch.where(v <= 0, -1, 0)).to(torch.int8)
        assert bool(torch.isnan(checkpoint8.unpack8(p)[row, group]).all())
    assert torch.equal(p.codes.cpu(), codes)
