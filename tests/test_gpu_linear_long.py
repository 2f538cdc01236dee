"""Linear layers and 8 bits of more rows than one launch has threads for (fewer than 2^32 along an axis): what is computed at the start, around
the ends of launches and at the very end, and zeros between."""
import pytest
import torch

from pytorch_winoconv_amd import checkpoint8, matrix_linear

import linear_oracle as lo

pytestmark = pytest.mark.gpu

T = torch.float16


def _places(rows):
    """Stretches of 300 rows: at either end, and around the powers of two where launches end (32 or 64 rows a workgroup)."""
    return [slice(a, a + 300) for a in [0] + [(1 << p) - k for p in (28, 29, 30) for k in (600, 150) if (1 << p) + 300 < rows] + [rows - 300]]


def _rows(rows, n, seed, places):
    """(on the GPU, zeros but for the places; those on the CPU)"""
    t = torch.zeros(rows, n, dtype=T, device="cuda")
    parts = []
    for i, s in enumerate(places):
        parts.append(torch.randn(300, n, generator=torch.Generator().manual_seed(seed + i)).to(T))
        t[s] = parts[-1].cuda()
    return t, parts


def test_forward(dev):
    rows = (1 << 30) + 70
    places = _places(rows)
    x, xs = _rows(rows, 1, 1, places)
    r, rs = _rows(rows, 1, 50, places)
    w, b = torch.tensor([[0.7]], dtype=T), torch.tensor([0.3], dtype=T)
    y, z = matrix_linear.linear_forward(x, w.cuda(), b.cuda(), r, "silu", True, True)
    for s, xp, rp in zip(places, xs, rs):
        want_y, want_z, by, bz = lo.forward(xp, w, b, rp, "silu", True)
        lo.within(z[s], want_z, bz, "z at %d" % s.start)
        lo.within(y[s], want_y, by, "y at %d" % s.start)
    # every other row is that of x = r = 0
    y0, z0, by, bz = (v.item() for v in lo.forward(torch.zeros(1, 1, dtype=T), w, b, torch.zeros(1, 1, dtype=T), "silu", True))
    for a, v, bound in ((y, y0, by), (z, z0, bz)):
        for s in places:
            a[s] = v
        low, high = a.aminmax()
        assert v - bound - lo.half_step(T) <= float(low) <= float(high) <= v + bound + lo.half_step(T)


def test_8_bits_and_their_gradients(dev):
    rows, C = (1 << 29) + 70, 3
    places = _places(rows)
    x, xs = _rows(rows, C, 3, places)
    packed = checkpoint8.pack8(x)
    del x
    kept = [lo.pack(xp) for xp in xs]
    for s, (codes, exps) in zip(places, kept):
        assert torch.equal(packed.codes[s].cpu(), codes) and torch.equal(packed.exponents[s].cpu(), exps)
    back = checkpoint8.unpack8(packed)
    for s, k in zip(places, kept):
        assert torch.equal(back[s].cpu().double(), lo.unpack(*k))
        back[s] = 0
    assert not bool(back.any())
    del back
    dy, ds = _rows(rows, 1, 90, places)
    w = torch.randn(1, C, generator=torch.Generator().manual_seed(7)).to(T)
    dx, dw, db, _ = matrix_linear.linear_backward(dy, packed, w.cuda())
    # (zeros add no roundings but those of the sums of parts; places overlap nowhere)
    want = lo.backward(torch.cat(ds), torch.cat([lo.unpack(*k) for k in kept]), w, None, "none")
    lo.within(dw, *want["dw"], "dw")
    lo.within(db, *want["db"], "db")
    lo.within(torch.cat([dx[s] for s in places]), *want["dx"], "dx")
    for s in places:
        dx[s] = 0
    assert not bool(dx.any())
