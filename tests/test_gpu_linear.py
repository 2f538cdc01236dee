"""Linear layers with an epilogue and their gradients against 64 bits, element by element, within what fp32 sums and the roundings of the
types can be off by."""
import pytest
import torch

from pytorch_winoconv_amd import checkpoint8, matrix_linear

import linear_oracle as lo

pytestmark = pytest.mark.gpu

# rows, C, K: one of everything, odd, around tiles and stages, long reductions, few and many rows
SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 31, 65), (8, 64, 64), (16, 512, 40), (33, 40, 72), (64, 64, 64), (65, 33, 17), (130, 257, 96), (200, 72, 264), (7, 1000, 3),
          (513, 16, 300), (257, 136, 520), (1, 4096, 24), (5, 2056, 1000), (17, 3000, 128), (1025, 8, 8), (300, 300, 301), (1000, 520, 776),
          (2000, 96, 640), (600, 501, 403), (600, 504, 403), (600, 501, 408), (4, 4104, 1001), (6, 136, 50), (9, 1032, 333), (16, 8, 17)]


def _inputs(rows, C, K, t, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g).to(t)
    w = (torch.randn(K, C, generator=g) * C ** -0.5).to(t)
    b = torch.randn(K, generator=g).to(t) if bias else None
    r = torch.randn(rows, K, generator=g).to(t)
    dy = torch.randn(rows, K, generator=g).to(t)
    return x, w, b, r, dy


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(dev, shape, t):
    for i, (act, residual, keep) in enumerate([("none", None, False), ("relu", "before", False), ("gelu", "after", True), ("gelu_tanh", None, True), ("silu", "before", True)]):
        x, w, b, r, _ = _inputs(*shape, t, 10 * i + shape[0], bias=i != 3)
        r = r if residual else None
        y, z, by, bz = lo.forward(x, w, b, r, act, residual == "after")
        got = matrix_linear.linear_forward(*_cuda(x, w, b, r), act, residual == "after", keep)
        if keep:
            lo.within(got[1], z, bz, "z " + act)
        got = got[0] if keep else got
        assert got.dtype == t
        lo.within(got, y, by, "y " + act)


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(dev, shape, t):
    for i, act in enumerate(lo.ACTS):
        x, w, b, r, dy = _inputs(*shape, t, 100 * i + shape[1])
        z = lo.forward(x, w, b, r, act, False)[1].to(t)
        wide = t if i % 2 else torch.float32
        want = lo.backward(dy, x, w, z, act, wide, wide)
        X, W, DY, Z = _cuda(x, w, dy, z)
        got = dict(zip(("dx", "dw", "db", "dz"), matrix_linear.linear_backward(DY, X, W, Z, act, need_dz=True, w_type=wide, b_type=wide)))
        assert got["dw"].dtype == wide and got["db"].dtype == wide and got["dx"].dtype == t
        for k, v in got.items():
            lo.within(v, *want[k], "%s %s" % (k, act))
        # one at a time: the same bits
        for k in got:
            need = {"need_" + n: n == k for n in got}
            one = matrix_linear.linear_backward(DY, X, W, Z, act, w_type=wide, b_type=wide, **need)
            assert [v is not None for v in one] == [n == k for n in got]
            assert torch.equal(dict(zip(got, one))[k], got[k])


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", [(3, 5, 7), (8, 64, 64), (33, 40, 72), (65, 33, 17), (200, 72, 264), (1000, 136, 96), (300, 300, 301), (1, 4096, 24), (600, 501, 403), (600, 504, 408)], ids=str)
def test_gradients_from_8_bits(dev, shape, t):
    for i, act in enumerate(lo.ACTS):
        x, w, b, r, dy = _inputs(*shape, t, 7 * i + shape[2])
        z = lo.forward(x, w, b, r, act, False)[1].to(t)
        px, pz = lo.pack(x), lo.pack(z, act == "relu")
        xv, zv = lo.unpack(*px), lo.unpack(*pz)
        if act == "relu":
            assert torch.equal(zv > 0, z.double() > 0)
        want = lo.backward(dy, xv, w, zv, act)
        P = [checkpoint8.Packed8(c.cuda(), e.cuda(), t) for c, e in (px, pz)]
        got = matrix_linear.linear_backward(dy.cuda(), P[0], w.cuda(), P[1], act, need_dz=True)
        for k, v in zip(("dx", "dw", "db", "dz"), got):
            lo.within(v, *want[k], "%s %s" % (k, act))


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("config", [31, 32, 33, 34])
def test_every_tile(dev, gemm_override, config, t):
    """Each kernel and tile on small ragged problems: one part of the reduction and several, one row of tiles and some."""
    gemm_override(config)
    for shape in [(1, 8, 8), (70, 40, 72), (300, 264, 328), (130, 1160, 264), (520, 72, 517), (65, 2000, 24)]:
        for act, keep in (("none", False), ("gelu", True), ("relu", False)):
            x, w, b, r, dy = _inputs(*shape, t, config)
            y, z, by, bz = lo.forward(x, w, b, r, act, keep)
            got = matrix_linear.linear_forward(*_cuda(x, w, b, r), act, keep, keep)
            if keep:
                lo.within(got[1], z, bz, "z %r" % (shape,))
            lo.within(got[0] if keep else got, y, by, "y %r" % (shape,))
            z = z.to(t)
            want = lo.backward(dy, x, w, z, act)
            for k, v in zip(("dx", "dw", "db", "dz"), matrix_linear.linear_backward(*_cuda(dy, x, w, z), act, need_dz=True)):
                lo.within(v, *want[k], "%s %r" % (k, shape))


@pytest.mark.parametrize("t", lo.TYPES[1:], ids=str)
@pytest.mark.parametrize("deep", [8, 40, 64, 96, 136])
def test_many_results(dev, t, deep):
    """Products of so many results that they take the largest tiles, the last of them ragged, over few to some stages of the reduction."""
    x, w, b, r, _ = _inputs(4090, deep, 4104, t, deep)
    y, z, by, bz = lo.forward(x, w, b, r, "gelu", True)
    got = matrix_linear.linear_forward(*_cuda(x, w, b, r), "gelu", True, True)
    lo.within(got[0], y, by, "y")
    lo.within(got[1], z, bz, "z")
    x, w, _, _, dy = _inputs(4106, 4104, deep, t, deep)
    dx = matrix_linear.linear_backward(dy.cuda(), None, w.cuda(), need_dw=False, need_db=False)[0]
    DY, W = dy.double(), w.double()
    lo.within(dx, DY @ W, lo.half_step(t) * (DY @ W).abs() + 2 * (deep + 8) * lo.SUM * (DY.abs() @ W.abs()) + lo.least(t), "dx")
    x, _, _, _, dy = _inputs(deep + 3, 4096, 4112, t, deep)
    X, DY = x.double(), dy.double()
    for wide in (t, torch.float32):
        dw = matrix_linear.linear_backward(dy.cuda(), x.cuda(), None, need_dx=False, need_db=False, w_type=wide)[1]
        lo.within(dw, DY.t() @ X, lo.half_step(wide) * (DY.t() @ X).abs() + 2 * (deep + 11) * lo.SUM * (DY.abs().t() @ X.abs()) + lo.least(wide), "dw")


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
def test_values_without_a_limit(dev, t):
    """Infinities and NaN: what a formula's limit is, and only where they stand."""
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([-inf, inf, nan, 0.0, -0.0, 30.0, -30.0, 6e4, -6e4], dtype=t)
    one = torch.ones(1, 1, dtype=t)
    for act in lo.ACTS:
        y = matrix_linear.linear_forward(z[:, None].cuda(), one.cuda(), activation=act)[:, 0].cpu().double()
        low = 0.0 if act != "none" else -inf
        assert y[0] == low and y[1] == inf and torch.isnan(y[2]) and y[3] == 0 and y[4] == 0
        assert y[5] == 30 and y[7] == z[7].double()
        if act != "none":
            assert abs(y[6]) < 1e-10 and y[8] == 0
            # slopes
            dz = matrix_linear.linear_backward(torch.ones(9, 1, dtype=t, device=dev), None, None, z[:, None].cuda(), act, need_dx=False, need_dw=False, need_db=False,
                                               need_dz=True)[3][:, 0].cpu().double()
            at0 = 0.0 if act == "relu" else 0.5
            assert dz[0] == 0 and dz[1] == 1 and torch.isnan(dz[2]) and dz[3] == at0 and dz[4] == at0 and dz[5] == 1 and abs(dz[6]) < 1e-10 and dz[7] == 1 and dz[8] == 0
    # a NaN in one row stays in its row and, in the parameters' gradients, in its channels
    x, w, b, _, dy = _inputs(70, 40, 72, t, 3)
    x[11, 5] = nan
    y = matrix_linear.linear_forward(*_cuda(x, w, b), activation="relu")
    assert torch.isnan(y[11]).all() and torch.isfinite(y[:11]).all() and torch.isfinite(y[12:]).all()
    dx, dw, db, _ = matrix_linear.linear_backward(*_cuda(dy, x, w))
    assert torch.isfinite(dx).all() and torch.isfinite(db).all() and torch.isnan(dw[:, 5]).all() and torch.isfinite(dw[:, :5]).all() and torch.isfinite(dw[:, 6:]).all()


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
def test_strides_starts_and_axes(dev, t):
    """Views that are not contiguous or start anywhere give what their copies give, and nothing beside an output is written."""
    x, w, b, r, dy = _cuda(*_inputs(96, 64, 80, t, 8))
    y = matrix_linear.linear_forward(x, w, b, r, "silu")
    wide = torch.randn(96, 130, device=dev).to(t)
    wide[:, 3:67] = x
    assert torch.equal(matrix_linear.linear_forward(wide[:, 3:67], w, b, r, "silu"), y)
    assert torch.equal(matrix_linear.linear_forward(x, w.t().contiguous().t(), b, r, "silu"), y)
    flat = torch.zeros(96 * 64 + 1, device=dev, dtype=t)
    flat[1:] = x.flatten()
    off = torch.zeros(80 * 64 + 3, device=dev, dtype=t)
    off[3:] = w.flatten()
    X, W = flat[1:].view(96, 64), off[3:].view(80, 64)
    by = lo.forward(*(None if v is None else v.cpu() for v in (x, w, b, r)), "silu", False)
    lo.within(matrix_linear.linear_forward(X, W, b, r, "silu"), by[0], by[2])
    assert torch.equal(matrix_linear.linear_forward(x.view(4, 24, 64), w, b, r.view(4, 24, 80), "silu").view(96, 80), y)
    # (N, C, H, W) of the convolutions
    img = x.view(2, 6, 8, 64).permute(0, 3, 1, 2)
    out = matrix_linear.linear(img, w, b, r.view(2, 6, 8, 80).permute(0, 3, 1, 2), "silu", channel_axis=1)
    assert out.shape == (2, 80, 6, 8) and out.is_contiguous(memory_format=torch.channels_last) and torch.equal(out.permute(0, 2, 3, 1).reshape(96, 80), y)
    want = matrix_linear.linear_backward(dy, x, w)
    for a, c in zip(matrix_linear.linear_backward(dy, wide[:, 3:67], w)[:3], want):
        assert torch.equal(a, c)
    expanded = torch.ones(1, device=dev, dtype=t).expand(96, 80)
    for a, c in zip(matrix_linear.linear_backward(expanded, x, w)[:3], matrix_linear.linear_backward(expanded.contiguous(), x, w)):
        assert torch.equal(a, c)
    full = lo.backward(dy.cpu(), x.cpu(), w.cpu(), x.cpu(), "none")
    for a, k in zip(matrix_linear.linear_backward(dy, X, W), ("dx", "dw", "db")):
        lo.within(a, *full[k], k)


def test_offsets_beyond_32_bits(dev):
    """More than 2^31 elements of x, and of its codes: rows at the very end, forward, both gradients and 8 bits."""
    t, C, K, rows = torch.float16, 64, 8, (1 << 25) + 1000
    x = torch.zeros(rows, C, dtype=t, device=dev)
    dy = torch.zeros(rows, K, dtype=t, device=dev)
    tail = slice(rows - 700, rows)
    xs, w, _, _, ds = _inputs(700, C, K, t, 3)
    x[tail], dy[tail] = xs.cuda(), ds.cuda()
    y, _, by, _ = lo.forward(xs, w, None, None, "relu", False)
    got = matrix_linear.linear_forward(x, w.cuda(), activation="relu")
    lo.within(got[tail], y, by, "y")
    assert not bool(got[:4096].any())
    del got
    p = checkpoint8.pack8(x)
    codes, exps = lo.pack(xs)
    assert torch.equal(p.codes[tail].cpu(), codes) and torch.equal(p.exponents[tail].cpu(), exps)
    back = checkpoint8.unpack8(p)
    assert torch.equal(back[tail].cpu().double(), lo.unpack(codes, exps)) and not bool(back[:4096].any())
    del p, back
    dx, dw, db, _ = matrix_linear.linear_backward(dy, x, w.cuda())
    want = lo.backward(ds, xs, w, xs, "none")
    lo.within(dx[tail], *want["dx"], "dx")
    # (zeros add no roundings but those of the sums of parts)
    lo.within(dw, *want["dw"], "dw")
    lo.within(db, *want["db"], "db")


def test_no_rows(dev, host_layer):
    w = torch.randn(5, 4, device=dev)
    for lead in ((0,), (3, 0)):
        x = torch.zeros(*lead, 4, device=dev)
        assert matrix_linear.linear_forward(x, w).shape == lead + (5,)
        dx, dw, db, dz = matrix_linear.linear_backward(torch.zeros(*lead, 5, device=dev), x, w, need_dz=True)
        assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros(5, device=dev)) and dz.shape == lead + (5,)
        p = checkpoint8.pack8(x)
        assert checkpoint8.unpack8(p).shape == x.shape


def test_both_host_layers_agree(dev, monkeypatch):
    from pytorch_winoconv_amd import engine
    x, w, b, r, dy = _cuda(*_inputs(77, 48, 56, torch.float16, 4))
    out = []
    for ext in (True, False):
        monkeypatch.setattr(engine, "USE_EXT", ext)
        y, z = matrix_linear.linear_forward(x, w, b, r, "gelu", keep_z=True)
        p = checkpoint8.pack8(x)
        out.append([y, z, p.codes, p.exponents, checkpoint8.unpack8(p), *matrix_linear.linear_backward(dy, p, w, z, "gelu", need_dz=True, w_type=torch.float32)])
    for a, c in zip(*out):
        assert a.dtype == c.dtype and torch.equal(a, c)


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (49, 77), (64, 256), (7, 1000), (1000, 8), (2, 4096), (333, 96)], ids=str)
def test_8_bits_are_exact(dev, shape, t):
    g = torch.Generator().manual_seed(shape[1])
    x = torch.randn(shape, generator=g) * torch.exp(6 * torch.randn(shape[0], 1, generator=g))
    x[torch.rand(shape, generator=g) < 0.2] = 0
    x = x.to(t)
    x.view(-1)[::7] = x.view(-1)[::7].clamp(-1, 1) * torch.finfo(t).smallest_normal
    for keep in (False, True):
        codes, exps = lo.pack(x, keep)
        p = checkpoint8.pack8(x.cuda(), keep)
        assert torch.equal(p.exponents.cpu(), exps) and torch.equal(p.codes.cpu(), codes)
        assert torch.equal(checkpoint8.unpack8(p).cpu().double().nan_to_num(), lo.unpack(codes, exps).nan_to_num())
        assert checkpoint8.unpack8(p).dtype == t
    lead = x.cuda().view(1, *shape)
    assert checkpoint8.pack8(lead).exponents.shape == (1, shape[0], (shape[1] + 31) // 32)


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
def test_8_bits_at_the_ends_of_the_types(dev, t):
    f = torch.finfo(t)
    least = f.smallest_normal * f.eps
    x = torch.zeros(12, 40, dtype=t)
    x[0, 0], x[0, 1] = f.max, -f.max
    x[1, 3] = least
    x[2, 5], x[2, 6] = float("inf"), 1
    x[3, 7], x[3, 39] = float("nan"), 2
    x[4, 0], x[4, 1], x[4, 2], x[4, 3] = 64, 0.5, 1.5, -2.5          # ties, to even
    x[5, 0], x[5, 1] = 127.75 if t == torch.float32 else 127.5, -127.5
    x[6, 30:34] = torch.tensor([1.0, -1.0, 1e-4, -1e-4])
    x[7] = f.smallest_normal
    for keep in (False, True):
        codes, exps = lo.pack(x, keep)
        p = checkpoint8.pack8(x.cuda(), keep)
        assert torch.equal(p.exponents.cpu(), exps) and torch.equal(p.codes.cpu(), codes)
        back = checkpoint8.unpack8(p).cpu()
        assert torch.isnan(back[2, :32]).all() and torch.isfinite(back[2, 32:]).all() and torch.isnan(back[3, :32]).all() and back[3, 39] == 2
        assert torch.isfinite(back[0]).all() and torch.equal(back[:2].double(), lo.unpack(codes, exps)[:2])
