"""Tensors in 4 bits and linear layers over them against 64 bits: codes bit for bit, results within what fp32 sums and one rounding can
be off by."""
import copy

import pytest
import torch

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import engine, matrix_linear, packed4

import linear_oracle as lo
import packed4_oracle as po

pytestmark = pytest.mark.gpu

# rows, C: one of everything, odd, around groups, stages and blocks of rows
PACK_SHAPES = [(1, 1), (1, 32), (3, 5), (31, 127), (32, 128), (33, 129), (64, 256), (65, 257), (7, 1000), (200, 72), (1, 8200), (513, 33)]


def _tensor(rows, C, t, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g) * torch.exp2(torch.randint(-8, 9, (rows, 1), generator=g).float())
    return x.to(t)


def _same(a, b):
    return bool((torch.isnan(a) == torch.isnan(b)).all()) and torch.equal(torch.nan_to_num(a, 0.25), torch.nan_to_num(b, 0.25))


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", PACK_SHAPES, ids=str)
def test_codes_and_values(dev, host_layer, shape, t):
    x = _tensor(*shape, t, sum(shape))
    p = packed4.pack4(x.cuda())
    codes, scales = po.pack(x)
    got = p.parts()
    assert torch.equal(got[0].cpu(), codes) and torch.equal(got[1].cpu(), scales)
    assert p.shape == x.shape and p.dtype == t
    for other in lo.TYPES:
        assert torch.equal(packed4.unpack4(p, other).cpu(), po.values(codes, scales, shape[1]).to(other))
    again = packed4.Packed4.from_parts(*got, shape[1], t)
    assert torch.equal(again.codes, p.codes) and torch.equal(again.scales, p.scales)


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
def test_borders_and_extremes(dev, t):
    """Each border between two levels, both signs, at scales over the type's whole range; zeros; infinities and NaN."""
    fi = torch.finfo(t)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    near = torch.cat([borders, borders * (1 + fi.eps), borders * (1 - fi.eps), torch.tensor([0.0, 6.0, 7.9, 4.0])])
    rows = []
    low, high = (-14, 13) if t == torch.float16 else (-126, 125)
    for k in (low + 3, -3, 0, 5, high):
        v = torch.zeros(64, dtype=torch.float64)
        v[:25] = near * 2.0 ** k
        v[32:57] = -near * 2.0 ** k
        rows.append(v)
    rows.append(torch.zeros(64, dtype=torch.float64))
    rows.append(torch.full((64,), fi.smallest_normal * fi.eps, dtype=torch.float64))      # the least number
    rows.append(torch.full((64,), fi.max, dtype=torch.float64))
    for bad in (float("inf"), float("-inf"), float("nan")):
        v = torch.ones(64, dtype=torch.float64)
        v[40] = bad
        rows.append(v)
    x = torch.stack(rows).to(t)
    p = packed4.pack4(x.cuda())
    codes, scales = po.pack(x)
    assert torch.equal(p.parts()[0].cpu(), codes) and torch.equal(p.parts()[1].cpu(), scales)
    assert _same(packed4.unpack4(p).cpu(), po.values(codes, scales, 64).to(t))


# rows, C, K: passes over w (up to 16 rows) of four, eight and sixteen rows of w a workgroup, several stages a place; tiles, whole and not, in parts; beyond them
SHAPES = [(1, 1, 1), (1, 128, 4), (1, 4096, 40), (2, 31, 65), (4, 4104, 1001), (5, 2056, 24), (8, 64, 64), (8, 136, 2100), (9, 1032, 333), (16, 520, 40), (17, 300, 128),
          (33, 257, 72), (48, 1000, 31), (64, 64, 64), (65, 33, 17), (130, 257, 96), (200, 72, 264), (257, 136, 520), (1025, 8, 8), (300, 300, 301), (600, 501, 403),
          (513, 1152, 300), (1000, 520, 776),
          (70, 1096, 700), (128, 8192, 136), (2050, 136, 72)]


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("x4", [False, True], ids=["x as it is", "x in 4 bits"])
def test_forward(dev, host_layer, shape, t, x4):
    rows, C, K = shape
    for i, (act, residual) in enumerate([("none", None), ("relu", "before"), ("gelu", "after"), ("gelu_tanh", None), ("silu", "before")]):
        g = torch.Generator().manual_seed(10 * i + rows)
        x, w = torch.randn(rows, C, generator=g).to(t), torch.randn(K, C, generator=g) * C ** -0.5
        b = torch.randn(K, generator=g).to(t) if i != 3 else None
        r = torch.randn(rows, K, generator=g).to(t) if residual else None
        wp = po.pack(w)
        W = po.values(*wp, C).to(t).double()
        w4 = packed4.Packed4.from_parts(*(v.cuda() for v in wp), C, t)
        given = packed4.pack4(x.cuda()) if x4 else x.cuda()
        X = po.values(*po.pack(x), C).to(t) if x4 else x
        y, _, by, _ = lo.forward(X, W, b, r, act, residual == "after")
        got = matrix_linear.linear_forward(given, w4, b if b is None else b.cuda(), r if r is None else r.cuda(), act, residual == "after")
        assert got.dtype == t
        lo.within(got, y, by, "%s %s" % (act, residual))


@pytest.mark.parametrize("x4", [False, True], ids=["x as it is", "x in 4 bits"])
def test_few_rows_over_a_large_weight(dev, x4):
    """More than 2^25 values, which 9 to 16 rows take on tiles; the weight's rows repeat, and so do the results."""
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(12, 8200, generator=g).bfloat16(), torch.randn(171, 8200, generator=g) * 0.01
    codes, scales = po.pack(w)
    w4 = packed4.Packed4.from_parts(codes.repeat(25, 1).cuda(), scales.repeat(25, 1).cuda(), 8200, torch.bfloat16)
    X = po.values(*po.pack(x), 8200) if x4 else x
    y, _, by, _ = lo.forward(X.bfloat16(), po.values(codes, scales, 8200), None, None, "none", False)
    got = matrix_linear.linear_forward(packed4.pack4(x.cuda()) if x4 else x.cuda(), w4)
    lo.within(got, y.repeat(1, 25), by.repeat(1, 25))


@pytest.mark.parametrize("config", [32, 33, 34])
def test_every_tile(dev, gemm_override, config):
    """The tiles that sizes choose, each at odd sizes, whole tiles, several parts."""
    gemm_override(config)
    for rows, C, K in [(300, 1000, 301), (512, 640, 512), (70, 8200, 70), (257, 128, 1000)]:
        g = torch.Generator().manual_seed(rows)
        x, w = torch.randn(rows, C, generator=g).bfloat16(), torch.randn(K, C, generator=g) * C ** -0.5
        r = torch.randn(rows, K, generator=g).bfloat16()
        X, W = po.values(*po.pack(x), C), po.values(*po.pack(w), C)
        y, _, by, _ = lo.forward(X.bfloat16(), W, None, r, "silu", True)
        w4 = packed4.pack4(w.cuda())
        lo.within(matrix_linear.linear_forward(packed4.pack4(x.cuda()), w4, None, r.cuda(), "silu", True), y, by, "%d %d %d" % (rows, C, K))


@pytest.mark.parametrize("rows", [3, 40, 100, 700])
def test_numbers_that_are_none(dev, rows):
    """A group with an infinity or a NaN makes its row of x, or its channel of w, NaN and nothing else."""
    g = torch.Generator().manual_seed(rows)
    x, w = torch.randn(rows, 300, generator=g).bfloat16(), torch.randn(70, 300, generator=g).bfloat16()
    x[1, 299], w[5, 3], w[69, 128] = float("nan"), float("inf"), float("-inf")
    bad = torch.zeros(rows, 70, dtype=torch.bool)
    bad[:, 5], bad[:, 69] = True, True
    w4 = packed4.pack4(w.cuda())
    got = matrix_linear.linear_forward(packed4.pack4(x.cuda()), w4)
    bad[1] = True
    assert torch.equal(torch.isnan(got).cpu(), bad)
    assert torch.equal(torch.isnan(matrix_linear.linear_forward(x.cuda(), w4)).cpu(), bad)


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("rows", [5, 64])
def test_infinite_inputs_stay_so(dev, rows, t):
    """x as it is: an infinity meets weights other than zero as an infinity."""
    x, w = torch.ones(rows, 64), torch.ones(24, 64)
    x[2, 7], x[3, 9] = float("inf"), float("-inf")
    got = matrix_linear.linear_forward(x.to(t).cuda(), packed4.pack4(w.cuda())).cpu().float()
    want = torch.full((rows, 24), 64.0)
    want[2], want[3] = float("inf"), float("-inf")
    assert torch.equal(got, want)


@pytest.mark.parametrize("act", lo.ACTS)
@pytest.mark.parametrize("shape", [(5, 200, 72), (130, 257, 96), (700, 1000, 520)], ids=str)
def test_gradients(dev, host_layer, act, shape):
    """x, bias and residual learn through a frozen weight."""
    rows, C, K = shape
    for t in lo.TYPES:
        g = torch.Generator().manual_seed(rows)
        x, w = torch.randn(rows, C, generator=g).to(t), torch.randn(K, C, generator=g) * C ** -0.5
        b, r, dy = torch.randn(K, generator=g).to(t), torch.randn(rows, K, generator=g).to(t), torch.randn(rows, K, generator=g).to(t)
        w4 = packed4.pack4(w.cuda())
        W = po.values(*po.pack(w), C).to(t).double()
        leaves = [v.cuda().requires_grad_() for v in (x, b, r)]
        y = matrix_linear.linear(leaves[0], w4, leaves[1], leaves[2], act)
        lo.within(y, *lo.forward(x, W, b, r, act, False)[::2][:2], "y")
        got = torch.autograd.grad(y, leaves, dy.cuda())
        # relu reads its gate from y, whose sign is z's
        z = lo.forward(x, W, b, r, act, False)[1]
        kept = matrix_linear.linear_forward(leaves[0], w4, leaves[1], leaves[2], act, keep_z=True)[1].detach().cpu()
        assert bool(((kept.double() - z).abs() <= lo.forward(x, W, b, r, act, False)[3]).all())
        want = lo.backward(dy, x, W, kept, act)
        for name, v in zip(("dx", "db", "dz"), got):
            lo.within(v, *want[name], "%s %s" % (name, act))


@pytest.mark.parametrize("act", lo.ACTS)
def test_gradient_of_x_alone(dev, host_layer, act):
    # passes over the packed weight (up to 512 rows, of fp32 all), in one part and several, and the weight widened
    for lead, C, K, t in [((1,), 96, 8, torch.float16), ((3, 2), 33, 65, torch.bfloat16), ((2, 70), 300, 129, torch.float32), ((513,), 1000, 40, torch.bfloat16),
                          ((8,), 17001, 100, torch.bfloat16), ((16,), 516, 4100, torch.float16), ((17,), 131, 517, torch.float32), ((32,), 1, 1, torch.float16),
                          ((2, 9), 129, 31, torch.bfloat16), ((4,), 520, 1024, torch.float32), ((33,), 64, 64, torch.bfloat16), ((64,), 700, 333, torch.float16), ((100,), 300, 129, torch.float32), ((128,), 520, 300, torch.float32), ((512,), 129, 96, torch.float16), ((700,), 1000, 40, torch.float16), ((1000,), 257, 65, torch.float32), ((200,), 2048, 777, torch.bfloat16), ((31,), 16500, 256, torch.float32)]:
        g = torch.Generator().manual_seed(C)
        w, dy, z = torch.randn(K, C, generator=g), torch.randn(*lead, K, generator=g).to(t), torch.randn(*lead, K, generator=g).to(t)
        w4 = packed4.pack4(w.cuda())
        W = po.values(*po.pack(w), C).to(t).double()
        want = lo.backward(dy.reshape(-1, K), torch.zeros(dy.numel() // K, C, dtype=t), W, z.reshape(-1, K), act)["dx"]
        odd = torch.empty(dy.numel() + 1, dtype=t, device=dev)[1:].view(dy.shape).copy_(dy.cuda())
        wide = torch.empty(*lead, 2 * K, dtype=t, device=dev)[..., ::2].copy_(dy.cuda())
        for given in (dy.cuda(), odd, wide):
            dx, dw, db, dz = matrix_linear.linear_backward(given, None, w4, z.cuda(), act, need_dw=False, need_db=False)
            assert dx.shape == lead + (C,) and dx.dtype == t and dx.is_contiguous() and dw is None and db is None and dz is None
            lo.within(dx.reshape(-1, C), *want, "dx")
        with pytest.raises(ValueError, match="weight|dy of shape"):
            matrix_linear.linear_backward(dy.cuda()[..., :-1].contiguous(), None, w4, z.cuda()[..., :-1].contiguous(), act, need_dw=False, need_db=False)


@pytest.mark.parametrize("act", ["none", "silu"])
def test_gradients_of_few_rows(dev, host_layer, act):
    """dx from the packed weight, and beside it the gradients of the bias and of the residual."""
    for rows, C, K, t in [(8, 260, 72, torch.float16), (20, 1000, 600, torch.bfloat16), (3, 40, 33, torch.float32)]:
        g = torch.Generator().manual_seed(K)
        w, dy, z = torch.randn(K, C, generator=g), torch.randn(rows, K, generator=g).to(t), torch.randn(rows, K, generator=g).to(t)
        w4, x = packed4.pack4(w.cuda()), torch.randn(rows, C, generator=g).to(t)
        want = lo.backward(dy, x, po.values(*po.pack(w), C).to(t).double(), z, act)
        got = matrix_linear.linear_backward(dy.cuda(), x.cuda(), w4, z.cuda(), act, need_dz=True)
        for name, v in zip(("dx", "dw", "db", "dz"), got):
            lo.within(v, *want[name], name)
        # a NaN, of dz or as a group of the weight, is a NaN of its row or group alone
        dy[1, 5] = float("nan")
        w4.scales[0, 0, 7, 0] = 255
        dx = matrix_linear.linear_backward(dy.cuda(), None, w4, z.cuda(), act, need_dw=False, need_db=False)[0].cpu()
        bad = torch.zeros(rows, C, dtype=torch.bool)
        bad[1], bad[:, :32] = True, True
        assert torch.equal(dx.isnan(), bad)


def test_strides_and_starts(dev, host_layer):
    g = torch.Generator().manual_seed(1)
    base = torch.randn(50, 203, generator=g).bfloat16().cuda()
    w4 = packed4.pack4(torch.randn(40, 100, generator=g).cuda())
    for x in (base[:, 1:101], base[::2, 100:200], base.t()[:100].t(), base[:, :100].as_strided((50, 100), (0, 1))):
        want = matrix_linear.linear_forward(x.contiguous().clone(), w4)
        assert torch.equal(matrix_linear.linear_forward(x, w4), want)
        p, q = packed4.pack4(x), packed4.pack4(x.contiguous().clone())
        assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    x = torch.randn(2, 3, 5, 100, generator=g).bfloat16().cuda()
    y = matrix_linear.linear_forward(x, w4)
    assert y.shape == (2, 3, 5, 40) and torch.equal(y.view(30, 40), matrix_linear.linear_forward(x.view(30, 100), w4))
    assert matrix_linear.linear_forward(packed4.pack4(x), w4).shape == (2, 3, 5, 40)
    none = matrix_linear.linear_forward(x[:0], w4)
    assert none.shape == (0, 3, 5, 40)
    assert matrix_linear.linear_forward(packed4.pack4(x[:0]), w4).shape == (0, 3, 5, 40)
    assert packed4.unpack4(packed4.pack4(x[:0])).shape == (0, 3, 5, 100)


def test_graph_and_stream(dev):
    """Captured and replayed beside eager work, and on another stream."""
    g = torch.Generator().manual_seed(2)
    w4 = packed4.pack4(torch.randn(520, 1000, generator=g).cuda())
    for rows in (1, 300):
        x = torch.randn(rows, 1000, generator=g).half().cuda()
        for x4 in (False, True):
            run = lambda: matrix_linear.linear_forward(packed4.pack4(x) if x4 else x, w4, activation="gelu")  # noqa: E731
            run()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = run()
            for seed in range(4):
                x.copy_(torch.randn(rows, 1000, generator=g).half())
                graph.replay()
                got, want = y.clone(), run()
                torch.cuda.synchronize()
                assert torch.equal(got, want)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                other = run()
            s.synchronize()
            assert torch.equal(other, want)


def test_same_bits_every_time(dev):
    g = torch.Generator().manual_seed(3)
    x, w4 = torch.randn(70, 8200, generator=g).bfloat16().cuda(), packed4.pack4(torch.randn(200, 8200, generator=g).cuda())
    for v in (x, packed4.pack4(x), x[:5], packed4.pack4(x[:5])):
        first = matrix_linear.linear_forward(v, w4)
        for _ in range(4):
            assert torch.equal(matrix_linear.linear_forward(v, w4), first)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("act", ["relu", "gelu"])
def test_checkpointed_layers(dev, checkpoint, act):
    """z kept in 8 bits behind a frozen weight: dx within what an unrounded z gives and 8 bits of a group's largest may change of it."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(70, 96, generator=g), torch.randn(64, 96, generator=g) * 0.1
    w4 = packed4.pack4(w.cuda())
    leaf = x.cuda().requires_grad_()
    y = matrix_linear.linear(leaf, w4, activation=act, checkpoint=checkpoint)
    dy = torch.randn(70, 64, generator=g)
    (dx,) = torch.autograd.grad(y, leaf, dy.cuda())
    W = po.values(*po.pack(w), 96)
    z = x.double() @ W.t()
    if checkpoint and act != "relu":
        # a slope moves by at most 1.13 (gelu's second derivative's largest is 0.8) of what z does, 2^-7 of its group's largest
        off = torch.full_like(z, 0.8 * 2.0 ** -7 * float(z.abs().max()))
    else:
        off = torch.full_like(z, 1e-5)
    want = (dy.double() * lo.slope(z, act)) @ W
    lo.within(dx, want, (dy.double().abs() * off) @ W.abs() + 1e-5)


def test_modules(dev):
    torch.manual_seed(6)
    for axis, shape in ((-1, (3, 5, 40)), (1, (2, 40, 6, 5))):
        layer = pkg.MatrixLinear(40, 72, activation="silu", channel_axis=axis).cuda()
        with torch.no_grad():
            layer.bias.normal_()
        x = torch.randn(shape).cuda()
        w = packed4.unpack4(packed4.pack4(layer.weight))
        want = matrix_linear.linear(x, w, layer.bias, None, "silu", channel_axis=axis)
        four = layer.pack4()
        assert torch.allclose(four(x), want, rtol=1e-5, atol=1e-5)
        assert torch.equal(four.weight.codes, packed4.pack4(layer.weight).codes)
        x4 = layer.pack4(x4=True)
        moved = x if axis == -1 else x.movedim(1, -1)
        rounded = packed4.unpack4(packed4.pack4(moved))
        want4 = matrix_linear.linear(rounded, w, layer.bias, None, "silu")
        got4 = x4(x) if axis == -1 else x4(x).movedim(1, -1)
        assert torch.allclose(got4, want4, rtol=1e-5, atol=1e-5)
        with pytest.raises(NotImplementedError, match="no gradient passes"):
            x4(x.clone().requires_grad_())
        # by the state dict into another layer, in another type
        other = pkg.MatrixLinear(40, 72, activation="silu", channel_axis=axis).cuda().pack4()
        other.load_state_dict(four.state_dict())
        assert torch.equal(other(x), four(x))
        half = copy.deepcopy(four).half()
        y = half(x.half())
        assert y.dtype == torch.float16 and torch.allclose(y.float(), want, rtol=2e-2, atol=2e-2)
        # the bias learns
        four(x).sum().backward()
        assert four.bias.grad is not None and not four.codes.is_floating_point()
    with pytest.raises(TypeError, match="Packed4"):
        pkg.MatrixLinear4(torch.randn(3, 4).cuda())


def test_beyond_32_bits(dev):
    """Codes of more than 2^31 bytes, results of more than 2^31 elements: the last rows are those of a call of their own."""
    x = torch.empty(70000, 65536, dtype=torch.float16, device="cuda")
    x[:100].normal_()
    x[-100:].normal_()
    x[100:-100] = 1
    p = packed4.pack4(x)
    assert p.codes.numel() > 1 << 31
    for part in (slice(0, 100), slice(-100, None)):
        q = packed4.pack4(x[part])
        assert torch.equal(p.codes[part], q.codes)
    last = packed4.unpack4(packed4.pack4(x[-100:]))
    del x
    back = packed4.unpack4(p)
    assert torch.equal(back[-100:], last) and bool((back[200:300] == 1).all())
    del back, p
    torch.cuda.empty_cache()
    g = torch.Generator().manual_seed(8)
    w = torch.randn(8200, 64, generator=g)
    w4, W = packed4.pack4(w.cuda()), po.values(*po.pack(w), 64)
    x = torch.randn(300000, 64, generator=g).half()
    for x4 in (False, True):
        y = matrix_linear.linear_forward(packed4.pack4(x.cuda()) if x4 else x.cuda(), w4)
        assert y.numel() > 1 << 31
        for part in (slice(0, 3), slice(-3, None)):
            X = po.values(*po.pack(x[part]), 64).half() if x4 else x[part]
            want, _, bound, _ = lo.forward(X, W, None, None, "none", False)
            lo.within(y[part], want, bound)
        del y


def test_gradients_captured_and_side_by_side(dev):
    g = torch.Generator().manual_seed(5)
    w4 = packed4.pack4(torch.randn(520, 300, generator=g).cuda())
    for rows, t in [(3, torch.float16), (40, torch.bfloat16), (70, torch.float32)]:
        z, dys = torch.randn(rows, 520, generator=g).to(t).cuda(), [torch.randn(rows, 520, generator=g).to(t).cuda() for _ in range(3)]
        grad = lambda dy: matrix_linear.linear_backward(dy, None, w4, z, "silu", need_dw=False)  # noqa: E731
        want = [grad(dy) for dy in dys]
        given = dys[0].clone()
        grad(given)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dx, _, db, _ = grad(given)
        for dy, (dx64, _, db64, _) in zip(dys + dys[:1], want + want[:1]):
            given.copy_(dy)
            graph.replay()
            other = grad(dys[1])                       # (eager work of the same shape beside the replay's results)
            assert torch.equal(dx, dx64) and torch.equal(db, db64) and torch.equal(other[0], want[1][0])
            torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in dys]
        torch.cuda.synchronize()
        got = []
        for s, dy in zip(streams, dys):
            with torch.cuda.stream(s):
                got.append([grad(dy) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) for runs, b in zip(got, want) for a in runs)


@pytest.mark.parametrize("t", lo.TYPES, ids=str)
@pytest.mark.parametrize("shape", [(3, 300, 72), (16, 520, 41), (64, 4096, 136), (200, 72, 264), (300, 1000, 77), (2050, 136, 72), (33, 257, 72)], ids=str)
def test_z_is_kept(dev, host_layer, shape, t):
    rows, C, K = shape
    for act, after in (("gelu", False), ("silu", True), ("none", False)):
        g = torch.Generator().manual_seed(rows + C)
        x, w = torch.randn(rows, C, generator=g).to(t), torch.randn(K, C, generator=g) * C ** -0.5
        b, r = torch.randn(K, generator=g).to(t), torch.randn(rows, K, generator=g).to(t)
        W = po.values(*po.pack(w), C).to(t).double()
        w4 = packed4.pack4(w.cuda())
        y, z = matrix_linear.linear_forward(x.cuda(), w4, b.cuda(), r.cuda(), act, after, keep_z=True)
        want = lo.forward(x, W, b, r, act, after)
        lo.within(y, want[0], want[2], "y " + act)
        lo.within(z, want[1], want[3], "z " + act)
        # y is that of a pass without z
        assert torch.equal(y, matrix_linear.linear_forward(x.cuda(), w4, b.cuda(), r.cuda(), act, after))
