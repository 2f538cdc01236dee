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
          (12, 8200, 4104), (70, 1096, 700), (128, 8192, 136), (2050, 136, 72)]


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
