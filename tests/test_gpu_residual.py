"""Joins of blocks to their stream, norms and dropout against 64 bits, value by value, forward and backward."""
import pytest
import torch

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import residual
from pytorch_winoconv_amd.residual import Drop, Norm

import residual_oracle as ro

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
# samples, rows of each, channels: one of everything, odd, around a thread's eight channels, a wavefront's and a workgroup's, rows beyond registers
SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 5), (1, 7, 9), (3, 11, 64), (2, 100, 63), (5, 1, 513), (3, 4, 1000), (2, 3, 1024), (1, 5, 1032), (2, 2, 2056), (3, 1, 4097), (1, 3, 8192),
          (2, 2, 8200), (1, 2, 16387), (1, 2, 33000), (300, 1, 40), (700, 2, 24), (4, 600, 72), (1, 1100, 640), (2, 700, 1500)]


def _inputs(shape, t, seed, post, pre, gate, stream=True, wide=False):
    g = torch.Generator().manual_seed(seed)
    n, per, C = shape
    own = torch.float32 if wide else t
    normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    norm = lambda kind: None if kind == "none" else (kind, (1 + 0.3 * normal(C)).to(own), (0.3 * normal(C)).to(own) if kind == "layer" else None, 1e-5)  # noqa: E731
    f, x = (normal(*shape) + 0.3).to(t), normal(*shape).to(t) if stream else None
    gt = {"none": None, "channel": lambda: normal(C).to(own), "sample": lambda: normal(n, C).to(own)}[gate]
    return f, x, norm(post), norm(pre), gt and gt(), normal(*shape).to(t), normal(*shape).to(t)


def _cuda(v):
    if isinstance(v, torch.Tensor):
        return v.cuda()
    return None if v is None else Norm(v[0], _cuda(v[1]), _cuda(v[2]), v[3])


# post, pre, gate, drop, per, stream
FORMS = [("none", "none", "none", 0.3, "element", False), ("none", "none", "none", 0.0, "element", True), ("none", "layer", "none", 0.0, "element", True),
         ("rms", "rms", "channel", 0.1, "element", True), ("layer", "layer", "sample", 0.4, "sample", True), ("layer", "none", "channel", 0.0, "element", True),
         ("rms", "none", "none", 0.2, "element", False), ("none", "rms", "sample", 0.5, "element", True), ("none", "none", "sample", 0.25, "sample", False)]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_join(dev, shape, t):
    for i, (post, pre, gate, p, per, stream) in enumerate(FORMS):
        what = " ".join(str(v) for v in FORMS[i])
        f, x, po, pr, gt, ds, dy = _inputs(shape, t, i + sum(shape), post, pre, gate, stream, wide=i % 2 == 1)
        seed, offset = 0x9876543210FEDCBA + i, (1 << 63) + i
        drop = (p, seed, offset, per) if p else None
        how = dict(post=_cuda(po), gate=_cuda(gt), pre=_cuda(pr), drop=Drop(*drop) if drop else None, stream_scale=0.75, block_scale=1.5)
        want = ro.forward(f, x, gt, po, pr, drop, 0.75, 1.5)
        s, y, stats = residual.join_forward(f.cuda(), _cuda(x), keep=True, **how)
        assert s.dtype == t
        ro.within(s, want[0], want[2], "s " + what)
        if pr is not None:
            ro.within(y, want[1], want[3], "y " + what)
        again = residual.join_forward(f.cuda(), _cuda(x), **how)
        assert torch.equal(again[0], s) and again[2] is None and (y is None or torch.equal(again[1], y))
        dy = dy if pr is not None else None
        for given in ((ds, dy), (None, dy) if pr is not None and i != 2 else (ds, None)):
            wanted = ro.backward(*given, f, gate=gt, post=po, pre=pr, drop=drop, a=0.75, b=1.5, **ro.of_s(s, want))
            got = residual.join_backward(_cuda(given[0]), _cuda(given[1]), f.cuda(), s, stats, need_stream=stream, **how)._asdict()
            for k, v in got.items():
                if k in wanted and v is not None:
                    ro.within(v, *wanted[k], what="d%s %s" % (k, what))
            assert {k for k, v in got.items() if v is not None} == set(wanted) - (set() if stream else {"stream"}) | ({"pre_weight", "pre_bias"} & {
                k for k in got if pr is not None and k.startswith("pre_") and getattr(how["pre"], k[4:]) is not None})
            if given[1] is None and pr is not None:
                assert not bool(got["pre_weight"].any())


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm(dev, host_layer, shape, kind, t):
    f, _, _, pr, _, _, dy = _inputs(shape, t, sum(shape), "none", kind, "none", False)
    n, X = _cuda(pr), f.cuda()
    want = ro.forward(f, None, None, None, pr, None, 1.0, 1.0)
    y, stats = residual.norm_forward(X, n, keep=True)
    ro.within(y, want[1], want[3], "y")
    assert torch.equal(residual.norm_forward(X, n), y)
    wanted = ro.backward(None, dy, f, f, None, None, pr, None, 1.0, 1.0)
    got = dict(zip(("block", "pre_weight", "pre_bias"), residual.norm_backward(dy.cuda(), X, stats, n)))
    for k, v in got.items():
        if v is not None:
            ro.within(v, *wanted[k], what="d" + k)
    alone = [residual.norm_backward(dy.cuda(), X, stats, n, *(i == j for j in range(3))) for i in range(3)]
    for i, k in enumerate(("block", "pre_weight", "pre_bias")):
        assert [v is not None for v in alone[i]] == [i == j and (j < 2 or kind == "layer") for j in range(3)]
        if got[k] is not None:
            assert torch.equal(alone[i][i], got[k])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_norm_without_parameters(dev, host_layer, t):
    for kind in ("rms", "layer"):
        for w, b in ((None, None), (None, torch.randn(40)), (torch.randn(40), None)):
            n = (kind, w, b, 1e-3)
            f, dy = torch.randn(6, 5, 40).to(t), torch.randn(6, 5, 40).to(t)
            want = ro.forward(f, None, None, None, n, None, 1.0, 1.0)
            y, stats = residual.norm_forward(f.cuda(), _cuda(n), keep=True)
            ro.within(y, want[1], want[3])
            wanted = ro.backward(None, dy, f, f, None, None, n, None, 1.0, 1.0)
            got = residual.norm_backward(dy.cuda(), f.cuda(), stats, _cuda(n))
            for k, v in zip(("block", "pre_weight", "pre_bias"), got):
                assert (v is not None) == (k in wanted)
                if v is not None:
                    ro.within(v, *wanted[k], what=k)


@pytest.mark.parametrize("p", [0.0, 1.0, 0.5, 2.0 ** -16, 1 - 2.0 ** -16, 0.1])
@pytest.mark.parametrize("per", ["element", "sample"])
def test_masks(dev, host_layer, p, per):
    """The mask bit for bit; infinities and NaN that are dropped are zeros; the same by a state on the GPU."""
    for shape in [(7,), (5, 24), (3, 4, 5), (40, 9, 129)]:
        x = torch.randn(shape) + 3
        seed, offset = (1 << 62) + 77, 123456789012
        kept, scale = ro.mask(shape, p, seed, offset, per)
        got = residual.dropout_forward(x.cuda(), Drop(p, seed, offset, per)).cpu()
        want = torch.where(kept, x * torch.tensor(scale, dtype=torch.float32), torch.zeros(()))
        assert torch.equal(got, want)
        state = torch.tensor([seed, offset], dtype=torch.int64).cuda()
        assert torch.equal(residual.dropout_forward(x.cuda(), Drop(p, state, 0, per)).cpu(), want)
        bad = torch.full(shape, float("nan"))
        got = residual.dropout_forward(bad.cuda(), Drop(p, seed, offset, per)).cpu()
        assert torch.equal(torch.isnan(got), kept) and not bool(got[~kept].any())


def test_share_that_is_kept(dev):
    """Within five deviations of a binomial count, and neighbouring offsets, seeds and rows without a common pattern."""
    x = torch.ones(2048, 1024).cuda()
    level = int(round(0.3 * 65536)) / 65536
    first = residual.dropout_forward(x, Drop(0.3, 1, 0)) > 0
    n = x.numel()
    for seed, offset in [(1, 0), (1, 1), (2, 0), (1, 1 << 32), (1 << 32, 0)]:
        kept = residual.dropout_forward(x, Drop(0.3, seed, offset)) > 0
        assert abs(int(kept.sum()) - n * (1 - level)) < 5 * (n * level * (1 - level)) ** 0.5
        if (seed, offset) != (1, 0):
            q = (1 - level) ** 2
            assert abs(int((kept & first).sum()) - n * q) < 5 * (n * q * (1 - q)) ** 0.5


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_numbers_that_are_none(dev, t):
    """They stay within their row."""
    f, x = torch.randn(6, 3, 72).to(t).cuda(), torch.randn(6, 3, 72).to(t).cuda()
    f[1, 0, 5], f[2, 1, 71], x[3, 2, 0] = float("nan"), float("inf"), float("-inf")
    s, y, _ = residual.join_forward(f, x, Norm("layer"), None, Norm("rms"))
    bad = torch.zeros(6, 3, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = bad[3, 2] = True
    assert torch.equal(~torch.isfinite(y).all(-1).cpu(), bad) and bool(torch.isnan(y[1, 0]).all())
    assert float(s[3, 2, 0]) == float("-inf") and bool(torch.isfinite(s[3, 2, 1:]).all())


def test_zero_rows_and_constants(dev):
    for kind in ("rms", "layer"):
        x = torch.zeros(4, 100).cuda()
        x[1] = 5
        y, stats = residual.norm_forward(x, Norm(kind), keep=True)
        want = torch.zeros(4, 100)
        if kind == "rms":
            want[1] = 5 / (25 + 1e-5) ** 0.5
        assert torch.allclose(y.cpu(), want, atol=1e-6)
        dx = residual.norm_backward(torch.ones(4, 100).cuda(), x, stats, Norm(kind))[0]
        assert bool(torch.isfinite(dx).all())


def test_large_means(dev):
    """A mean of a thousand deviations: the variance does not cancel.  The mean is off by at most (C / 512 + 256) 2^-24 of itself, a row's share of the bound."""
    x = torch.randn(64, 1000) + 1000
    pr = ("layer", None, None, 1e-5)
    want = ro.forward(x, None, None, None, pr, None, 1.0, 1.0)
    y = residual.norm_forward(x.cuda(), _cuda(pr))
    ro.within(y, want[1], want[3])
    assert float((y.cpu().double() - want[1]).norm() / want[1].norm()) < 1e-3


def test_strides_axes_and_starts(dev, host_layer):
    g = torch.Generator().manual_seed(4)
    base = torch.randn(6, 8, 205, generator=g).bfloat16().cuda()
    n = Norm("layer", torch.randn(100, generator=g).bfloat16().cuda(), torch.randn(200, generator=g).bfloat16().cuda()[::2])
    drop = Drop(0.2, 5, 6)
    for f in (base[..., 1:101], base[:, ::2, 100:200], base.transpose(0, 1)[..., :100], base[:, :1, :100].expand(6, 8, 100)):
        x = f.flip(0)
        want = residual.join_forward(f.contiguous().clone(), x.contiguous().clone(), n, None, n, drop)
        got = residual.join_forward(f, x, n, None, n, drop)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # (N, C, H, W), in either memory order
    f, x = torch.randn(2, 100, 5, 3, generator=g).bfloat16().cuda(), torch.randn(2, 100, 5, 3, generator=g).bfloat16().cuda()
    last = [v.permute(0, 2, 3, 1) for v in (f, x)]
    want = residual.join(last[0].contiguous(), last[1].contiguous(), n, None, n, drop)
    for a, b in ((f, x), (f.to(memory_format=torch.channels_last), x)):
        got = residual.join(a, b, n, None, n, drop, channel_axis=1)
        for u, v in zip(got, want):
            assert torch.equal(u, v.permute(0, 3, 1, 2)) and u.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(residual.norm(f, n, 1), residual.norm(last[0], n).permute(0, 3, 1, 2))
    assert torch.equal(residual.dropout(f, drop, 1), residual.dropout(last[0], drop).permute(0, 3, 1, 2))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_autograd(dev, host_layer, t):
    """Each gradient, float32 parameters, tensors that need none, results that go nowhere."""
    for i, (post, pre, gate, p, per, stream) in enumerate(FORMS):
        f, x, po, pr, gt, ds, dy = _inputs((3, 5, 72), t, i, post, pre, gate, stream, wide=True)
        drop = (p, 3, 4, per) if p else None
        leaves = {"block": _cuda(f), "stream": _cuda(x), "gate": _cuda(gt)}
        norms = {}
        for name, n in (("post", po), ("pre", pr)):
            norms[name] = _cuda(n)
            if n is not None:
                leaves.update({name + "_weight": norms[name].weight, name + "_bias": norms[name].bias})
        leaves = {k: v.requires_grad_() for k, v in leaves.items() if v is not None}
        call = lambda: residual.join(leaves["block"], leaves.get("stream"), norms["post"], leaves.get("gate"), norms["pre"], Drop(*drop) if drop else None, 0.75, 1.5)  # noqa: E731
        out = call()
        s, y = out if pr is not None else (out, None)
        exact = ro.forward(f, x, gt, po, pr, drop, 0.75, 1.5)
        for given in ([ds, dy], [None, dy], [ds, None]) if pr is not None else ([ds, None],):
            wanted = ro.backward(*given, f, gate=gt, post=po, pre=pr, drop=drop, a=0.75, b=1.5, **ro.of_s(s, exact))
            pairs = [(o, v.cuda()) for o, v in zip((s, y), given) if v is not None]
            got = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [v for _, v in pairs], retain_graph=True, allow_unused=True)
            for k, v in zip(leaves, got):
                if k in wanted:
                    assert v.dtype == leaves[k].dtype
                    ro.within(v, *wanted[k], what="d%s %d" % (k, i))
        for k in leaves:
            for other in leaves.values():
                other.requires_grad_(False)
            leaves[k].requires_grad_()
            out = call()
            outs = list(out) if pr is not None else [out]
            got = torch.autograd.grad(outs, [leaves[k]], [ds.cuda(), dy.cuda()][:len(outs)])[0]
            ro.within(got, *ro.backward(ds, dy if pr is not None else None, f, gate=gt, post=po, pre=pr, drop=drop, a=0.75, b=1.5, **ro.of_s(s, exact))[k], what=k)


@pytest.mark.parametrize("t", TYPES[1:], ids=str)
def test_gradients_from_a_rounded_s(dev, host_layer, t):
    """Without the block, pre's gradient goes by s as it is given; a norm behind a join whose s went nowhere, and one whose stream is missing, compute it again."""
    f, x, _, pr, _, ds, dy = _inputs((3, 5, 72), t, 1, "none", "layer", "none")
    n = _cuda(pr)
    s, y, stats = residual.join_forward(f.cuda(), x.cuda(), pre=n, keep=True)
    want = ro.forward(f, x, None, None, pr, None, 1.0, 1.0)
    got = residual.join_backward(ds.cuda(), dy.cuda(), None, s, stats, pre=n)
    for k, (v, bound) in ro.backward(ds, dy, f, s.cpu(), None, None, pr, None, 1.0, 1.0, s_exact=want[0]).items():
        ro.within(getattr(got, k), v, bound, k)
    again = residual.join_backward(ds.cuda(), dy.cuda(), f.cuda(), None, stats, pre=n)
    for k, (v, bound) in ro.backward(ds, dy, f, want[0], None, None, pr, None, 1.0, 1.0, s_off=want[4]).items():
        ro.within(getattr(again, k), v, bound, k)
    leaf = f.cuda().requires_grad_()
    _, y = residual.join(leaf, None, pre=n)
    (df,) = torch.autograd.grad(y, leaf, dy.cuda())
    want = ro.forward(f, None, None, None, pr, None, 1.0, 1.0)
    ro.within(df, *ro.backward(None, dy, f, want[0], None, None, pr, None, 1.0, 1.0, s_off=want[4])["block"], what="alone")


def test_nothing_to_do(dev, host_layer):
    n = Norm("layer", torch.ones(8).cuda().requires_grad_(), torch.ones(8).cuda().requires_grad_())
    gate = torch.ones(8).cuda().requires_grad_()
    for shape in ((0, 8), (3, 0, 8)):
        f = torch.zeros(shape).cuda().requires_grad_()
        s, y = residual.join(f, f, n, gate, n, Drop(0.5, 1))
        assert s.shape == shape and y.shape == shape
        grads = torch.autograd.grad([s, y], [f, n.weight, n.bias, gate], [torch.zeros_like(s), torch.zeros_like(y)])
        assert grads[0].shape == shape and not any(bool(v.any()) for v in grads[1:])


def test_modules_and_captured_passes(dev):
    """A stack of blocks in training, eager and captured; a replay draws another mask."""
    torch.manual_seed(0)
    blocks = [residual.matrix_block(72, 200), residual.matrix_block(72, 136, "silu")]
    stack = pkg.ResidualStack(blocks, 72, post=True, gate=0.5, drop=0.4, per="element", counter=True).cuda()
    x = torch.randn(4, 33, 72).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    params = list(stack.parameters())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(stack(x).sum(), params)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = stack(x)
        grads = torch.autograd.grad(y.square().sum(), params)
    seen = []
    for i in range(4):
        states = [d.state.clone() for d in stack.drops]
        graph.replay()
        torch.cuda.synchronize()
        got, got_grads = y.clone(), [v.clone() for v in grads]
        after = [d.state.clone() for d in stack.drops]
        for d, st, now in zip(stack.drops, states, after):
            assert int(now[1]) == int(st[1]) + 1
            d.state.copy_(st)
        eager = stack(x)
        want = torch.autograd.grad(eager.square().sum(), params)
        assert torch.equal(got, eager.detach())
        for a, b in zip(got_grads, want):
            assert torch.equal(a, b)
        del eager, want
        seen.append(got)
    assert not torch.equal(seen[0], seen[1])


def test_stack_against_torch(dev):
    """In float32 and evaluation: the same layers by torch in 64 bits; then with weights in 4 bits against unpacked ones."""
    torch.manual_seed(1)
    for kind in ("rms", "layer"):
        stack = pkg.ResidualStack([residual.matrix_block(40, 64) for _ in range(3)], 40, kind, post=True, gate=0.7, drop=0.3, stream_scale=0.9).cuda().eval()
        x = torch.randn(5, 7, 40)

        def reference():
            wide = lambda v: None if v is None else v.detach().double().cpu()  # noqa: E731
            v = x.double()
            n = lambda m, v: ro.norm(v, kind, wide(m.weight), wide(m.bias), m.eps)  # noqa: E731
            for i, b in enumerate(stack.blocks):
                h = n(stack.pre[i], v)
                for layer in b:
                    w = layer.weight if isinstance(layer, pkg.MatrixLinear) else pkg.packed4.unpack4(layer.weight, torch.float32)
                    h = torch.nn.functional.linear(h, wide(w), wide(layer.bias))
                    h = torch.nn.functional.gelu(h) if layer.activation == "gelu" else h
                v = 0.9 * v + wide(stack.gates[i]) * n(stack.post[i], h)
            return n(stack.pre[3], v)
        y = stack(x.cuda())
        assert float((y.detach().cpu().double() - reference()).norm() / reference().norm()) < 1e-5
        stack.pack4()
        assert all(isinstance(layer, pkg.MatrixLinear4) for b in stack.blocks for layer in b)
        y = stack(x.cuda())
        assert float((y.detach().cpu().double() - reference()).norm() / reference().norm()) < 1e-5
        # inputs in 4 bits too: serving, no gradient
        stack = pkg.ResidualStack([residual.matrix_block(40, 64) for _ in range(2)], 40, kind, gate=0.7).cuda().eval().pack4(True)
        with torch.no_grad():
            y = stack(x.cuda())
        assert y.shape == x.shape and bool(torch.isfinite(y).all()) and all(layer.x4 for b in stack.blocks for layer in b)


def test_gradients_by_differences(dev):
    """A training step of a stack in float32 against central differences of the oracle's 64 bits: along one direction of every parameter."""
    torch.manual_seed(2)
    stack = pkg.ResidualStack([residual.matrix_block(24, 40, "silu")], 24, "rms", gate=0.8, drop=0.0).cuda()
    x = torch.randn(6, 5, 24)
    weight = torch.randn(6, 5, 24)
    params = dict(stack.named_parameters())
    grads = dict(zip(params, torch.autograd.grad((stack(x.cuda()) * weight.cuda()).sum(), list(params.values()))))

    def total(p):
        v = x.double()
        h = ro.norm(v, "rms", p["pre.0.weight"], None, 1e-5)
        h = torch.nn.functional.silu(torch.nn.functional.linear(h, p["blocks.0.0.weight"], p["blocks.0.0.bias"]))
        h = torch.nn.functional.linear(h, p["blocks.0.1.weight"], p["blocks.0.1.bias"])
        return float((ro.norm(v + p["gates.0"] * h, "rms", p["pre.1.weight"], None, 1e-5) * weight.double()).sum())
    values = {k: v.detach().double().cpu() for k, v in params.items()}
    for k in params:
        d = torch.randn(values[k].shape, dtype=torch.float64)
        up, down = (total({**values, k: values[k] + step * d}) for step in (1e-5, -1e-5))
        slope = (up - down) / 2e-5
        scale = float(grads[k].double().cpu().norm() * d.norm())
        assert abs(slope - float((grads[k].double().cpu() * d).sum())) < 1e-4 * scale, k


def test_dropout_module(dev):
    torch.manual_seed(3)
    m = pkg.Dropout(0.25).cuda()
    x = torch.ones(50, 64).cuda()
    a, b = m(x), m(x)
    assert not torch.equal(a, b) and m.calls == 2
    state = m.state_dict()
    c = m(x)
    other = pkg.Dropout(0.25)
    other.load_state_dict(state)
    assert torch.equal(other(x), c)
    assert torch.equal(m.eval()(x), x)
    assert torch.equal(pkg.Dropout(0.0)(x), x)
    leaf = x.clone().requires_grad_()
    y = m.train()(leaf)
    (grad,) = torch.autograd.grad(y, leaf, x)
    assert torch.equal(grad, y.detach())


def test_stream_and_two_at_once(dev):
    f = [torch.randn(500, 40, 96).cuda() for _ in range(2)]
    n = Norm("layer", torch.randn(96).cuda(), torch.randn(96).cuda())
    gate = torch.randn(500, 96).cuda()

    def step(v):
        s, y, stats = residual.join_forward(v, v, n, gate, n, Drop(0.2, 9), keep=True)
        return (s, y) + tuple(residual.join_backward(s, y, v, s, stats, n, gate, n, Drop(0.2, 9)))
    want = [step(v) for v in f]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in f]
    got = []
    for v, st in zip(f, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append([step(v) for _ in range(3)])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for once in g:
            assert all(torch.equal(a, b) for a, b in zip(w, once))


def test_beyond_32_bits(dev):
    """More than 2^31 elements: the last rows are those of a call of their own, and their mask is theirs."""
    rows, C = 300000, 8200
    f = torch.empty(rows, C, dtype=torch.bfloat16, device="cuda").normal_()
    n = Norm("layer", torch.randn(C).cuda(), torch.randn(C).cuda())
    y, stats = residual.norm_forward(f, n, keep=True)
    assert f.numel() > 1 << 31 and torch.equal(y[-5:], residual.norm_forward(f[-5:], n))
    dx, dw, db = residual.norm_backward(y, f, stats, n)
    assert torch.equal(dx[-5:], residual.norm_backward(y[-5:], f[-5:], stats[-5:].clone(), n)[0])
    assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())
    del dx
    s = residual.join_forward(f, y, drop=Drop(0.3, 11, 12))[0]
    kept = (ro.words(5, C, 11, 12, rows - 5)[:, :C] >= int(round(0.3 * 65536))).cuda()
    scale = 65536 / (65536 - int(round(0.3 * 65536)))
    want = y[-5:].float() + torch.where(kept, f[-5:].float() * scale, torch.zeros((), device="cuda"))
    assert float((s[-5:].float() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


@pytest.mark.parametrize("C", [40, 1000, 2056])
def test_many_samples(dev, C):
    """More samples than workgroups, of few rows each: the sums behind a sample's gate."""
    for t in (torch.float32, torch.bfloat16):
        f, x, po, pr, gt, ds, dy = _inputs((1500, 3, C), t, C, "layer", "rms", "sample")
        how = dict(post=_cuda(po), gate=_cuda(gt), pre=_cuda(pr), drop=Drop(0.2, 1, 2, "sample"))
        s, y, stats = residual.join_forward(f.cuda(), x.cuda(), keep=True, **how)
        want = ro.forward(f, x, gt, po, pr, (0.2, 1, 2, "sample"), 1.0, 1.0)
        ro.within(s, want[0], want[2], "s")
        wanted = ro.backward(ds, dy, f, gate=gt, post=po, pre=pr, drop=(0.2, 1, 2, "sample"), a=1.0, b=1.0, **ro.of_s(s, want))
        got = residual.join_backward(ds.cuda(), dy.cuda(), f.cuda(), s, stats, **how)._asdict()
        for k, (v, bound) in wanted.items():
            ro.within(got[k], v, bound, k)


def test_same_bits_every_time(dev):
    f, x, po, pr, gt, ds, dy = _inputs((4, 600, 520), torch.bfloat16, 1, "layer", "layer", "channel")
    how = dict(post=_cuda(po), gate=_cuda(gt), pre=_cuda(pr), drop=Drop(0.2, 1, 2))
    args = [v.cuda() for v in (f, x, ds, dy)]

    def step():
        s, y, stats = residual.join_forward(args[0], args[1], keep=True, **how)
        return (s, y) + tuple(residual.join_backward(args[2], args[3], args[0], s, stats, **how))
    first = step()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


@pytest.mark.parametrize("rows,C", [(5000, 4104), (17000, 523), (600, 70001)])
def test_rows_in_pieces(dev, rows, C):
    """Joins without a norm whose rows are taken in pieces, more rows than workgroups: the mask of narrower rows, and the sum value by value."""
    g = torch.Generator().manual_seed(C)
    f, x = torch.randn(rows, C, generator=g).cuda(), torch.randn(rows, C, generator=g).cuda()
    gate, drop = torch.randn(C, generator=g).cuda(), Drop(0.25, 11, 12)
    out = residual.dropout_forward(f, drop)
    assert torch.equal(out[:, :512], residual.dropout_forward(f[:, :512].contiguous(), drop))
    kept = out != 0
    assert torch.equal(out, torch.where(kept, f * torch.tensor(1 / 0.75, device=dev), torch.zeros_like(f)))
    # (the share of n channels: a standard deviation of sqrt(3 / 16 / n); six of them)
    assert abs(kept.double().mean().item() - 0.75) < 6 * (3 / 16 / (rows * C)) ** 0.5
    s, _, _ = residual.join_forward(f, x, gate=gate, drop=drop, stream_scale=0.5, block_scale=2.0)
    block = torch.where(kept, f.double() * gate.double() * (2.0 / 0.75), torch.zeros((), dtype=torch.float64, device=dev))
    # four roundings of the block's factors and products, one of the share, one of the sum
    bound = (5 * block.abs() + (block + 0.5 * x.double()).abs()) * 2.0 ** -23
    assert ((s.double() - (block + 0.5 * x.double())).abs() <= bound).all()
