"""MatrixLinear and layers that keep their input in 8 bits, as a network trains them: gradients against 64 bits and differences, streams, captured
graphs, parameters of another type, and a block of convolutions and linear layers together."""
import pytest
import torch
import torch.nn.functional as F

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import checkpoint8, matrix_linear

import linear_oracle as lo

pytestmark = pytest.mark.gpu


def _layer(C, K, seed, dev, t=torch.float32, **kw):
    layer = pkg.MatrixLinear(C, K, **kw)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        layer.weight.copy_(torch.randn(K, C, generator=g) * C ** -0.5)
        if layer.bias is not None:
            layer.bias.copy_(torch.randn(K, generator=g))
    return layer.to(dev, t)


@pytest.mark.parametrize("act", lo.ACTS)
@pytest.mark.parametrize("after", [False, True])
def test_gradients_against_autograd_in_64_bits(dev, act, after):
    layer = _layer(40, 56, 3, dev, activation=act, residual_after=after)
    g = torch.Generator().manual_seed(1)
    x, r, dy = (torch.randn(5, 9, n, generator=g) for n in (40, 56, 56))
    X, R = x.to(dev).requires_grad_(), r.to(dev).requires_grad_()
    y = layer(X, R)
    y.backward(dy.to(dev))
    x64, r64, w64, b64 = (v.detach().cpu().double().requires_grad_() for v in (x, r, layer.weight, layer.bias))
    z = F.linear(x64, w64, b64)
    z = z if after else z + r64
    y64 = lo.act(z, act) + (r64 if after else 0)
    y64.backward(dy.double())
    for a, c in ((y, y64), (X.grad, x64.grad), (R.grad, r64.grad), (layer.weight.grad, w64.grad), (layer.bias.grad, b64.grad)):
        # sums of at most 56 fp32 products of numbers about 1: 64 roundings of 2^-24 each, of sums of up to 64 (in the 2-norm far less)
        assert float((a.detach().cpu().double() - c.detach()).abs().max()) <= 64 * 64 * lo.SUM


@pytest.mark.parametrize("act", lo.ACTS)
def test_gradients_against_differences(dev, act):
    """In fp32: the change of <y, dy> along a direction, by central differences of y taken in 64 bits on the CPU from the layer's own formula."""
    layer = _layer(24, 32, 5, dev, activation=act)
    g = torch.Generator().manual_seed(2)
    x, dy, dx = (torch.randn(20, n, generator=g) for n in (24, 32, 24))
    X = x.to(dev).requires_grad_()
    layer(X).backward(dy.to(dev))
    w, b = layer.weight.detach().cpu().double(), layer.bias.detach().cpu().double()
    h = 1e-5
    f = lambda v: float((lo.act(v @ w.t() + b, act) * dy.double()).sum())  # noqa: E731
    change = (f(x.double() + h * dx.double()) - f(x.double() - h * dx.double())) / (2 * h)
    got = float((X.grad.cpu().double() * dx.double()).sum())
    # relu: a unit may turn within h, which changes the difference by less than h |slope| each; the rest is fp32's rounding of 480 terms
    assert abs(got - change) <= 1e-3 * max(1.0, abs(change)) if act == "relu" else abs(got - change) <= 2e-4 * max(1.0, abs(change))


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
def test_parameters_in_fp32_get_their_gradients_unrounded(dev, t):
    layer = _layer(72, 48, 6, dev, activation="gelu")
    x = torch.randn(64, 72, device=dev).to(t).requires_grad_()
    dy = torch.randn(64, 48, device=dev).to(t)
    layer(x).backward(dy)
    assert layer.weight.grad.dtype == torch.float32 and x.grad.dtype == t
    w, b = layer.weight.detach().to(t), layer.bias.detach().to(t)
    y, z = matrix_linear.linear_forward(x.detach(), w, b, None, "gelu", keep_z=True)
    want = matrix_linear.linear_backward(dy, x.detach(), w, z, "gelu", w_type=torch.float32, b_type=torch.float32)
    for a, c in zip((x.grad, layer.weight.grad, layer.bias.grad), want):
        assert torch.equal(a, c)


def _kept_bytes(fn):
    """Bytes of the tensors that fn's graph keeps beside its leaves."""
    seen = {}

    def pack(t):
        if not t.is_leaf or not t.requires_grad:
            seen[t.data_ptr()] = t.numel() * t.element_size()
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = fn()
    return y, sum(seen.values())


@pytest.mark.parametrize("act", lo.ACTS)
@pytest.mark.parametrize("after", [False, True])
def test_a_layer_that_keeps_8_bits(dev, act, after):
    """Its gradients are those of the tensors that the 8 bits stand for, relu's gate is z's own, and it keeps about half."""
    t = torch.float16
    layer = _layer(96, 64, 9, dev, t, activation=act, residual_after=after, checkpoint="int8")
    x = torch.randn(128, 96, device=dev).to(t).requires_grad_()
    r = torch.randn(128, 64, device=dev).to(t).requires_grad_()
    dy = torch.randn(128, 64, device=dev).to(t)
    y, kept = _kept_bytes(lambda: layer(x, r))
    y.backward(dy)
    full = pkg.MatrixLinear(96, 64, activation=act, residual_after=after).to(dev, t)
    full.load_state_dict(layer.state_dict())
    assert torch.equal(full(x, r), y)
    z = matrix_linear.linear_forward(x.detach(), layer.weight.detach(), layer.bias.detach(), None if after else r.detach())
    px, pz = checkpoint8.pack8(x.detach()), checkpoint8.pack8(z, act == "relu")
    dx, dw, db, dz = matrix_linear.linear_backward(dy, px, layer.weight.detach(), pz, act, need_dz=True)
    for a, c in ((x.grad, dx), (r.grad, dy if after else dz), (layer.weight.grad, dw), (layer.bias.grad, db)):
        assert torch.equal(a, c)
    if act == "relu":
        assert torch.equal(dz != 0, (z > 0) & (dy != 0))
    assert kept <= 1.04 * (x.numel() + (y.numel() if act != "none" else 0))


@pytest.mark.parametrize("t,cin,cout,k,stride", [(torch.float16, 64, 64, 3, 1), (torch.bfloat16, 40, 24, 3, 2), (torch.float32, 20, 36, 5, 1), (torch.float16, 32, 48, 1, 1)])
def test_a_convolution_that_keeps_8_bits(dev, t, cin, cout, k, stride):
    conv = pkg.WinoConv2d(cin, cout, k, stride, k // 2, checkpoint="int8").to(dev, t)
    same = pkg.WinoConv2d(cin, cout, k, stride, k // 2).to(dev, t)
    same.load_state_dict(conv.state_dict())
    for memory in (torch.channels_last, torch.contiguous_format):
        x = torch.randn(3, cin, 14, 13, device=dev).to(t).contiguous(memory_format=memory)
        xq = checkpoint8.unpack8(checkpoint8.pack8(x.permute(0, 2, 3, 1))).permute(0, 3, 1, 2)
        a, b = x.clone(memory_format=memory).requires_grad_(), x.clone(memory_format=memory).requires_grad_()
        for layer in (conv, same):
            layer.zero_grad()
        y, kept = _kept_bytes(lambda: conv(a))
        assert kept <= 1.1 * x.numel() * (32 * -(-cin // 32)) / cin
        dy = torch.randn_like(y)
        y.backward(dy)
        y2 = same(b)
        assert torch.equal(y, y2)
        y2.backward(dy)
        assert torch.equal(a.grad, b.grad) and torch.equal(conv.bias.grad, same.bias.grad)
        # the weight gradient is the one of what the 8 bits stand for
        same.zero_grad()
        same(xq.contiguous(memory_format=torch.channels_last).requires_grad_()).backward(dy)
        assert torch.equal(conv.weight.grad, same.weight.grad)
    with torch.no_grad():
        assert torch.equal(conv(x), same(x))
    frozen = pkg.WinoConv3d(8, 8, 3, 1, 1, checkpoint="int8").to(dev, t).requires_grad_(False)
    x = torch.randn(1, 8, 4, 6, 6, device=dev).to(t).requires_grad_()
    frozen(x).sum().backward()
    assert x.grad is not None
    with pytest.raises(NotImplementedError, match="torch runs this one"):
        pkg.WinoConv2d(8, 8, 3, groups=2, checkpoint="int8").to(dev, t)(torch.randn(1, 8, 9, 9, device=dev).to(t))


def test_gradients_are_not_differentiable_themselves(dev):
    layer = _layer(16, 16, 1, dev, activation="silu")
    x = torch.randn(4, 16, device=dev, requires_grad=True)
    g, = torch.autograd.grad(layer(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def _block(dev, t, checkpoint):
    """A convolution, a 1x1 layer around it with its input as the residual, and a classifier: 8 -> 16 -> 8 channels."""
    torch.manual_seed(4)
    conv = pkg.WinoConv2d(32, 64, 3, 1, 1, checkpoint=checkpoint)
    up = pkg.MatrixLinear(64, 32, activation="relu", channel_axis=1, checkpoint=checkpoint)
    head = pkg.MatrixLinear(32, 10, activation="none", checkpoint=checkpoint)
    return torch.nn.ModuleList([conv, up, head]).to(dev, t)


def _block_step(layers, x, dy):
    conv, up, head = layers
    h = up(torch.relu(conv(x)), residual=x)
    y = head(h.mean(dim=(2, 3)))
    grads = torch.autograd.grad(y, [x] + [p for layer in layers for p in layer.parameters()], dy)
    # no graph of this pass outlives it: torch ends the process where a backward pass is captured while an eager graph of the same leaves lives
    return y.detach(), grads


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_layers_together_and_captured(dev, checkpoint):
    """A training step of the block in fp32 against 64 bits, then captured and replayed three times with other inputs between eager work."""
    layers = _block(dev, torch.float32, checkpoint)
    x = torch.randn(4, 32, 12, 10, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_()
    dy = torch.randn(4, 10, device=dev)
    y, grads = _block_step(layers, x, dy)
    ref = [p.detach().cpu().double().requires_grad_() for layer in layers for p in layer.parameters()]
    x64 = x.detach().cpu().double().requires_grad_()
    h = torch.relu(F.conv2d(x64, ref[0], ref[1], padding=1))
    h = torch.relu(torch.einsum("nchw,kc->nkhw", h, ref[2][:, :]) + ref[3][None, :, None, None] + x64)
    y64 = F.linear(h.mean(dim=(2, 3)), ref[4], ref[5])
    g64 = torch.autograd.grad(y64, [x64] + ref, dy.cpu().double())
    # 8 bits are off by at most 2^-7 of a group's largest, half of that on average, signs at random; a relu may turn at fp32's rounding of 0
    tol = 2.0 ** -7 if checkpoint else 1e-4
    assert float((y.cpu().double() - y64.detach()).norm() / y64.norm()) <= 1e-4
    for a, c in zip(grads, g64):
        assert float((a.cpu().double() - c).norm() / c.norm()) <= tol

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block_step(layers, x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _block_step(layers, x, dy)
    for seed in range(3):
        g = torch.Generator(device=dev).manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=dev))
            dy.copy_(torch.randn(dy.shape, generator=g, device=dev))
        want = _block_step(layers, x, dy)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0])
        for a, c in zip(out[1], want[1]):
            assert torch.equal(a, c)


def test_two_streams_at_once(dev):
    t = torch.bfloat16
    sets = []
    for i in range(2):
        g = torch.Generator(device=dev).manual_seed(i)
        x, w, dy = (torch.randn(s, generator=g, device=dev).to(t) for s in ((700, 256), (320, 256), (700, 320)))
        sets.append((x, w, dy, [matrix_linear.linear_forward(x, w, activation="gelu", keep_z=True)]))
        sets[-1][3].append(matrix_linear.linear_backward(dy, checkpoint8.pack8(x), w, sets[-1][3][0][1], "gelu"))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[], []]
    for _ in range(5):
        for s, (x, w, dy, _), out in zip(streams, sets, results):
            with torch.cuda.stream(s):
                y, z = matrix_linear.linear_forward(x, w, activation="gelu", keep_z=True)
                out.append((y, z, *matrix_linear.linear_backward(dy, checkpoint8.pack8(x), w, z, "gelu")[:3]))
    torch.cuda.synchronize()
    for (x, w, dy, want), out in zip(sets, results):
        for got in out:
            for a, c in zip(got, (*want[0], *want[1][:3])):
                assert torch.equal(a, c)
