"""Layers over a weight in 4 bits inside models that are moved, saved and loaded."""
import pytest
import torch

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import matrix_linear, packed4

pytestmark = pytest.mark.gpu


def _step(layer, x):
    leaf = x.clone().requires_grad_()
    y = layer(leaf)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    return y.detach(), dx


@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("images", [1, 40])
def test_memory_formats(dev, host_layer, images, t):
    """Beside convolutions, whose tensors' layout is not the scales': results and the gradient of x stay as they were, few pixels and many."""
    torch.manual_seed(0)
    layer = pkg.MatrixLinear(300, 72, activation="silu", channel_axis=1).cuda().to(t).pack4()
    model = torch.nn.Sequential(torch.nn.Conv2d(4, 300, 1).to(t).cuda(), layer)
    x = torch.randn(images, 300, 3, 5, device=dev).to(t)
    want = _step(layer, x)
    with torch.no_grad():
        want4 = matrix_linear.linear(packed4.pack4(x.movedim(1, -1)), layer.weight)
    model.to(memory_format=torch.channels_last)
    for given in (x, x.to(memory_format=torch.channels_last)):
        assert all(torch.equal(a, b) for a, b in zip(_step(layer, given), want))
    assert torch.equal(matrix_linear.linear(packed4.pack4(x.movedim(1, -1)), layer.weight), want4)
    assert torch.equal(packed4.unpack4(layer.weight), packed4.unpack4(packed4.Packed4(layer.codes, layer.scales.unflatten(2, (32, 4)), 300, t)))


def test_parts_that_lie_otherwise(dev, host_layer):
    """Codes and scales with other strides and starts, of the weight and of x."""
    torch.manual_seed(1)
    for rows in (3, 40, 600):
        w, x = packed4.pack4(torch.randn(70, 300, device=dev)), packed4.pack4(torch.randn(rows, 300, device=dev).half())
        z, dy = torch.randn(rows, 70, device=dev).half(), torch.randn(rows, 70, device=dev).half()

        def results(w, x):
            full = packed4.unpack4(x)
            return (matrix_linear.linear_forward(x, w), matrix_linear.linear_forward(full, w), full, packed4.unpack4(w, torch.float32),
                    matrix_linear.linear_backward(dy, None, w, z, "gelu", need_dw=False, need_db=False)[0],
                    matrix_linear.linear_backward(dy, None, w, z, "gelu", need_dw=False)[0])
        want = results(w, x)
        for move in (lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2),
                     lambda v: torch.empty(v.numel() + 1, dtype=torch.uint8, device=dev)[1:].view(v.shape).copy_(v)):
            others = []
            for p in (w, x):
                other = packed4.Packed4(p.codes, p.scales, 300, p.dtype)
                other.codes, other.scales = move(p.codes), move(p.scales)
                others.append(other)
            assert all(torch.equal(a, b) for a, b in zip(results(*others), want))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_checkpoints_are_kept(dev, checkpoint):
    """What a layer keeps for its backward pass, and its gradient, are those of `linear` with the same checkpoint."""
    torch.manual_seed(2)
    layer = pkg.MatrixLinear(96, 64, activation="gelu", checkpoint=checkpoint).cuda()
    four, x = layer.pack4(), torch.randn(70, 96, device=dev)

    def kept(call):
        held = []
        leaf = x.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda v: (held.append((v.dtype, v.numel())), v)[1], lambda v: v):
            y = call(leaf)
        return held, torch.autograd.grad(y.sum(), leaf)[0]
    got, want = kept(four), kept(lambda v: matrix_linear.linear(v, four.weight, four.bias, None, "gelu", checkpoint=checkpoint))
    assert got[0] == want[0] and torch.equal(got[1], want[1])
    assert ((torch.int8, 70 * 64) in got[0]) == (checkpoint == "int8") and ((torch.float32, 70 * 64) in got[0]) == (checkpoint is None)
