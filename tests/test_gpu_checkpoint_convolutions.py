"""Convolutions that keep their input in 8 bits, where the tests of the linear layers do not take them: trained 3-D layers, and fp32 parameters
on 16-bit activations."""
import pytest
import torch

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import checkpoint8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nd", [2, 3])
@pytest.mark.parametrize("t,parameters", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float16, torch.float32),
                                          (torch.bfloat16, torch.float32)], ids=str)
@pytest.mark.parametrize("cin,cout,k,stride", [(64, 32, 3, 1), (24, 40, 3, 2), (20, 36, 5, 1), (40, 16, 1, 1)])
def test_trained_layers(dev, host_layer, nd, t, parameters, cin, cout, k, stride):
    make = pkg.WinoConv2d if nd == 2 else pkg.WinoConv3d
    conv, same = (make(cin, cout, k, stride, k // 2, checkpoint=c).to(dev, parameters) for c in ("int8", None))
    same.load_state_dict(conv.state_dict())
    memory = torch.channels_last if nd == 2 else torch.channels_last_3d
    last = lambda v: v.movedim(1, -1)  # noqa: E731
    for given in (memory, torch.contiguous_format):
        x = torch.randn(2, cin, *((4,) if nd == 3 else ()), 10, 9, device=dev).to(t).contiguous(memory_format=given)
        packed = checkpoint8.pack8(last(x))
        xq = checkpoint8.unpack8(packed).movedim(-1, 1)
        kept = []

        def keep(v):
            kept.append(v)
            return v
        a, b, q = (v.clone(memory_format=torch.preserve_format).requires_grad_() for v in (x, x, xq))
        conv.zero_grad()
        with torch.autograd.graph.saved_tensors_hooks(keep, lambda v: v):
            y = conv(a)
        assert any(v.dtype == torch.int8 and v.numel() == x.numel() for v in kept)
        assert not any(v.shape == x.shape and v.dtype == t for v in kept)
        dy = torch.randn_like(y)
        y.backward(dy)
        same.zero_grad()
        y2 = same(b)
        y2.backward(dy)
        assert torch.equal(y, y2) and torch.equal(a.grad, b.grad) and torch.equal(conv.bias.grad, same.bias.grad)
        assert conv.weight.grad.dtype == parameters and conv.bias.grad.dtype == parameters
        # the weight gradient is the one of what the 8 bits stand for
        same.zero_grad()
        same(q).backward(dy)
        assert torch.equal(conv.weight.grad, same.weight.grad)
