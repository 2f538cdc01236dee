"""Arguments of linear layers and 8 bits that the C ABI could not tell apart from others, refused on the CPU before any launch."""
import pytest
import torch
from torch.autograd import forward_ad

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import checkpoint8, matrix_linear


def test_channels_beyond_an_int(host_layer):
    """2^32 + 32 channels would be 32 of them behind an int."""
    n = (1 << 32) + 32
    wide = torch.zeros(1, dtype=torch.float16).expand(1, n)
    codes = torch.zeros(1, dtype=torch.int8)
    with pytest.raises(ValueError, match="pack8: 4294967328 channels"):
        checkpoint8.pack8(wide)
    with pytest.raises(ValueError, match="unpack8: 4294967328 channels"):
        checkpoint8.unpack8(checkpoint8._made(codes.expand(1, n), codes.expand(1, n // 32), torch.float16))
    with pytest.raises(ValueError, match="linear_forward: 4294967328 channels"):
        matrix_linear.linear_forward(wide, wide)
    with pytest.raises(ValueError, match="linear_forward: 4294967328 channels"):
        matrix_linear.linear_forward(wide[:, :1], wide.t())
    with pytest.raises(ValueError, match="linear_backward: 4294967328 channels"):
        matrix_linear.linear_backward(wide, None, None, need_dx=False, need_dw=False)
    with pytest.raises(ValueError, match="linear_backward: 4294967328 channels"):
        matrix_linear.linear_backward(wide[:, :1], wide, None, need_dx=False)


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(which):
    """A tangent would be dropped without a word, gradients asked for or not."""
    ts = [torch.randn(s) for s in ((3, 4), (5, 4), (5,), (3, 5))]
    with forward_ad.dual_level():
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        for t in (ts[0], ts[0].detach().requires_grad_() if which else ts[0]):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                matrix_linear.linear(t, *ts[1:])
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            matrix_linear.linear(*ts)
        if which == 0:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                pkg.MatrixLinear(4, 5, channel_axis=1)(ts[0].view(1, 3, 4).movedim(2, 1))
    # outside of a level, and within one without tangents, it goes on to the checks of the layer
    ts = [torch.randn(s) for s in ((3, 4), (5, 4), (5,), (3, 5))]
    with pytest.raises(ValueError, match="GPU only"):
        matrix_linear.linear(*ts)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="GPU only"):
        matrix_linear.linear(*ts)


def test_operands_without_axes_are_named():
    dy, x, w, point = torch.randn(3, 5), torch.randn(3, 4), torch.randn(5, 4), torch.tensor(1.0)
    with pytest.raises(ValueError, match="w of shape"):
        matrix_linear.linear_backward(dy, x, point)
    with pytest.raises(ValueError, match="x of shape"):
        matrix_linear.linear_backward(dy, point, None, need_dx=False)
    with pytest.raises(ValueError, match="the residual has shape"):
        matrix_linear.linear(torch.randn(2, 4, 3, 3), w, None, torch.randn(5), channel_axis=1)
