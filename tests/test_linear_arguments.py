"""Arguments of linear layers and 8 bits that the C ABI could not tell apart from others, refused on the CPU before any launch."""
import pytest
import torch

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
