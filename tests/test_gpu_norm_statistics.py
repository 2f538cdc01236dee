"""Values that the backward pass normalises are those of the forward pass, where the mean is many deviations too."""
import pytest
import torch

from pytorch_winoconv_amd import residual
from pytorch_winoconv_amd.residual import Drop, Norm

pytestmark = pytest.mark.gpu

# a team of one lane, of several, of wavefronts, two vectors a thread, rows that registers do not hold, even and odd
CHANNELS = [8, 5, 100, 333, 1000, 2056, 4097, 8192, 12001, 16384, 20000]


def _row(C, mean, deviation):
    g = torch.Generator().manual_seed(C)
    return torch.randn(1, C, generator=g) * deviation + mean


def _normalised(v, stats):
    """By the mean and the inverse deviation that the forward pass kept: a difference and a product, either rounded."""
    return (v.float() - stats[0, 0]) * stats[0, 1]


@pytest.mark.parametrize("C", CHANNELS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_alone(dev, host_layer, kind, C):
    """dw of one row and dy = 1 is the normalised row itself, y without parameters: bit for bit in float32, since either rounds a difference and a product."""
    for mean, deviation in ((0, 1), (10, 1), (1000, 1), (100, 0), (-3e4, 1e-2)):
        x = _row(C, mean, deviation).cuda()
        y, stats = residual.norm_forward(x, Norm(kind), keep=True)
        n = Norm(kind, torch.ones(C, device=dev))
        dw = residual.norm_backward(torch.ones_like(x), x, stats, n, need_dx=False)[1]
        assert torch.equal(dw, y[0]) and torch.equal(y, _normalised(x, stats)), (mean, deviation)
        if deviation == 0 and kind == "layer":
            assert not bool(dw.any())


@pytest.mark.parametrize("C", CHANNELS)
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_norm_behind_a_block(dev, t, C):
    """The same of post: its dw is the normalised block."""
    for mean, deviation in ((0, 1), (10, 1), (1000, 1), (100, 0)):
        f = _row(C, mean, deviation).cuda().to(t)
        w = Norm("layer", torch.ones(C, device=dev))
        s, _, stats = residual.join_forward(f, None, post=w, keep=True)
        got = residual.join_backward(torch.ones_like(f), None, f, s, stats, post=w, need_block=False, need_stream=False)
        assert got.post_weight.dtype == torch.float32 and torch.equal(got.post_weight, _normalised(f, stats[0])[0]), (mean, deviation)


@pytest.mark.parametrize("C", CHANNELS)
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16], ids=str)
def test_norm_of_s_computed_again(dev, t, C):
    """Of 16-bit types pre's dw is by s as it was before its rounding: of a stream alone, whose block is dropped, the stream's own."""
    x = _row(C, 100, 1).cuda().to(t)
    f, w, drop = torch.full_like(x, 7), Norm("layer", torch.ones(C, device=dev)), Drop(1.0, 1)
    s, _, stats = residual.join_forward(f, x, pre=w, drop=drop, keep=True)
    got = residual.join_backward(None, torch.ones_like(f), f, s, stats, pre=w, drop=drop, need_block=False, need_stream=False)
    assert torch.equal(got.pre_weight, _normalised(x, stats[1])[0])
