"""Modules of joins and dropout in training: checkpointed, copied, in the forms that stacks of layers take."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import residual

import residual_oracle as ro

pytestmark = pytest.mark.gpu


def _grads(y, x, params):
    for v in [x] + params:
        v.grad = None
    y.square().sum().backward()
    return [v.grad for v in [x] + params]


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("counter", [False, True])
@pytest.mark.parametrize("per", ["element", "sample"])
def test_checkpointed_dropout(dev, host_layer, per, counter, reentrant):
    """The mask of a pass that is run again is that of its result, also with another pass between."""
    m = pkg.Dropout(0.4, per, seed=3, counter=counter).cuda()
    leaves = [(torch.rand(40, 3, 72, device=dev) + 1).requires_grad_() for _ in range(2)]
    ys = [checkpoint(lambda v: m(v * 2).exp(), x, use_reentrant=reentrant) for x in leaves]
    for i in (1, 0):
        ys[i].sum().backward()
        assert torch.equal(leaves[i].grad != 0, ys[i] != 1)
    assert not torch.equal(ys[0] != 1, ys[1] != 1) and (int(m.state[1]) if counter else m.calls) == 2


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("counter", [False, True])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
def test_checkpointed_stacks(dev, t, counter, reentrant):
    """Whole and block by block: results and gradients of the stack that is not checkpointed, bit for bit."""
    def make():
        torch.manual_seed(4)
        return pkg.ResidualStack([residual.matrix_block(72, 200, "silu") for _ in range(2)], 72, "rms", post=True, gate=0.5, drop=0.3, per="element", counter=counter).cuda().to(t)
    stack, plain = make(), make()
    for _ in range(3):
        x = torch.randn(4, 33, 72, device=dev).to(t).requires_grad_()
        y, want = checkpoint(stack, x, use_reentrant=reentrant), plain(x)
        assert torch.equal(y, want)
        got = _grads(y, x, list(stack.parameters()))
        for a, b in zip(got, _grads(want, x, list(plain.parameters()))):
            assert torch.equal(a, b)


def test_runs_again_that_cannot_be_told(dev):
    m = pkg.Dropout(0.4).cuda()
    x = torch.randn(6, 24, device=dev).requires_grad_()
    y = checkpoint(lambda v: m(v.sin()).exp(), x, use_reentrant=False, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match="run again in a backward pass"):
        y.sum().backward()


def test_stacks_of_layers_packed(dev):
    """A block that is a layer itself is served in 4 bits as the layers in other blocks are."""
    torch.manual_seed(5)
    layer = pkg.MatrixLinear(72, 72, activation="silu")
    stack = pkg.ResidualStack([layer, residual.matrix_block(72, 136), torch.nn.Sequential(layer, layer)], 72, "rms").cuda().eval()
    x = torch.randn(5, 72, device=dev)
    with torch.no_grad():
        for m in stack.blocks.modules():
            if isinstance(m, pkg.MatrixLinear):
                m.weight.copy_(pkg.packed4.unpack4(pkg.packed4.pack4(m.weight)))
        want = stack(x)
        got = stack.pack4()(x)
    # (the same values in 4 bits, fp32 sums of 72 and 136 products in another order)
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())
    assert isinstance(stack.blocks[0], pkg.MatrixLinear4) and stack.blocks[2][0] is stack.blocks[2][1] is stack.blocks[0]


@pytest.mark.parametrize("counter", [False, True])
def test_copies_draw_their_own_masks(dev, counter):
    """Blocks that are copies of one another, as stacks are often made."""
    torch.manual_seed(6)
    m = pkg.Dropout(0.5, counter=counter).cuda()
    x = torch.ones(50, 64, device=dev)
    layers = [m] + [copy.deepcopy(m) for _ in range(3)]
    masks = [layer(x) != 0 for layer in layers]
    for i in range(4):
        for j in range(i):
            # (800 of 3200, six deviations of 24.5)
            assert abs(int((masks[i] & masks[j]).sum()) - 800) < 147
    other = pkg.Dropout(0.5, counter=counter).cuda()
    other.load_state_dict(layers[2].state_dict())
    assert torch.equal(other(x), layers[2](x))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,C", [(5000, 4104), (17000, 523), (600, 70001)])
def test_masks_of_rows_in_pieces(dev, rows, C, t):
    """Joins without a norm, whose rows are taken in pieces by fewer workgroups than there are rows: the first, the middle and the last rows' masks bit for bit, all channels of them."""
    level, seed, offset = 16384, 11, 1 << 40 | 12
    f = torch.randn(rows, C, device=dev).to(t).abs() + 0.25
    x, drop = torch.randn(rows, C, device=dev).to(t), residual.Drop(0.25, seed, offset)
    out = residual.dropout_forward(f, drop)
    s = residual.join_forward(f, x, drop=drop, stream_scale=0.0)[0]
    df = residual.join_backward(f, None, None, None, None, drop=drop, need_stream=False).block
    for first in (0, 2047, rows // 2 + 1, rows - 6):
        first = min(first, rows - 6)
        kept = (ro.words(6, C, seed, offset, first)[:, :C] >= level).to(dev)
        for v in (out, s, df):
            assert torch.equal(v[first:first + 6] != 0, kept)
