"""What a MatrixLinear4 keeps of its weight when its module is moved, saved and loaded; on the CPU, where the layer's kernels are not reached."""
import copy
import io

import pytest
import torch
from torch.autograd import forward_ad

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import matrix_linear, packed4
from pytorch_winoconv_amd.packed4 import Packed4

import packed4_oracle as po


def _packed(rows=70, C=300, t=torch.bfloat16):
    return Packed4.from_parts(*po.pack(torch.randn(rows, C)), C, t)


def _taken(layer, monkeypatch):
    """The weight that the layer's forward pass hands to its kernel."""
    seen = []
    monkeypatch.setattr(matrix_linear, "linear", lambda x, w, *_, **__: seen.append(w))
    layer(torch.zeros(2, layer.in_features))
    monkeypatch.undo()
    w = packed4.settled(seen[0])
    return Packed4(w.codes, packed4.four_axes(w.scales), w.channels, w.dtype)


def _same(a, b):
    return a.shape == b.shape and torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and a.codes.is_contiguous() and a.scales.is_contiguous()


@pytest.mark.parametrize("memory_format", [torch.channels_last, torch.channels_last_3d, torch.preserve_format], ids=str)
def test_memory_formats(monkeypatch, memory_format):
    """The layouts of convolutions' tensors are none of the scales'."""
    w = _packed()
    layer = pkg.MatrixLinear4(w, torch.randn(70), channel_axis=1)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 300, 3) if memory_format is not torch.channels_last_3d else torch.nn.Conv3d(3, 300, 3), layer)
    model.to(memory_format=memory_format)
    assert layer.codes.is_contiguous() and layer.scales.is_contiguous()
    assert _same(layer.weight, w) and _same(_taken(layer, monkeypatch), w)


def test_state_dicts(monkeypatch):
    """Into another layer, by copy and by assignment, also of scales with an axis each for rows and groups, in any memory order."""
    w = _packed()
    state = pkg.MatrixLinear4(w).state_dict()
    for assign in (False, True):
        for scales in (state["scales"], w.scales, w.scales.to(memory_format=torch.channels_last), torch.zeros(w.scales.numel() + 1, dtype=torch.uint8)[1:].view(w.scales.shape).copy_(w.scales)):
            given = {"codes": state["codes"], "scales": scales}
            other = pkg.MatrixLinear4(_packed())
            other.load_state_dict(given, assign=assign)
            assert given["scales"] is scales
            assert _same(other.weight, w) and _same(_taken(other, monkeypatch), w)
    with pytest.raises(RuntimeError, match="size mismatch"):
        pkg.MatrixLinear4(_packed(70, 500)).load_state_dict(state)


def test_copies(monkeypatch):
    w = _packed()
    layer = pkg.MatrixLinear4(w)
    buffer = io.BytesIO()
    torch.save(layer.state_dict(), buffer)
    buffer.seek(0)
    loaded = pkg.MatrixLinear4(_packed())
    loaded.load_state_dict(torch.load(buffer, weights_only=True))
    for other in (copy.deepcopy(layer), copy.deepcopy(layer).half(), loaded):
        assert _same(_taken(other, monkeypatch), w)


def test_parts_that_lie_otherwise():
    """A tensor in 4 bits whose parts were replaced: copied where they lie otherwise, refused where they are not its."""
    w = _packed()
    assert packed4.settled(w) is w
    odd = torch.zeros(w.codes.numel() + 1, dtype=torch.uint8)[1:].view(w.codes.shape).copy_(w.codes)
    for codes, scales in ((w.codes.t().contiguous().t(), w.scales), (odd, w.scales), (w.codes, w.scales.to(memory_format=torch.channels_last)),
                          (w.codes, w.scales.transpose(1, 2).contiguous().transpose(1, 2))):
        other = Packed4(w.codes, w.scales, 300, torch.bfloat16)
        other.codes, other.scales = codes, scales
        assert _same(packed4.settled(other), w)
    for codes, scales in ((w.codes[:40], w.scales), (w.codes, w.scales[:1]), (w.codes[:, :64], w.scales)):
        other = Packed4(w.codes, w.scales, 300, torch.bfloat16)
        other.codes, other.scales = codes, scales
        with pytest.raises(ValueError, match="Packed4: codes of shape"):
            packed4.settled(other)


def test_checkpoints_are_kept(monkeypatch):
    """A layer that keeps z in 8 bits does so with its weight in 4."""
    monkeypatch.setattr(matrix_linear, "pack4", lambda w: Packed4.from_parts(*po.pack(w.detach()), w.shape[1], w.dtype))
    seen = []
    for checkpoint in (None, "int8"):
        layer = pkg.MatrixLinear(40, 72, activation="gelu", checkpoint=checkpoint)
        for four in (layer.pack4(), copy.deepcopy(layer.pack4()), pkg.MatrixLinear4(layer.pack4().weight, layer.bias, "gelu", checkpoint=checkpoint)):
            assert four.checkpoint == checkpoint
            with monkeypatch.context() as m:
                m.setattr(matrix_linear, "linear", lambda x, w, b, r, act, after, kept, axis: seen.append(kept))
                four(torch.zeros(3, 40))
            assert seen.pop() == checkpoint
    with pytest.raises(ValueError, match="checkpoint"):
        pkg.MatrixLinear4(_packed(), checkpoint="fp8")
    stack = pkg.ResidualStack([pkg.residual.matrix_block(40, 64, checkpoint="int8")], 40).pack4()
    assert [m.checkpoint for m in stack.blocks[0]] == ["int8", "int8"]


@pytest.mark.parametrize("which", ["x", "bias", "residual"])
def test_forward_mode_is_refused(monkeypatch, which):
    """Also where x is in 4 bits, or put into them by the layer: a tangent would be lost."""
    monkeypatch.setattr(matrix_linear, "pack4", lambda x: Packed4.from_parts(*po.pack(x.detach()), x.shape[1], x.dtype))
    w = _packed(70, 300, torch.float32)
    layer = pkg.MatrixLinear4(w, torch.zeros(70), x4=True)
    with forward_ad.dual_level():
        ts = {"x": torch.randn(3, 300), "bias": torch.zeros(70), "residual": torch.zeros(3, 70)}
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                if which != "bias":
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        layer(ts["x"], ts["residual"])
                if which != "x":
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        matrix_linear.linear(_packed(3, 300, torch.float32), w, ts["bias"], ts["residual"])
