"""Linear layers over the channels of a tensor - 1x1 convolutions of channel-last pixels, expanding and contracting layers, classifiers -
with bias, activation and residual in the epilogue of the product, and their gradients (the reference takes such layers from torch).

    z = x wT + bias (+ residual),   y = act(z) (+ residual)

act is one of "none", "relu", "gelu", "gelu_tanh" and "silu"; the residual stands before the activation, or behind it with
residual_after=True.  Sums and activations are fp32, y is rounded once.  In the gradients of an activation dz = dy act'(z) is rounded to
the type of the tensors before both products, which the matrix cores take: with 16-bit types and gelu or silu their error in the 2-norm is 1.4 times that
of an unrounded dz (bf16 0.0023 of 0.0017).  float32, float16 and bfloat16; tensors that are not contiguous
are copied first.  The GPU only.

A frozen weight may be in 4 bits (packed4.Packed4): x then meets its values in x's type, or, in 4 bits itself, its values as they are; gradients
pass through it to x, bias and residual.
"""
import ctypes

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, engine
from ._lib import LinearDesc, LinearGradients, check
from .checkpoint8 import Packed8, check_channels, pack8, pack_gates
from .packed4 import Packed4, _made as _made4, four_axes, linear4_ext, linear4_forward, pack4, settled as settled4

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation %r: one of %s" % (name, ", ".join(sorted(ACTIVATIONS))))
    return ACTIVATIONS[name]


def _check_weight(shape, w, what):
    if len(w.shape) != 2 or len(shape) < 1 or shape[-1] != w.shape[1] or not w.shape[0] or not w.shape[1]:
        raise ValueError("%s of shape %r and a weight of shape %r: expected (..., C) and (K, C), neither of them 0" % (what, tuple(shape), tuple(w.shape)))


def _check_like(t, shape, dtype, device, what):
    """Shape, type and device that the C ABI cannot see."""
    if t is None:
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %r, expected %r" % (what, tuple(t.shape), tuple(shape)))
    if t.dtype != dtype:
        raise TypeError("%s is %s, the layer's tensors are %s: they must share one dtype" % (what, t.dtype, dtype))
    if t.device != device:
        raise ValueError("%s is on %s, expected %s" % (what, t.device, device))


def _rows(shape):
    n = 1
    for v in shape[:-1]:
        n *= v
    return n


def _contiguous(t):
    """Contiguous and, for 16-byte loads, starting at a multiple of 16 bytes."""
    if t is None:
        return None
    t = t.detach().contiguous()
    return t.clone() if engine.misaligned(t) else t


def _desc(rows, C, K, dtype, activation, residual_after=False):
    return LinearDesc(rows, C, K, engine._DTYPES[dtype], activation, int(bool(residual_after)))


def linear_forward(x, w, bias=None, residual=None, activation="none", residual_after=False, keep_z=False):
    """y (..., K) for x (..., C) and w (K, C); with keep_z (y, z).  bias (K) and residual (..., K) of x's type, or None.  w may be a
    Packed4, and then x too, whose result is of the type that x reads as."""
    act = _activation(activation)
    if isinstance(w, Packed4) or isinstance(x, Packed4):
        return _linear4(x, w, bias, residual, activation, residual_after, keep_z)
    if engine.USE_EXT:
        y = engine._ext.linear_forward(x, w, bias, residual, act, bool(residual_after), bool(keep_z))
        if y is not None:
            return y
    _check_weight(x.shape, w, "x")
    K, C = w.shape
    check_channels(max(K, C), "linear_forward")
    shape = tuple(x.shape[:-1]) + (K,)
    _check_like(w, (K, C), x.dtype, x.device, "the weight")
    _check_like(bias, (K,), x.dtype, x.device, "the bias")
    _check_like(residual, shape, x.dtype, x.device, "the residual")
    engine._require_gpu(x, w, bias, residual)
    x, w, bias, residual = (_contiguous(t) for t in (x, w, bias, residual))
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if keep_z else None
    lib, d, nbytes = _lib.load(), _desc(_rows(shape), C, K, x.dtype, act, residual_after), ctypes.c_size_t()
    check(lib.wc_linear_workspace_bytes(ctypes.byref(d), ctypes.byref(nbytes)))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=x.device)
    with engine._on_device(x):
        p = engine._ptr
        check(lib.wc_linear_forward(ctypes.byref(d), p(x), p(w), p(bias), p(residual), p(y), p(z), p(ws), nbytes.value, engine._stream(x)))
    return (y, z) if keep_z else y


def _linear4(x, w, bias, residual, activation, residual_after, keep_z):
    """linear_forward over a Packed4 w."""
    if not isinstance(w, Packed4):
        raise TypeError("linear_forward: x in 4 bits takes a weight in 4 bits, got a tensor")
    y = linear4_ext(x, w, bias, residual, ACTIVATIONS[activation], residual_after, keep_z)
    if y is not None:
        return y
    _check_weight(x.shape, w, "x")
    K = w.shape[0]
    shape = tuple(x.shape[:-1]) + (K,)
    if keep_z and isinstance(x, Packed4):
        raise NotImplementedError("linear_forward: no z of an x in 4 bits, which has no gradient")
    _check_like(bias, (K,), x.dtype, x.device, "the bias")
    _check_like(residual, shape, x.dtype, x.device, "the residual")
    return linear4_forward(x, w, bias, residual, ACTIVATIONS[activation], residual_after, keep_z)


def linear_backward(dy, x, w, z=None, activation="none", need_dx=True, need_dw=True, need_db=True, need_dz=False, w_type=None, b_type=None):
    """(dx, dw, db, dz) of linear_forward, None for those not asked for, from dy (..., K), x (..., C), w (K, C) and, with an
    activation, z; x and z may be Packed8.  For relu anything with z's sign does, y among it where no residual stands behind the activation.
    dw and db come in `w_type` and `b_type` (x's type; float32 sums unrounded, of products with the rounded dz; db's are of dz before
    that).  relu's gradient is 0 at z = 0 and NaN where z is.  dz is the gradient of z and so of a residual before
    the activation; without an activation that is dy itself.  x may be None without need_dw, w without need_dx.  w may be a Packed4, whose values
    are read in dy's type."""
    act = _activation(activation)
    if isinstance(w, Packed4) and engine.USE_EXT and need_dx and not (need_dw or need_db or need_dz or isinstance(z, Packed8)):
        dx = engine._ext.linear4_backward(dy, w.codes, w.scales, w.channels, z, act)
        if dx is not None:
            return dx, None, None, None
    dtype, device = dy.dtype, dy.device
    if dy.dim() < 1 or not dy.shape[-1]:
        raise ValueError("dy of shape %r: expected (..., K)" % (tuple(dy.shape),))
    K, lead = dy.shape[-1], tuple(dy.shape[:-1])
    if (need_dx and w is None) or (need_dw and x is None):
        raise ValueError("linear_backward: dx needs w, dw needs x")
    for t, what in ((w, "w"), (x, "x")):
        if t is not None and len(t.shape) < 1:
            raise ValueError("%s of shape (): expected %s" % (what, "(K, C)" if what == "w" else "(..., C)"))
    C = w.shape[-1] if w is not None else x.shape[-1] if x is not None else 1
    check_channels(max(K, C), "linear_backward")
    if w is not None:
        _check_weight((C,), w, "x")
        _check_like(w, (K, C), w.dtype if isinstance(w, Packed4) else dtype, device, "the weight")
    if need_dw:
        if not C:
            raise ValueError("x of shape %r: expected (..., C)" % (tuple(x.shape),))
        _check_like(x, lead + (C,), dtype, device, "x")
    if act:
        if z is None:
            raise ValueError("linear_backward: the gradient of %r needs z" % activation)
        _check_like(z, tuple(dy.shape), dtype, device, "z")
    if not dy.is_cuda:
        raise ValueError("winoconv runs on the GPU only: got a %s tensor" % device)
    engine._require_gpu(dy)
    packed, w = (settled4(w) if need_dx else None, None) if isinstance(w, Packed4) else (None, w)
    w_type, b_type = w_type or dtype, b_type or dtype
    w_own, b_own = (t if t == torch.float32 else dtype for t in (w_type, b_type))
    if need_dz and not act:
        dz, need_dz = dy, False
    else:
        dz = None
    rows = _rows(dy.shape)
    new = lambda shape, t: torch.empty(shape, dtype=t, device=device)  # noqa: E731
    if rows == 0:
        return (new(lead + (C,), dtype) if need_dx else None, torch.zeros((K, C), dtype=w_type, device=device) if need_dw else None,
                torch.zeros(K, dtype=b_type, device=device) if need_db else None, torch.empty_like(dy) if need_dz else dz)
    x, z = x if need_dw else None, z if act else None
    if not (need_dx or need_dw or need_db or need_dz):
        return None, None, None, dz
    split = lambda t: (t.codes, t.exponents) if isinstance(t, Packed8) else (_contiguous(t), None)  # noqa: E731
    (x_data, x_exp), (z_data, z_exp) = split(x), split(z)
    if engine.USE_EXT:
        dx, dw, db, own_dz = engine._ext.linear_backward(dy, x_data, x_exp, w, z_data, z_exp, C, act, bool(need_dx), bool(need_dw), bool(need_db),
                                                         bool(need_dz), w_own, b_own, *((None, None) if packed is None else (packed.codes, packed.scales)))
    else:
        dy, w = _contiguous(dy), _contiguous(w)
        dx = new(lead + (C,), dtype) if need_dx else None
        dw = new((K, C), w_own) if need_dw else None
        db = new((K,), b_own) if need_db else None
        own_dz = new(lead + (K,), dtype) if need_dz else None
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        lib, d, nbytes = _lib.load(), _desc(rows, C, K, dtype, act), ctypes.c_size_t()
        g = LinearGradients(at(dy), at(x_data), at(x_exp), at(w), at(z_data), at(z_exp), at(dx), at(dw), engine._DTYPES[w_own], at(db),
                            engine._DTYPES[b_own], at(own_dz))
        name, w4 = ("wc_linear_backward", ()) if packed is None else ("wc_linear4_backward", (ctypes.byref(packed._pointers()),))
        check(getattr(lib, name + "_workspace_bytes")(ctypes.byref(d), ctypes.byref(g), ctypes.byref(nbytes)))
        ws = new((nbytes.value,), torch.uint8)
        with engine._on_device(dy):
            check(getattr(lib, name)(ctypes.byref(d), ctypes.byref(g), *w4, engine._ptr(ws), nbytes.value, engine._stream(dy)))
    return (dx, dw if dw is None or w_type == w_own else dw.to(w_type), db if db is None or b_type == b_own else db.to(b_type),
            dz if own_dz is None else own_dz)


def _check_checkpoint(checkpoint):
    if checkpoint not in (None, "int8"):
        raise ValueError("checkpoint %r: None or 'int8'" % (checkpoint,))


class LinearFunction(torch.autograd.Function):
    """linear_forward with gradients.  Parameters of another type than x's are cast for the products, and their gradients come back in
    theirs, float32 ones unrounded.  A Packed4 w has none."""

    @staticmethod
    def forward(ctx, x, w, bias, residual, activation, residual_after, checkpoint):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        ctx.types = (w.dtype, None if bias is None else bias.dtype)
        ctx.channels4 = w.channels if isinstance(w, Packed4) else None
        ctx.conf = (activation, residual_after, checkpoint is not None)
        own = lambda t: t if t is None or isinstance(t, Packed4) or t.dtype == x.dtype else t.to(x.dtype)  # noqa: E731
        w, bias = own(w), own(bias)
        slope = activation != "none" and (need_x or need_w or need_b or (need_r and not residual_after))
        by_sign = activation == "relu"
        z = None
        if slope and not (by_sign and not (residual_after and residual is not None)):
            y, z = linear_forward(x, w, bias, residual, activation, residual_after, keep_z=True)
        else:
            y = linear_forward(x, w, bias, residual, activation, residual_after)
            if slope:
                z = y
        kept = [None if not need_w else x, None if not need_x else w, z]
        if checkpoint is not None:
            packed = [None if t is None else pack(t) for t, pack in ((kept[0], pack8), (z, pack_gates if by_sign else pack8))]
            kept = [packed[0] and packed[0].codes, kept[1], packed[1] and packed[1].codes, packed[0] and packed[0].exponents, packed[1] and packed[1].exponents]
        if ctx.channels4 is not None:
            kept[1:2] = [None, None] if kept[1] is None else [kept[1].codes, kept[1].scales]
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        activation, residual_after, packed = ctx.conf
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        kept = list(ctx.saved_tensors)
        if ctx.channels4 is not None:
            kept[1:3] = [None if kept[1] is None else _made4(kept[1], kept[2], ctx.channels4, dy.dtype)]
        x, w, z = kept[:3]
        if packed:
            x_exp, z_exp = kept[3:]
            x, z = (None if c is None else Packed8(c, e, dy.dtype) for c, e in ((x, x_exp), (z, z_exp)))
        w_type, b_type = ctx.types
        dx, dw, db, dz = linear_backward(dy, x, w, z, activation, need_x, need_w, need_b, need_r and not residual_after, w_type, b_type)
        return dx, dw, db, dy if need_r and residual_after else dz, None, None, None


def _refuse_tangents(given):
    # (asked of torch for each tensor only within a level of forward mode: 3 us)
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise NotImplementedError("linear has no forward-mode derivative: a tangent of its operands would be lost")


def linear(x, w, bias=None, residual=None, activation="none", residual_after=False, checkpoint=None, channel_axis=-1):
    """linear_forward with gradients.  checkpoint="int8" keeps x and z in 8 bits for the backward pass (checkpoint8); relu's gate
    stays z's own, so that of its gradients the weight's alone differs.  channel_axis: the axis of the channels in x and the residual, so that 1 takes the (N, C, H, W) tensors of the convolutions; a
    tensor in channel-last memory is used as it is, and the result is one.  Reverse mode, once: operands with a forward-mode tangent are refused.
    w may be a Packed4, through which gradients pass to x, bias and residual; with an x in 4 bits too there are none."""
    _check_checkpoint(checkpoint)
    _activation(activation)
    if isinstance(x, Packed4):
        if channel_axis not in (-1, len(x.shape) - 1):
            raise ValueError("linear: channel_axis %r of an x in 4 bits, whose channels are last" % (channel_axis,))
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (bias, residual)):
            raise NotImplementedError("linear: no gradient passes a layer whose x is in 4 bits")
        _refuse_tangents((bias, residual))
        return linear_forward(x, w, bias, residual, activation, residual_after)
    if channel_axis not in (-1, x.dim() - 1):
        if residual is not None and residual.dim() != x.dim():
            raise ValueError("the residual has shape %r, expected that of the result: %d axes" % (tuple(residual.shape), x.dim()))
        x = x.movedim(channel_axis, -1)
        residual = None if residual is None else residual.movedim(channel_axis, -1)
        return linear(x, w, bias, residual, activation, residual_after, checkpoint).movedim(-1, channel_axis)
    given = [t for t in (x, w, bias, residual) if t is not None and not isinstance(t, Packed4)]
    _refuse_tangents(given)
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        return LinearFunction.apply(x, w, bias, residual, activation, bool(residual_after), checkpoint)
    own = lambda t: t if t is None or isinstance(t, Packed4) or t.dtype == x.dtype else t.to(x.dtype)  # noqa: E731
    return linear_forward(x, own(w), own(bias), residual, activation, residual_after)


class MatrixLinear(nn.Module):
    """nn.Linear with activation and residual in one kernel, beside WinoConv2d / WinoConv3d: forward(x, residual=None).  With
    channel_axis=1 it is their 1x1 convolution, on the same (N, C, [D,] H, W) tensors.  A pass may be captured into a graph; as with every torch
    module, no eager autograd graph of the same parameters may be alive while a backward pass is captured."""

    def __init__(self, in_features, out_features, bias=True, activation="none", residual_after=False, checkpoint=None, channel_axis=-1,
                 device=None, dtype=None):
        super().__init__()
        _activation(activation)
        _check_checkpoint(checkpoint)
        self.in_features, self.out_features = in_features, out_features
        self.activation, self.residual_after, self.checkpoint, self.channel_axis = activation, residual_after, checkpoint, channel_axis
        self.weight = nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.empty(out_features, device=device, dtype=dtype)) if bias else None
        nn.init.kaiming_normal_(self.weight)
        if self.bias is not None:
            nn.init.zeros_(self.bias)

    def forward(self, x, residual=None):
        return linear(x, self.weight, self.bias, residual, self.activation, self.residual_after, self.checkpoint, self.channel_axis)

    def extra_repr(self):
        return "%d, %d, bias=%s, activation=%r" % (self.in_features, self.out_features, self.bias is not None, self.activation)

    def pack4(self, x4=False):
        """This layer for serving or behind trained ones: a MatrixLinear4 whose weight is this one's in 4 bits.  x4: its inputs are put into 4
        bits too, which many rows take to the matrix cores' 4-bit rate; gradients do not pass it then."""
        layer = MatrixLinear4.__new__(MatrixLinear4)
        nn.Module.__init__(layer)
        w4 = pack4(self.weight)
        layer._hold(w4, self.bias, self.activation, self.residual_after, self.channel_axis, x4, self.checkpoint)
        return layer


class MatrixLinear4(nn.Module):
    """A linear layer whose weight is frozen, in 4 bits (MatrixLinear.pack4, or of a Packed4 w (out_features, in_features)): 1/2 + 1/32 bytes a
    weight, which is what a layer of few rows reads.  The weight is in the buffers `codes` and `scales` (with one axis for a stage's 32 rows and 4 groups: of a
    buffer of four axes Module.to(memory_format=...) would change the strides); the bias is a parameter, which with x4 does not learn either.  checkpoint: as
    MatrixLinear's, of z."""

    checkpoint = None                        # (of layers that were saved whole before they had one)

    def __init__(self, weight, bias=None, activation="none", residual_after=False, channel_axis=-1, x4=False, checkpoint=None):
        super().__init__()
        _activation(activation)
        _check_checkpoint(checkpoint)
        if not isinstance(weight, Packed4) or len(weight.shape) != 2:
            raise TypeError("MatrixLinear4: the weight is a Packed4 of two axes")
        self._hold(weight, bias, activation, residual_after, channel_axis, x4, checkpoint)

    def _hold(self, w4, bias, activation, residual_after, channel_axis, x4, checkpoint):
        self.out_features, self.in_features = w4.shape
        self.activation, self.residual_after, self.channel_axis, self.x4, self.checkpoint = activation, residual_after, channel_axis, bool(x4), checkpoint
        self.dtype = w4.dtype
        self.register_buffer("codes", w4.codes)
        self.register_buffer("scales", w4.scales.flatten(2))
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone(), requires_grad=bias.requires_grad and not x4)

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        # (a Packed4's own scales, of four axes)
        scales = state_dict.get(prefix + "scales")
        if isinstance(scales, torch.Tensor) and scales.dim() == 4:
            state_dict[prefix + "scales"] = scales.flatten(2)
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    @property
    def weight(self):
        """The Packed4 of the buffers as they are now."""
        return Packed4(self.codes, four_axes(self.scales), self.in_features, self.dtype)

    def forward(self, x, residual=None):
        # (the kernels read the scales whatever their axes; where the buffers do not lie as they read them, the calls copy)
        w = _made4(self.codes, self.scales, self.in_features, self.dtype)
        if not self.x4:
            return linear(x, w, self.bias, residual, self.activation, self.residual_after, self.checkpoint, self.channel_axis)
        if torch.is_grad_enabled() and x.requires_grad:
            raise NotImplementedError("MatrixLinear4: no gradient passes a layer that puts its inputs into 4 bits")
        _refuse_tangents((x,))
        axis = self.channel_axis
        if axis not in (-1, x.dim() - 1):
            return self._last(x.movedim(axis, -1), w, None if residual is None else residual.movedim(axis, -1)).movedim(-1, axis)
        return self._last(x, w, residual)

    def _last(self, x, w, residual):
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        return linear(pack4(x), w, bias, residual, self.activation, self.residual_after)

    def extra_repr(self):
        return "%d, %d, bias=%s, activation=%r, x4=%r" % (self.in_features, self.out_features, self.bias is not None, self.activation, self.x4)
