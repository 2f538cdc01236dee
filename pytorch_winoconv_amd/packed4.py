"""Tensors in microscaled 4-bit floating point, the OCP formats' MXFP4, for the weights (and activations) of linear layers (the reference has
neither).

The groups of 32 neighbouring channels (the last axis) share a scale 2^e, e = floor(log2(largest magnitude)) - 2 but at least -127; a value is
kept as the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times the scale, ties to the even code, at most 6 of it.  It is off by at most a
quarter of itself, or a quarter of the scale where that is more.  Groups with an infinity or a NaN read as NaN.  Memory: 1/2 + 1/32 bytes a
value.  matrix_linear.linear_forward, linear and MatrixLinear4 take such weights; a tensor reads in any of the engine's types, rounded where
that type does not hold its values (float16 below 2^-24 and above 65504).
"""
import ctypes

import torch

from . import _lib, engine
from ._lib import Packed4Parts, check

GROUP, STAGE, ROWS = 32, 128, 32
MOST_CHANNELS = 1 << 22


def check_channels(n, who):
    """What offsets within a tile's rows allow; the C ABI takes channels as an int."""
    if n > MOST_CHANNELS:
        raise ValueError("%s: %d channels, at most 2^22" % (who, n))


def _rows(shape):
    n = 1
    for v in shape[:-1]:
        n *= v
    return n


class Packed4:
    """A tensor of `shape` in 4 bits.  Its rows are padded to whole stages of 128 channels, S of them: `codes` uint8 of its shape with 64 S bytes in
    the place of its channels, the lower channel in a byte's low half; `scales` uint8 (ceil(rows / 32), S, 32, 4), e + 127, the order
    in which the product reads them; zeros in either's padding.  `dtype` is the type that it reads as where no other is asked for."""

    __slots__ = ("codes", "scales", "channels", "dtype")

    def __init__(self, codes, scales, channels, dtype):
        if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor) or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("Packed4: codes and scales are uint8 tensors")
        if dtype not in engine._DTYPES:
            raise TypeError("winoconv supports float32, float16 and bfloat16, got %s" % dtype)
        channels = int(channels)
        check_channels(channels, "Packed4")
        stages = -(-channels // STAGE)
        if codes.dim() < 1 or channels < 1 or codes.shape[-1] != 64 * stages or tuple(scales.shape) != (-(-_rows(codes.shape) // ROWS), stages, ROWS, 4):
            raise ValueError("Packed4: codes of shape %r and scales of shape %r for %d channels: expected (..., %d) and (ceil(rows / 32), %d, 32, 4)"
                             % (tuple(codes.shape), tuple(scales.shape), channels, 64 * stages, stages))
        if codes.device != scales.device:
            raise ValueError("Packed4: codes are on %s, scales on %s" % (codes.device, scales.device))
        self.codes, self.scales = (t.clone() if engine.misaligned(t) else t for t in (codes.detach().contiguous(), scales.detach().contiguous()))
        self.channels, self.dtype = channels, dtype

    @classmethod
    def from_parts(cls, codes, scales, channels, dtype):
        """From the plain order of checkpoints: codes uint8 (..., ceil(C / 2)), two to a byte, and scales uint8 (..., ceil(C / 32)), e + 127."""
        channels = int(channels)
        check_channels(channels, "Packed4.from_parts")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("Packed4.from_parts: codes and scales are uint8, got %s and %s" % (codes.dtype, scales.dtype))
        lead, groups = tuple(codes.shape[:-1]), -(-channels // GROUP)
        if codes.dim() < 1 or channels < 1 or codes.shape[-1] != -(-channels // 2) or tuple(scales.shape) != lead + (groups,):
            raise ValueError("Packed4.from_parts: codes of shape %r and scales of shape %r for %d channels: expected (..., %d) and (..., %d)"
                             % (tuple(codes.shape), tuple(scales.shape), channels, -(-channels // 2), groups))
        stages, rows = -(-channels // STAGE), _rows(codes.shape)
        blocks = -(-rows // ROWS)
        wide = torch.zeros(lead + (64 * stages,), dtype=torch.uint8, device=codes.device)
        wide[..., :codes.shape[-1]] = codes
        if channels % 2:
            wide[..., channels // 2] &= 15
        tiled = torch.zeros(blocks * ROWS, stages * 4, dtype=torch.uint8, device=codes.device)
        tiled[:rows, :groups] = scales.reshape(rows, groups)
        return cls(wide, tiled.view(blocks, ROWS, stages, 4).permute(0, 2, 1, 3), channels, dtype)

    def parts(self):
        """(codes, scales) in the plain order that from_parts takes."""
        rows, groups = _rows(self.codes.shape), -(-self.channels // GROUP)
        blocks, stages = self.scales.shape[:2]
        scales = self.scales.permute(0, 2, 1, 3).reshape(blocks * ROWS, stages * 4)[:rows, :groups]
        return self.codes[..., :-(-self.channels // 2)].contiguous(), scales.reshape(tuple(self.codes.shape[:-1]) + (groups,)).contiguous()

    @property
    def shape(self):
        return torch.Size(tuple(self.codes.shape[:-1]) + (self.channels,))

    @property
    def device(self):
        return self.codes.device

    def _pointers(self):
        return Packed4Parts(self.codes.data_ptr(), self.scales.data_ptr())


def _made(codes, scales, channels, dtype):
    """A Packed4 of parts that belong together."""
    p = Packed4.__new__(Packed4)
    p.codes, p.scales, p.channels, p.dtype = codes, scales, channels, dtype
    return p


def four_axes(scales):
    """The scales of a Packed4, of which a module's buffer has the last two axes in one."""
    return scales.unflatten(2, (ROWS, 4)) if scales.dim() == 3 else scales


def _belong(p):
    """Whether codes and scales lie as the kernels read them: whole, one after the other, from multiples of 16 bytes."""
    codes, scales = p.codes, p.scales
    if engine.USE_EXT and codes.is_cuda:
        return engine._ext.packed4_fits(codes, scales, p.channels)
    stages = -(-p.channels // STAGE)
    return (codes.is_contiguous() and scales.is_contiguous() and not engine.misaligned(codes, scales) and codes.dtype == scales.dtype == torch.uint8
            and codes.device == scales.device and codes.shape[-1] == 64 * stages and scales.numel() == -(-_rows(codes.shape) // ROWS) * stages * ROWS * 4)


def settled(p):
    """A Packed4 whose parts the kernels may read: p as it is, or its parts copied where they lie otherwise (a module's buffers take other strides and starts
    when it is moved or loaded); parts that are not each other's are refused."""
    return p if _belong(p) else Packed4(p.codes, four_axes(p.scales), p.channels, p.dtype)


def pack4(x):
    """x (..., C) in 4 bits."""
    if engine.USE_EXT:
        parts = engine._ext.pack4(x)
        if parts is not None:
            return _made(*parts, x.shape[-1], x.dtype)
    if x.dim() < 1 or not x.shape[-1]:
        raise ValueError("pack4: a tensor of shape %r: expected (..., C), C not 0" % (tuple(x.shape),))
    check_channels(x.shape[-1], "pack4")
    engine._require_gpu(x)
    x = x.detach().contiguous()
    C, rows = x.shape[-1], _rows(x.shape)
    stages = -(-C // STAGE)
    new = lambda shape: torch.empty(shape, dtype=torch.uint8, device=x.device)  # noqa: E731
    codes, scales = new(tuple(x.shape[:-1]) + (64 * stages,)), new((-(-rows // ROWS), stages, ROWS, 4))
    if rows:
        with engine._on_device(x):
            check(_lib.load().wc_pack4(engine._ptr(x), engine._ptr(codes), engine._ptr(scales), rows, C, engine._DTYPES[x.dtype], engine._stream(x)))
    return _made(codes, scales, C, x.dtype)


def unpack4(packed, dtype=None):
    """The tensor that a Packed4 stands for, contiguous, in its type or in `dtype`."""
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in engine._DTYPES:
        raise TypeError("winoconv supports float32, float16 and bfloat16, got %s" % dtype)
    if not packed.codes.is_cuda:
        raise ValueError("winoconv runs on the GPU only: got a %s tensor" % packed.device)
    packed = settled(packed)
    if engine.USE_EXT and packed.codes.numel():
        return engine._ext.unpack4(packed.codes, packed.scales, packed.channels, dtype)
    x = torch.empty(packed.shape, dtype=dtype, device=packed.device)
    if x.numel():
        with engine._on_device(x):
            check(_lib.load().wc_unpack4(engine._ptr(packed.codes), engine._ptr(packed.scales), engine._ptr(x), _rows(x.shape), packed.channels,
                                         engine._DTYPES[dtype], engine._stream(x)))
    return x


def linear4_ext(x, w, bias, residual, activation, residual_after, keep_z=False):
    """linear4_forward by the compiled host layer, which takes operands that fit together and lie as the kernels read them; None for others."""
    if not engine.USE_EXT or not w.codes.is_cuda or w.codes.dim() != 2:
        return None
    if not isinstance(x, Packed4):
        return engine._ext.linear4_forward(x, None, None, None, w.codes, w.scales, w.channels, bias, residual, activation, bool(residual_after), bool(keep_z))
    if keep_z or x.channels != w.channels:
        return None
    return engine._ext.linear4_forward(None, x.codes, x.scales, x.dtype, w.codes, w.scales, w.channels, bias, residual, activation, bool(residual_after), False)


def linear4_forward(x, w, bias, residual, activation, residual_after, keep_z=False):
    """matrix_linear.linear_forward for w a Packed4 (K, C) and x a tensor (..., C) or, without z, a Packed4; activation is its number."""
    y = linear4_ext(x, w, bias, residual, activation, residual_after, keep_z)
    if y is not None:
        return y
    packed, w = isinstance(x, Packed4), settled(w)
    x, C = settled(x) if packed else x, w.channels
    K, shape, dtype = w.codes.shape[0], tuple(x.shape[:-1]) + (w.codes.shape[0],), x.dtype
    if packed:
        if not x.codes.is_cuda:
            raise ValueError("winoconv runs on the GPU only: got a %s tensor" % x.device)
        engine._require_gpu(bias, residual)
    else:
        engine._require_gpu(x, bias, residual)
    if w.device != x.device:
        raise ValueError("the weight is on %s, expected %s" % (w.device, x.device))
    y = torch.empty(shape, dtype=dtype, device=x.device)
    z = torch.empty_like(y) if keep_z else None
    rows = _rows(shape)
    own = lambda t: t.clone() if engine.misaligned(t) else t  # noqa: E731
    x_, bias, residual = (None if t is None else own(t.detach().contiguous()) for t in (None if packed else x, bias, residual))
    lib, nbytes = _lib.load(), ctypes.c_size_t()
    d = _lib.LinearDesc(rows, C, K, engine._DTYPES[dtype], activation, int(bool(residual_after)))
    check(lib.wc_linear4_workspace_bytes(ctypes.byref(d), int(packed), ctypes.byref(nbytes)))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=x.device)
    w4, x4 = w._pointers(), x._pointers() if packed else None
    with engine._on_device(y):
        p = engine._ptr
        check(lib.wc_linear4_forward(ctypes.byref(d), p(x_), ctypes.byref(x4) if packed else None, ctypes.byref(w4), p(bias), p(residual), p(y), p(z), p(ws),
                                     nbytes.value, engine._stream(y)))
    return (y, z) if keep_z else y
