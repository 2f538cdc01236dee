"""Activations in 8 bits between the forward and the backward pass (the reference has neither).

The groups of 32 neighbouring channels (the last axis) share a step 2^e, e = floor(log2(largest magnitude)) - 6 but at least -126;
a value is kept as the nearest whole number of steps, ties to even, at most 127 either way, and reads as that number times the step, which
every type it came from holds exactly.  It is off by at most 2^-7 of its group's largest, or 2^-127 where that is more.  Groups with an infinity or a NaN read as NaN.
Memory: 1 + 1/32 bytes a value.  WinoConv2d / WinoConv3d and MatrixLinear keep their inputs so with checkpoint="int8".
"""
import ctypes

import torch

from . import _lib, engine
from ._lib import check

GROUP = 32


def check_channels(n, who):
    """The C ABI takes channels as an int, which ctypes would cut to 32 bits."""
    if n > 1 << 24:
        raise ValueError("%s: %d channels, at most 2^24" % (who, n))


class Packed8:
    """A tensor in 8 bits: `codes` int8 of its shape, `exponents` int8 of its shape with ceil(C / 32) groups in the place of
    its C channels, both contiguous, and the type that it reads as."""

    __slots__ = ("codes", "exponents", "dtype")

    def __init__(self, codes, exponents, dtype):
        if codes.dtype != torch.int8 or exponents.dtype != torch.int8:
            raise TypeError("Packed8: codes and exponents are int8, got %s and %s" % (codes.dtype, exponents.dtype))
        if dtype not in engine._DTYPES:
            raise TypeError("winoconv supports float32, float16 and bfloat16, got %s" % dtype)
        if codes.dim() < 1 or tuple(exponents.shape) != tuple(codes.shape[:-1]) + ((codes.shape[-1] + GROUP - 1) // GROUP,):
            raise ValueError("Packed8: codes of shape %r need exponents for groups of %d channels, got shape %r"
                             % (tuple(codes.shape), GROUP, tuple(exponents.shape)))
        if codes.device != exponents.device:
            raise ValueError("Packed8: codes are on %s, exponents on %s" % (codes.device, exponents.device))
        self.codes, self.exponents, self.dtype = codes.contiguous(), exponents.contiguous(), dtype

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device


def _made(codes, exponents, dtype):
    """A Packed8 of parts that belong together."""
    p = Packed8.__new__(Packed8)
    p.codes, p.exponents, p.dtype = codes, exponents, dtype
    return p


def pack8(x, keep_sign=False):
    """x (..., C) in 8 bits.  `keep_sign`: values other than zero keep a code other than zero (one step), for tensors that are read by
    their sign alone, as a ReLU's gradient reads them."""
    return _pack(x, int(bool(keep_sign)))


def pack_gates(z):
    """z in 8 bits for the gradient of a ReLU and nothing else: pack8 with `keep_sign`, and in groups with an infinity or a NaN the other channels
    keep their gates too."""
    return _pack(z, 2)


def _pack(x, keep_sign):
    if engine.USE_EXT:
        parts = engine._ext.pack8(x, keep_sign)
        if parts is not None:
            return _made(*parts, x.dtype)
    if x.dim() < 1:
        raise ValueError("pack8: a tensor of at least one axis, its channels last")
    check_channels(x.shape[-1], "pack8")
    engine._require_gpu(x)
    x = x.detach().contiguous()
    C = x.shape[-1]
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    exponents = torch.empty(tuple(x.shape[:-1]) + ((C + GROUP - 1) // GROUP,), dtype=torch.int8, device=x.device)
    if x.numel():
        with engine._on_device(x):
            check(_lib.load().wc_pack8(engine._ptr(x), engine._ptr(codes), engine._ptr(exponents), x.numel() // C, C, engine._DTYPES[x.dtype],
                                       keep_sign, engine._stream(x)))
    return Packed8(codes, exponents, x.dtype)


def unpack8(packed):
    """The tensor that a Packed8 stands for, contiguous, in its type."""
    check_channels(packed.shape[-1], "unpack8")
    if not packed.codes.is_cuda:
        raise ValueError("winoconv runs on the GPU only: got a %s tensor" % packed.device)
    if engine.USE_EXT:
        x = engine._ext.unpack8(packed.codes, packed.exponents, packed.dtype)
        if x is not None:
            return x
    x = torch.empty(packed.shape, dtype=packed.dtype, device=packed.device)
    if x.numel():
        C = x.shape[-1]
        with engine._on_device(x):
            check(_lib.load().wc_unpack8(engine._ptr(packed.codes), engine._ptr(packed.exponents), engine._ptr(x), x.numel() // C, C,
                                         engine._DTYPES[x.dtype], engine._stream(x)))
    return x
