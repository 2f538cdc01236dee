"""Arguments of tensors in 4 bits that do not fit together, refused on the CPU before any launch."""
import ctypes

import pytest
import torch

from pytorch_winoconv_amd import _lib, matrix_linear, packed4
from pytorch_winoconv_amd.packed4 import Packed4

import packed4_oracle as po


def _packed(rows=5, C=200, t=torch.bfloat16):
    return Packed4.from_parts(*po.pack(torch.randn(rows, C)), C, t)


def test_parts_there_and_back():
    for rows, C in [(1, 1), (5, 33), (32, 128), (33, 129), (70, 1000)]:
        codes, scales = po.pack(torch.randn(rows, C))
        p = Packed4.from_parts(codes, scales, C, torch.float16)
        assert p.shape == (rows, C) and p.codes.shape == (rows, (C + 127) // 128 * 64)
        got = p.parts()
        assert torch.equal(got[0], codes) and torch.equal(got[1], scales)
        # what lies behind the channels and rows is zero, also where the given byte's other half is not
        if C % 2:
            codes[:, -1] |= 0xf0
            assert torch.equal(Packed4.from_parts(codes, scales, C, torch.float16).codes, p.codes)
        assert int(p.codes[:, (C + 1) // 2:].sum()) == 0


def test_parts_that_do_not_fit():
    codes, scales = po.pack(torch.randn(5, 200))
    for c, s, n in [(codes, scales, 202), (codes, scales[:, :-1], 200), (codes[:-1], scales, 200), (codes, scales, 0), (codes[0, 0], scales, 1)]:
        with pytest.raises(ValueError, match="Packed4.from_parts"):
            Packed4.from_parts(c, s, n, torch.float16)
    with pytest.raises(TypeError, match="uint8"):
        Packed4.from_parts(codes.to(torch.int8), scales, 200, torch.float16)
    p = _packed()
    with pytest.raises(TypeError, match="uint8"):
        Packed4(p.codes.int(), p.scales, 200, torch.float16)
    with pytest.raises(TypeError, match="float64"):
        Packed4(p.codes, p.scales, 200, torch.float64)
    for c, s, n in [(p.codes, p.scales, 300), (p.codes, p.scales, 100), (p.codes[:, :-1], p.scales, 200), (p.codes, p.scales[:, :1], 200)]:
        with pytest.raises(ValueError, match="Packed4: codes of shape"):
            Packed4(c, s, n, torch.float16)
    with pytest.raises(ValueError, match="4194305 channels"):
        Packed4(p.codes, p.scales, (1 << 22) + 1, torch.float16)
    with pytest.raises(ValueError, match="4194305 channels"):
        packed4.pack4(torch.zeros(1).expand(1, (1 << 22) + 1))


def test_cpu_tensors_are_refused(host_layer):
    p = _packed()
    with pytest.raises(ValueError, match="GPU only"):
        packed4.pack4(torch.randn(3, 4))
    with pytest.raises(ValueError, match="GPU only"):
        packed4.unpack4(p)
    for x in (torch.randn(3, 200), _packed(3)):
        with pytest.raises(ValueError, match="GPU only"):
            matrix_linear.linear_forward(x, p)
    for shape in ((), (3, 0)):
        with pytest.raises(ValueError, match="pack4: a tensor of shape"):
            packed4.pack4(torch.zeros(shape))
    with pytest.raises(TypeError, match="float64"):
        packed4.unpack4(p, torch.float64)


def test_operands_that_do_not_fit():
    w, x = _packed(5, 200), torch.randn(3, 200).bfloat16()
    with pytest.raises(ValueError, match="weight of shape"):
        matrix_linear.linear_forward(x[:, :-1], w)
    with pytest.raises(ValueError, match="weight of shape"):
        matrix_linear.linear_forward(_packed(3, 199), w)
    with pytest.raises(ValueError, match="weight of shape"):
        matrix_linear.linear_forward(x, Packed4.from_parts(*(v.view((1,) + v.shape) for v in w.parts()), 200, torch.bfloat16))
    with pytest.raises(TypeError, match="takes a weight in 4 bits"):
        matrix_linear.linear_forward(_packed(3), torch.randn(5, 200).bfloat16())
    with pytest.raises(NotImplementedError, match="no z"):
        matrix_linear.linear_forward(_packed(3), w, keep_z=True)
    with pytest.raises(ValueError, match="the bias has shape"):
        matrix_linear.linear_forward(x, w, torch.zeros(4).bfloat16())
    with pytest.raises(TypeError, match="the bias is"):
        matrix_linear.linear_forward(x, w, torch.zeros(5))
    with pytest.raises(ValueError, match="the residual has shape"):
        matrix_linear.linear_forward(x, w, None, torch.zeros(3, 4).bfloat16())
    with pytest.raises(ValueError, match="activation"):
        matrix_linear.linear_forward(x, w, activation="tanh")
    with pytest.raises(ValueError, match="the weight has shape"):
        matrix_linear.linear_backward(torch.randn(3, 4), None, w, need_dw=False)
    with pytest.raises(TypeError, match="takes a weight in 4 bits"):
        matrix_linear.linear(_packed(3), torch.randn(5, 200).bfloat16())
    with pytest.raises(NotImplementedError, match="no gradient passes"):
        matrix_linear.linear(_packed(3), w, torch.zeros(5).bfloat16().requires_grad_())
    with pytest.raises(ValueError, match="channel_axis"):
        matrix_linear.linear(_packed(3), w, channel_axis=0)


def test_c_entry_points_refuse():
    lib = _lib.load()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.wc_packed4_bytes(33, 129, ctypes.byref(a), ctypes.byref(b)) == 0 and (a.value, b.value) == (33 * 128, 2 * 2 * 128)
    assert lib.wc_packed4_bytes(33, 0, ctypes.byref(a), ctypes.byref(b)) == _lib.WC_ERR_BAD_ARG
    assert lib.wc_packed4_bytes(33, (1 << 22) + 1, ctypes.byref(a), ctypes.byref(b)) == _lib.WC_ERR_UNSUPPORTED
    assert lib.wc_packed4_bytes(33, 4, None, None) == _lib.WC_ERR_BAD_ARG
    assert lib.wc_pack4(None, None, None, 0, 4, 0, None) == 0
    assert lib.wc_pack4(None, None, None, 1, 4, 0, None) == _lib.WC_ERR_BAD_ARG
    assert lib.wc_unpack4(None, None, None, 1, 4, 7, None) == _lib.WC_ERR_BAD_ARG
    assert lib.wc_pack4(256, 8, 256, 1, 4, 0, None) == _lib.WC_ERR_BAD_ARG
    assert lib.wc_unpack4(256, 24, 256, 1, 4, 0, None) == _lib.WC_ERR_BAD_ARG
    d = _lib.LinearDesc(3000, 256, 64, _lib.WC_F16, 0, 0)
    n = ctypes.c_size_t()
    assert lib.wc_linear4_workspace_bytes(ctypes.byref(d), 0, ctypes.byref(n)) == 0 and n.value >= 64 * 256 * 2
    w, at = _lib.Packed4Parts(256, 256), ctypes.c_void_p(256)
    run = lambda x, x4, w, y, ws=None, size=0: lib.wc_linear4_forward(ctypes.byref(d), x, x4, w, None, None, y, None, ws, size, None)  # noqa: E731
    assert run(None, None, ctypes.byref(w), at) == _lib.WC_ERR_BAD_ARG
    assert run(at, ctypes.byref(w), ctypes.byref(w), at) == _lib.WC_ERR_BAD_ARG
    assert run(at, None, None, at) == _lib.WC_ERR_BAD_ARG
    assert run(at, None, ctypes.byref(_lib.Packed4Parts(256, 8)), at) == _lib.WC_ERR_BAD_ARG
    assert run(at, None, ctypes.byref(w), at) == _lib.WC_ERR_WORKSPACE
    assert run(at, None, ctypes.byref(w), at, ctypes.c_void_p(8), n.value) == _lib.WC_ERR_WORKSPACE
    d.K = (1 << 22) + 1
    assert lib.wc_linear4_workspace_bytes(ctypes.byref(d), 0, ctypes.byref(n)) == _lib.WC_ERR_UNSUPPORTED


def test_c_gradients_refuse():
    lib = _lib.load()
    n, w = ctypes.c_size_t(), _lib.Packed4Parts(256, 256)
    for rows, act in [(3, 0), (3, 2), (600, 0), (600, 2)]:
        d = _lib.LinearDesc(rows, 256, 64, _lib.WC_F16, act, 0)
        grads = lambda dy=256, w=None, z=256, dx=256, x=None, dw=None, db=None: _lib.LinearGradients(dy, x, None, w, z, None, dx, dw, _lib.WC_F16, db, _lib.WC_F32, None)  # noqa: E731,B023
        size = lambda g: (lib.wc_linear4_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(g), ctypes.byref(n)), n.value)  # noqa: E731,B023
        run = lambda g, w4, ws=None, size=0: lib.wc_linear4_backward(ctypes.byref(d), ctypes.byref(g), w4, ws, size, None)  # noqa: E731,B023
        rc, need = size(grads())
        # dz of few rows, or the weight widened
        assert rc == 0 and need >= (0 if rows == 3 and not act else rows * 64 * 2 if rows == 3 else 64 * 256 * 2)
        at = ctypes.c_void_p(256)
        assert run(grads(dy=None), ctypes.byref(w), at, need) == _lib.WC_ERR_BAD_ARG
        assert run(grads(w=256), ctypes.byref(w), at, need) == _lib.WC_ERR_BAD_ARG
        assert run(grads(), None, at, need) == _lib.WC_ERR_BAD_ARG
        assert run(grads(), ctypes.byref(_lib.Packed4Parts(256, 8)), at, need) == _lib.WC_ERR_BAD_ARG
        if act:
            assert run(grads(z=None), ctypes.byref(w), at, need) == _lib.WC_ERR_BAD_ARG
        if need:
            assert run(grads(), ctypes.byref(w), at, need - 1) == _lib.WC_ERR_WORKSPACE
            assert run(grads(), ctypes.byref(w), ctypes.c_void_p(8), need) == _lib.WC_ERR_WORKSPACE
        d.rows = 0
        assert size(grads()) == (0, 0) and run(grads(), ctypes.byref(w)) == _lib.WC_ERR_BAD_ARG
        d.rows, d.C = rows, 0
        assert size(grads())[0] == _lib.WC_ERR_BAD_ARG
        d.C = (1 << 22) + 1
        assert size(grads())[0] == _lib.WC_ERR_UNSUPPORTED
    assert lib.wc_linear4_backward_workspace_bytes(ctypes.byref(d), None, ctypes.byref(n)) == _lib.WC_ERR_BAD_ARG
