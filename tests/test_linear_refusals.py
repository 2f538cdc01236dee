"""What linear layers and activations in 8 bits refuse, on the CPU: host layers before any launch, entry points by their status."""
import ctypes

import pytest
import torch

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import _lib, checkpoint8, matrix_linear

import linear_oracle as lo


def test_operands_are_checked_by_name(host_layer):
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    f = matrix_linear.linear_forward
    with pytest.raises(ValueError, match="GPU only"):
        f(x, w)
    with pytest.raises(ValueError, match="activation 'swish'"):
        f(x, w, activation="swish")
    with pytest.raises(ValueError, match="expected \\(..., C\\) and \\(K, C\\)"):
        f(x, torch.randn(5, 3))
    with pytest.raises(ValueError, match="expected \\(..., C\\) and \\(K, C\\)"):
        f(torch.tensor(1.0), w)
    with pytest.raises(ValueError, match="neither of them 0"):
        f(torch.randn(3, 0), torch.randn(5, 0))
    with pytest.raises(ValueError, match="the bias has shape"):
        f(x, w, torch.randn(4))
    with pytest.raises(TypeError, match="the bias is torch.float16"):
        f(x, w, torch.randn(5).half())
    with pytest.raises(TypeError, match="the weight is torch.float16"):
        f(x, w.half())
    with pytest.raises(ValueError, match="the residual has shape"):
        f(x, w, None, torch.randn(5))
    with pytest.raises(ValueError, match="GPU only"):
        pkg.MatrixLinear(4, 5)(x)
    with pytest.raises(ValueError, match="checkpoint"):
        pkg.MatrixLinear(4, 5, checkpoint="fp8")
    with pytest.raises(ValueError, match="checkpoint"):
        pkg.WinoConv2d(4, 4, 3, checkpoint=8)


def test_gradients_check_what_they_read(host_layer):
    dy, x, w = torch.randn(3, 5), torch.randn(3, 4), torch.randn(5, 4)
    g = matrix_linear.linear_backward
    with pytest.raises(ValueError, match="needs z"):
        g(dy, x, w, None, "gelu")
    with pytest.raises(ValueError, match="z has shape"):
        g(dy, x, w, x, "gelu")
    with pytest.raises(ValueError, match="dx needs w"):
        g(dy, x, None)
    with pytest.raises(ValueError, match="dw needs x"):
        g(dy, None, w)
    with pytest.raises(ValueError, match="x has shape"):
        g(dy, x[:2], w)
    with pytest.raises(TypeError, match="x is torch.float16"):
        g(dy, x.half(), w)
    with pytest.raises(ValueError, match="GPU only"):
        g(dy, x, w)


def test_packed_tensors_check_their_parts(host_layer):
    codes, exps = torch.zeros(3, 40, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.int8)
    p = checkpoint8.Packed8(codes, exps, torch.float16)
    assert p.shape == (3, 40)
    with pytest.raises(ValueError, match="groups of 32"):
        checkpoint8.Packed8(codes, exps[:, :1], torch.float16)
    with pytest.raises(TypeError, match="int8"):
        checkpoint8.Packed8(codes.int(), exps, torch.float16)
    with pytest.raises(TypeError, match="supports float32"):
        checkpoint8.Packed8(codes, exps, torch.float64)
    with pytest.raises(ValueError, match="GPU only"):
        checkpoint8.unpack8(p)
    with pytest.raises(ValueError, match="GPU only"):
        checkpoint8.pack8(torch.zeros(3))
    with pytest.raises(ValueError, match="expected"):
        matrix_linear.linear_backward(torch.zeros(3, 5, dtype=torch.float16), p, torch.zeros(5, 39, dtype=torch.float16))


@pytest.mark.parametrize("rows,C,K,dtype,act,rc", [
    (-1, 4, 4, 1, 0, -1), (4, 0, 4, 1, 0, -1), (4, 4, 0, 1, 0, -1), (4, 4, 4, 3, 0, -1), (4, 4, 4, 1, 5, -1), (4, 4, 4, 1, -1, -1),
    (1 << 31, 4, 4, 1, 0, -2), (4, (1 << 24) + 1, 4, 1, 0, -2), (4, 4, (1 << 24) + 1, 1, 0, -2), (4, 4, 4, 1, 0, 0)])
def test_descriptors(rows, C, K, dtype, act, rc):
    n = ctypes.c_size_t()
    d = _lib.LinearDesc(rows, C, K, dtype, act, 0)
    assert _lib.load().wc_linear_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == rc
    g = _lib.LinearGradients()
    assert _lib.load().wc_linear_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(g), ctypes.byref(n)) == rc


def test_entry_points_refuse_before_a_launch():
    lib, one = _lib.load(), ctypes.c_void_p(256)
    d = _lib.LinearDesc(4, 4, 4, 1, 2, 0)
    assert lib.wc_linear_forward(None, one, one, None, None, one, None, None, 0, None) == -1
    assert lib.wc_linear_forward(ctypes.byref(d), None, one, None, None, one, None, None, 0, None) == -1
    assert lib.wc_linear_forward(ctypes.byref(d), one, one, None, None, None, None, None, 0, None) == -1
    empty = _lib.LinearDesc(0, 4, 4, 1, 2, 0)
    assert lib.wc_linear_forward(ctypes.byref(empty), None, None, None, None, None, None, None, 0, None) == 0
    g = _lib.LinearGradients(dy=256, x=256, w=256, dx=256, dw=256, dw_dtype=1)
    n = ctypes.c_size_t()
    assert lib.wc_linear_backward(ctypes.byref(empty), ctypes.byref(g), one, 1 << 30, None) == -1      # no rows
    assert lib.wc_linear_backward(ctypes.byref(d), ctypes.byref(g), one, 1 << 30, None) == -1          # no z
    g.z = 256
    g.dw_dtype = 2                                                                                      # neither the operands' type nor fp32
    assert lib.wc_linear_backward(ctypes.byref(d), ctypes.byref(g), one, 1 << 30, None) == -1
    g.dw_dtype = 1
    assert lib.wc_linear_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(g), ctypes.byref(n)) == 0 and n.value > 0
    assert lib.wc_linear_backward(ctypes.byref(d), ctypes.byref(g), one, n.value - 1, None) == -3
    assert lib.wc_linear_backward(ctypes.byref(d), ctypes.byref(g), None, n.value, None) == -3
    assert lib.wc_linear_backward(ctypes.byref(d), ctypes.byref(g), ctypes.c_void_p(128), n.value, None) == -3
    assert b"aligned" in lib.wc_last_error()
    assert lib.wc_pack8(None, one, one, 4, 4, 1, 0, None) == -1
    assert lib.wc_pack8(one, one, one, 4, 0, 1, 0, None) == -1
    assert lib.wc_unpack8(one, None, one, 4, 4, 1, None) == -1
    assert lib.wc_unpack8(None, None, None, 0, 4, 1, None) == 0


def test_the_oracle_of_8_bits_is_half_a_step_off():
    g = torch.Generator().manual_seed(5)
    for t in lo.TYPES:
        x = (torch.randn(50, 77, generator=g) * torch.exp(4 * torch.randn(50, 1, generator=g))).to(t)
        codes, exps = lo.pack(x)
        step = torch.ldexp(torch.ones(()).double(), exps.to(torch.int64)).repeat_interleave(32, 1)[:, :77]
        v = lo.unpack(codes, exps)
        off = (v - x.double()).abs()
        assert bool((off <= torch.where(x.double().abs() > 127.5 * step, step, step / 2)).all())
        assert torch.equal(v.to(t).double(), v)                            # what it reads as is of x's type
        assert int(codes.abs().max()) <= 127 and int(codes.int().abs().amax(1).min()) >= 32
        assert torch.equal(lo.pack(v.to(t))[0], codes) and torch.equal(lo.pack(v.to(t))[1], exps)
    codes, exps = lo.pack(torch.tensor([[3e-45, 0.0, 1.0], [float("inf"), 1.0, 0.0], [0.0, 0.0, 0.0]]), keep_sign=True)
    assert codes.tolist() == [[1, 0, 64], [0, 0, 0], [0, 0, 0]] and exps.tolist() == [[-6], [127], [-126]]


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: where there is no GPU a launch fails and nothing is read")
def test_a_workspace_of_the_stated_size_is_enough():
    """Whatever stands in the epilogue and wherever the operands start, which the sizes are asked for without."""
    import random
    lib, rng, n = _lib.load(), random.Random(7), ctypes.c_size_t()
    for _ in range(1500):
        d = _lib.LinearDesc(rng.choice([1, 3, 8, 16, 17, 64, 300, 777, 5000, 200000]), rng.choice([1, 8, 40, 77, 264, 1000, 4096, 25088]),
                            rng.choice([1, 8, 77, 264, 328, 1000, 4096]), rng.randrange(3), rng.randrange(5), rng.randrange(2))
        at = lambda p=1.0: (1 << 30) + rng.choice([0, 0, 2]) if rng.random() < p else None  # noqa: E731
        assert lib.wc_linear_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == 0
        rc = lib.wc_linear_forward(ctypes.byref(d), at(), at(), at(0.5), at(0.5), at(), at(0.5), ctypes.c_void_p(1 << 40), n.value, None)
        assert rc == -4, (rc, lib.wc_last_error(), d.rows, d.C, d.K)
        g = _lib.LinearGradients(dy=at(), x=at(), x_exponents=at(0.3), w=at(), z=at(), z_exponents=at(0.3), dx=at(0.7), dw=at(), dw_dtype=0, db=at(0.5), db_dtype=0, dz=at(0.3))
        assert lib.wc_linear_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(g), ctypes.byref(n)) == 0
        rc = lib.wc_linear_backward(ctypes.byref(d), ctypes.byref(g), ctypes.c_void_p(1 << 40), n.value, None)
        assert rc == -4, (rc, lib.wc_last_error(), d.rows, d.C, d.K)
