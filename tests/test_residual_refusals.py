"""The oracle of joins against differentiation of the definition; arguments that do not fit together, refused on the CPU before any launch."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import pytorch_winoconv_amd as pkg
from pytorch_winoconv_amd import _lib, residual
from pytorch_winoconv_amd.residual import Drop, Norm

import residual_oracle as ro


@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "channel", "sample"])
def test_oracle_is_the_derivative(post, pre, gate):
    g = torch.Generator().manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    make = lambda kind: None if kind == "none" else (kind, normal(5), normal(5) if kind == "layer" else None, 1e-2)  # noqa: E731
    f, x, po, pr = normal(3, 4, 5), normal(3, 4, 5), make(post), make(pre)
    gt = {"none": None, "channel": normal(5), "sample": normal(3, 5)}[gate]
    drop = (0.3, 12345678901234567, 1 << 40, "element")
    leaves = {"block": f, "stream": x, "gate": gt}
    for name, n in (("post", po), ("pre", pr)):
        if n is not None:
            leaves.update({name + "_weight": n[1], name + "_bias": n[2]})
    leaves = {k: v.requires_grad_() for k, v in leaves.items() if v is not None}
    s, y = ro.join(f, x, gt, po, pr, drop, 0.7, 1.3)
    ds, dy = normal(3, 4, 5), normal(3, 4, 5) if pr else None
    want = torch.autograd.grad([s] + ([y] if pr else []), list(leaves.values()), [ds] + ([dy] if pr else []))
    off = lambda v: None if v is None else v.detach()  # noqa: E731
    parts = lambda n: None if n is None else (n[0], off(n[1]), off(n[2]), n[3])  # noqa: E731
    got = ro.backward(ds, dy, f.detach(), s.detach(), off(gt), parts(po), parts(pr), drop, 0.7, 1.3)
    assert set(got) == set(leaves)
    for k, v in zip(leaves, want):
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-12), k
    # and against differences
    def total(f):
        s, y = ro.join(f, x.detach(), off(gt), parts(po), parts(pr), drop, 0.7, 1.3)
        return (s * ds).sum() + ((y * dy).sum() if pr else 0)
    step = 1e-6
    for i in (0, 17, 59):
        e = torch.zeros(60, dtype=torch.float64)
        e[i] = step
        e = e.view(3, 4, 5)
        assert abs(float((total(f.detach() + e) - total(f.detach() - e)) / (2 * step) - got["block"][0].flatten()[i])) < 1e-6


def test_generator_has_the_published_values():
    """The known answers that the generator's authors publish with it, Philox4x32-10 of a counter and a key of zeros."""
    zeros = ro.words(1, 8, 0, 0)[0]
    assert [int(zeros[2 * i] + (zeros[2 * i + 1] << 16)) for i in range(4)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def test_drop_arguments():
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            Drop(p, 0)
    with pytest.raises(ValueError, match="'element' or 'sample'"):
        Drop(0.1, 0, 0, "row")
    for seed, offset in [(-1, 0), (0, -1), (1 << 64, 0), (0, 1 << 64)]:
        with pytest.raises(ValueError, match="seed"):
            Drop(0.1, seed, offset)
    for state in (torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="int64 tensor"):
            Drop(0.1, state)
    assert [Drop(p, 0).level for p in (0, 1, 0.5, 2.0 ** -17, 1 - 2.0 ** -18)] == [0, 65536, 32768, 0, 65536]


def test_norm_arguments():
    with pytest.raises(ValueError, match="layer, rms"):
        Norm("batch")
    for eps in (-1e-5, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="eps"):
            Norm("rms", eps=eps)
    with pytest.raises(ValueError, match="layer, rms"):
        pkg.BlockNorm(8, "batch")


def test_cpu_tensors_are_refused(host_layer):
    x = torch.randn(3, 4)
    for call in (lambda: residual.norm(x, Norm("rms")), lambda: residual.dropout(x, Drop(0.1, 0)), lambda: residual.join(x, x), lambda: pkg.BlockNorm(4)(x),
                 lambda: residual.join_backward(x, None, None, None, None), lambda: residual.norm_backward(x, x, torch.zeros(3, 2), Norm("rms"))):
        with pytest.raises(ValueError, match="GPU only"):
            call()
    for shape in ((), (3, 0)):
        with pytest.raises(ValueError, match="a tensor of shape"):
            residual.norm(torch.zeros(shape), Norm("rms"))
    with pytest.raises(ValueError, match="16777217 channels"):
        residual.dropout(torch.zeros(1).expand(1, (1 << 24) + 1), Drop(0.1, 0))


def test_operands_that_do_not_fit(host_layer):
    f, C = torch.randn(3, 2, 4).half(), 4
    half = lambda *s: torch.zeros(*s).half()  # noqa: E731
    for call, error, match in [
            (lambda: residual.join(f, f[:2]), ValueError, "the stream has shape"),
            (lambda: residual.join(f, f.float()), TypeError, "the stream is"),
            (lambda: residual.join(f, f[0], channel_axis=1), ValueError, "the stream has shape"),
            (lambda: residual.join(f, gate=half(3)), ValueError, "the gate has shape"),
            (lambda: residual.join(f, gate=half(2, C)), ValueError, "the gate has shape"),
            (lambda: residual.join(f, gate=half(3, 2, C)), ValueError, "the gate has shape"),
            (lambda: residual.join(f, gate=half(C).bfloat16()), TypeError, "the gate is"),
            (lambda: residual.join(f, post=Norm("rms", half(3))), ValueError, "the weight of post"),
            (lambda: residual.join(f, pre=Norm("layer", half(C), half(3))), ValueError, "the bias of pre"),
            (lambda: residual.join(f, pre=Norm("layer", half(C), torch.zeros(C))), TypeError, "share one dtype"),
            (lambda: residual.norm(f, Norm("rms", half(C).bfloat16())), TypeError, "the weight of pre"),
            (lambda: residual.join_backward(None, None, f, f, None), ValueError, "neither ds nor dy"),
            (lambda: residual.join_backward(f, f, f, f, None), ValueError, "dy without pre"),
            (lambda: residual.join_backward(f, None, None, f, None, post=Norm("rms")), ValueError, "need block"),
            (lambda: residual.join_backward(f, None, None, f, None, gate=half(C)), ValueError, "need block"),
            (lambda: residual.join_backward(None, f, None, None, None, pre=Norm("rms")), ValueError, "needs s"),
            (lambda: residual.join_backward(None, f, None, f, None, pre=Norm("rms")), ValueError, "statistics of pre"),
            (lambda: residual.join_backward(None, f, f, f, (None, torch.zeros(6, 2)), pre=Norm("rms")), ValueError, "holds the stream"),
            (lambda: residual.join_backward(None, f, f, f, (None, torch.zeros(6, 2), f[:2]), pre=Norm("rms")), ValueError, "the stream has shape"),
            (lambda: residual.join_backward(f, None, f, f, (torch.zeros(5, 2), None), post=Norm("rms")), ValueError, "statistics of post"),
            (lambda: residual.join_backward(f, None, f[:2], f, None), ValueError, "block has shape")]:
        with pytest.raises(error, match=match):
            call()


@pytest.mark.parametrize("which", range(7))
def test_forward_mode_is_refused(which):
    ts = [torch.randn(s) for s in ((3, 4), (3, 4), (4,), (4,), (4,), (4,), (4,))]
    with forward_ad.dual_level():
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                residual.join(ts[0], ts[1], Norm("layer", ts[3], ts[4]), ts[2], Norm("layer", ts[5], ts[6]))


def test_c_entry_points_refuse():
    lib = _lib.load()
    at = ctypes.c_void_p(256)
    none = _lib.NormParts(0, 0.0, None, None, 0)

    def desc(**more):
        d = _lib.JoinDesc(12, 3, 8, _lib.WC_F16, 1.0, 1.0, 0, _lib.WC_F16, 0, 0, 0, 0, None, none, none)
        for k, v in more.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    forward = lambda d, f=at, x=None, gate=None, s=at, y=None: lib.wc_join_forward(d, f, x, gate, s, y, None, None, None)  # noqa: E731
    rms = _lib.NormParts(1, 1e-5, None, None, _lib.WC_F16)
    for more in (dict(C=0), dict(dtype=5), dict(samples=5), dict(samples=0), dict(rows=-1), dict(gate_rows=2), dict(drop_level=65537), dict(drop_level=-1),
                 dict(post=_lib.NormParts(3, 1e-5, None, None, 1)), dict(pre=_lib.NormParts(1, -1.0, None, None, 1)), dict(pre=_lib.NormParts(1, 1e-5, None, None, 2)),
                 dict(gate_rows=3, gate_dtype=2)):
        assert forward(desc(**more)) == _lib.WC_ERR_BAD_ARG, more
    assert forward(desc(C=(1 << 24) + 1)) == _lib.WC_ERR_UNSUPPORTED
    assert forward(desc(rows=0, samples=1), None, None, None, None) == 0
    assert forward(desc(), None) == _lib.WC_ERR_BAD_ARG
    assert forward(desc(), s=None) == _lib.WC_ERR_BAD_ARG
    assert forward(desc(), y=at) == _lib.WC_ERR_BAD_ARG
    assert forward(desc(gate_rows=3)) == _lib.WC_ERR_BAD_ARG
    assert forward(desc(), gate=at) == _lib.WC_ERR_BAD_ARG
    assert lib.wc_join_forward(desc(pre=rms), at, None, None, at, at, None, 260, None) == _lib.WC_ERR_BAD_ARG
    n = ctypes.c_size_t()

    def backward(d, ws=None, size=0, **given):
        return lib.wc_join_backward(d, ctypes.byref(_lib.JoinGradients(**given)), ws, size, None)
    assert backward(desc()) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(rows=0, samples=1), ds=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(), dy=256, df=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(pre=rms), dy=256, df=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(post=rms), ds=256, df=256, f=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(post=rms), ds=256, df=256, post_stats=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(), ds=256, df=256, dgate=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(), ds=256, df=256, dpost_weight=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(), ds=256, df=256, dpre_bias=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(gate_rows=3), ds=256, df=256) == _lib.WC_ERR_BAD_ARG
    assert backward(desc(post=rms), ds=256, df=256, f=256, post_stats=260) == _lib.WC_ERR_BAD_ARG
    q = _lib.JoinGradients(dy=256, s=256, pre_stats=256, df=256, dpre_weight=256)
    assert lib.wc_join_backward_workspace_bytes(desc(pre=rms), ctypes.byref(q), ctypes.byref(n)) == 0 and n.value > 0
    assert lib.wc_join_backward(desc(pre=rms), ctypes.byref(q), None, 0, None) == _lib.WC_ERR_WORKSPACE
    assert lib.wc_join_backward(desc(pre=rms), ctypes.byref(q), ctypes.c_void_p(8), n.value, None) == _lib.WC_ERR_WORKSPACE
