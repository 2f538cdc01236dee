"""What joins the blocks of a residual network to its stream, in one pass over memory each way (the reference leaves all of it to torch):

    s = stream_scale x + block_scale gate drop(post(f)),   y = pre(s)

f is what a block gave, x the stream, post the norm behind the block, pre the norm before the next one; all but f may be missing, so that a
norm alone and dropout alone are the same kernels.  Norms are over the channels (the last axis): "rms", v w / sqrt(mean(v^2) + eps), and
"layer", (v - mean) w / sqrt(var + eps) + bias.  gate is one value a channel, (C,), or one a sample and channel, (N, C), where the samples are the first
axis of f.  Arithmetic and sums are fp32, s and y are rounded once (y is of s before that).  float32, float16 and
bfloat16; parameters and gate of that type or float32.  The GPU only.  In 16-bit types the backward pass computes s again from f and x, since a norm's
gradient from the rounded s is 1.4 times as far from the exact one.

Dropout draws its mask from a counter-based generator, Philox4x32-10, by seed, offset, row and channel, and draws it again for the backward pass: nothing
of it is stored, and the same numbers give the same mask whatever the strides, the launch or the type.  Each channel has 16 bits: the
probability is the nearest multiple of 2^-16, and what is kept is divided by exactly the share that is.
"""
import collections
import copy
import ctypes
import math

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, engine
from ._lib import NormParts, check
from .matrix_linear import MatrixLinear

KINDS = {"rms": 1, "layer": 2}
Gradients = collections.namedtuple("Gradients", "block stream post_weight post_bias gate pre_weight pre_bias")


class Norm:
    """A norm over channels: its kind, "rms" or "layer", weight (C,) or None (1), bias (C,) or None (0), and what is added to the variance."""

    __slots__ = ("kind", "weight", "bias", "eps")

    def __init__(self, kind, weight=None, bias=None, eps=1e-5):
        if kind not in KINDS:
            raise ValueError("norm %r: one of %s" % (kind, ", ".join(sorted(KINDS))))
        if not (eps >= 0 and math.isfinite(eps)):
            raise ValueError("norm: eps %r" % (eps,))
        self.kind, self.weight, self.bias, self.eps = kind, weight, bias, float(eps)


class Drop:
    """Dropout with probability p, by seed and offset below 2^64 (a call counts its offset up), "element" by element or a whole "sample" at a time.
    seed may be an int64 tensor (seed, offset) on the GPU, which the kernels read, also in a graph's replays; it must stay as it is until the backward
    pass has run."""

    __slots__ = ("p", "level", "seed", "offset", "per")

    def __init__(self, p, seed, offset=0, per="element"):
        if not 0 <= p <= 1:
            raise ValueError("dropout: probability %r" % (p,))
        if per not in ("element", "sample"):
            raise ValueError("dropout per %r: 'element' or 'sample'" % (per,))
        if isinstance(seed, torch.Tensor):
            if seed.dtype != torch.int64 or tuple(seed.shape) != (2,) or not seed.is_contiguous() or offset:
                raise ValueError("dropout: seed and offset in one contiguous int64 tensor (2,), got %s of shape %r and offset %r"
                                 % (seed.dtype, tuple(seed.shape), offset))
        elif not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
            raise ValueError("dropout: seed %r and offset %r, from 0 to 2^64 - 1" % (seed, offset))
        self.p, self.level, self.seed, self.offset, self.per = p, int(round(p * 65536)), seed, offset, per


def _rows(shape):
    n = 1
    for v in shape[:-1]:
        n *= v
    return n


def _own_type(t, like, what):
    if t.dtype != like.dtype and t.dtype != torch.float32:
        raise TypeError("%s is %s, the tensors are %s: their type or float32" % (what, t.dtype, like.dtype))
    if t.device != like.device:
        raise ValueError("%s is on %s, expected %s" % (what, t.device, like.device))


def _check_norm(n, f, what):
    if n is None:
        return
    C = f.shape[-1]
    for t, part in ((n.weight, "weight"), (n.bias, "bias")):
        if t is None:
            continue
        if tuple(t.shape) != (C,):
            raise ValueError("the %s of %s has shape %r, expected (%d,)" % (part, what, tuple(t.shape), C))
        _own_type(t, f, "the %s of %s" % (part, what))
    if n.weight is not None and n.bias is not None and n.weight.dtype != n.bias.dtype:
        raise TypeError("weight and bias of %s are %s and %s: they must share one dtype" % (what, n.weight.dtype, n.bias.dtype))


def _check_like(t, f, what):
    if t is None:
        return
    if t.shape != f.shape:
        raise ValueError("%s has shape %r, expected %r" % (what, tuple(t.shape), tuple(f.shape)))
    if t.dtype != f.dtype:
        raise TypeError("%s is %s, the tensors are %s: they must share one dtype" % (what, t.dtype, f.dtype))
    if t.device != f.device:
        raise ValueError("%s is on %s, expected %s" % (what, t.device, f.device))


def _samples(f):
    return f.shape[0] if f.dim() > 1 else 1


def _check_block(f, post, gate, pre, drop, others):
    """Shapes, types and devices that the C ABI cannot see; others: {what: tensor of f's shape and type, or None}."""
    if f.dim() < 1 or not f.shape[-1]:
        raise ValueError("a tensor of shape %r: expected (..., C), C not 0" % (tuple(f.shape),))
    if f.shape[-1] > 1 << 24:
        raise ValueError("%d channels, at most 2^24" % f.shape[-1])
    for what, t in others.items():
        _check_like(t, f, what)
    _check_norm(post, f, "post")
    _check_norm(pre, f, "pre")
    if gate is not None:
        C = f.shape[-1]
        if tuple(gate.shape) not in ((C,), (_samples(f), C)):
            raise ValueError("the gate has shape %r, expected (%d,) or (%d, %d)" % (tuple(gate.shape), C, _samples(f), C))
        _own_type(gate, f, "the gate")
    if drop is not None and isinstance(drop.seed, torch.Tensor) and drop.seed.device != f.device:
        raise ValueError("dropout's seed is on %s, expected %s" % (drop.seed.device, f.device))
    engine._require_gpu(f)


def _plain(t):
    return None if t is None else t.detach().contiguous()


def _parts(n, f):
    """A norm's struct, and the tensors that it points to."""
    if n is None:
        return NormParts(0, 0.0, None, None, engine._DTYPES[f.dtype]), ()
    w, b = _plain(n.weight), _plain(n.bias)
    given = w if w is not None else b
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return NormParts(KINDS[n.kind], n.eps, at(w), at(b), engine._DTYPES[f.dtype if given is None else given.dtype]), (w, b)


def _desc(f, post, gate, pre, drop, stream_scale, block_scale):
    (po, keep1), (pr, keep2) = _parts(post, f), _parts(pre, f)
    rows = _rows(f.shape)
    d = _lib.JoinDesc(rows, _samples(f) if rows else 1, f.shape[-1], engine._DTYPES[f.dtype], stream_scale, block_scale, 0 if gate is None else _rows(gate.shape),
                      engine._DTYPES[f.dtype if gate is None else gate.dtype], 0, 0, 0, 0, None, po, pr)
    if drop is not None:
        d.drop_level, d.drop_per_sample = drop.level, int(drop.per == "sample")
        if isinstance(drop.seed, torch.Tensor):
            d.drop_state = drop.seed.data_ptr()
        else:
            d.drop_seed, d.drop_offset = drop.seed, drop.offset
    return d, (keep1, keep2)


def _ext_norm(n):
    return (0, 0.0, None, None) if n is None else (KINDS[n.kind], n.eps, n.weight, n.bias)


def _ext_drop(drop):
    if drop is None:
        return 0, False, 0, 0, None
    if isinstance(drop.seed, torch.Tensor):
        return drop.level, drop.per == "sample", 0, 0, drop.seed
    return drop.level, drop.per == "sample", drop.seed, drop.offset, None


def _forward(f, x, post, gate, pre, drop, stream_scale, block_scale, need_s, keep):
    """(s, y, (post's statistics, pre's))."""
    if engine.USE_EXT:
        out = engine._ext.join_forward(f, x, gate, float(stream_scale), float(block_scale), *_ext_norm(post), *_ext_norm(pre), *_ext_drop(drop), need_s, keep)
        if out is not None:
            return out[0], out[1], (out[2], out[3])
    _check_block(f, post, gate, pre, drop, {"the stream": x})
    f, x, gate = _plain(f), _plain(x), _plain(gate)
    d, kept = _desc(f, post, gate, pre, drop, stream_scale, block_scale)
    s = torch.empty_like(f) if need_s else None
    y = torch.empty_like(f) if pre is not None else None
    new = lambda wanted: torch.empty((d.rows, 2), dtype=torch.float32, device=f.device) if wanted else None  # noqa: E731
    post_stats, pre_stats = new(keep and post is not None), new(keep and pre is not None)
    if d.rows:
        p = engine._ptr
        with engine._on_device(f):
            check(_lib.load().wc_join_forward(ctypes.byref(d), p(f), p(x), p(gate), p(s), p(y), p(post_stats), p(pre_stats), engine._stream(f)))
    return s, y, (post_stats, pre_stats)


def join_forward(block, stream=None, post=None, gate=None, pre=None, drop=None, stream_scale=1.0, block_scale=1.0, keep=False):
    """(s, y, stats) for block = f (..., C) and stream = x of its shape, post and pre Norms, drop a Drop; y is None without pre.  stats is what join_backward
    wants, where keep is true."""
    s, y, stats = _forward(block, stream, post, gate, pre, drop, stream_scale, block_scale, True, bool(keep))
    return s, y, stats + ((stream,) if _again(block, pre) else ()) if keep else None


def _again(block, pre):
    """Whether the backward pass computes s again, unrounded, from block and stream."""
    return pre is not None and block.dtype != torch.float32


def join_backward(ds, dy, block, s, stats, post=None, gate=None, pre=None, drop=None, stream_scale=1.0, block_scale=1.0, need_block=True, need_stream=True,
                  need_gate=True, need_post=True, need_pre=True):
    """Gradients(block, stream, post_weight, post_bias, gate, pre_weight, pre_bias) of join_forward, None for those not asked for or of what is not there, each
    of the type of what it belongs to.  ds or dy may be None, for an s or y that went nowhere; block may be None where there is neither post nor a gate that
    wants its gradient, s without pre, or where block is given.  stats of 16-bit types with pre hold the stream, as it must still be; s is then computed again, unless
    block is None."""
    given = ds if ds is not None else dy
    if given is None:
        raise ValueError("join_backward: neither ds nor dy")
    if dy is not None and pre is None:
        raise ValueError("join_backward: dy without pre, whose result y is")
    through = pre if dy is not None else None
    need_gate = need_gate and gate is not None
    post_stats, pre_stats = stats[:2] if stats is not None else (None, None)
    again = through is not None and block is not None and stats is not None and len(stats) > 2
    x = stats[2] if again else None
    if (post is not None or need_gate) and block is None:
        raise ValueError("join_backward: the gradients of post and the gate need block")
    if through is not None and block is not None and given.dtype != torch.float32 and not again:
        raise ValueError("join_backward: of 16-bit types stats holds the stream too, as join_forward kept it")
    if through is not None and s is None and not again:
        raise ValueError("join_backward: the gradient of pre needs s, or block and what join_forward kept")
    if engine.USE_EXT and through is pre:
        out = engine._ext.join_backward(ds, dy, block, s, x, again, gate, post_stats, pre_stats, float(stream_scale), float(block_scale), *_ext_norm(post), *_ext_norm(pre),
                                        *_ext_drop(drop), need_block, need_stream, need_gate, need_post, need_pre)
        if out is not None:
            df, dx, pw, pb, qw, qb, dg = out
            return Gradients(df, dx, qw, qb, dg, pw, pb)
    rows = _rows(given.shape)
    for n, t, what in ((post, post_stats, "post"), (through, pre_stats, "pre")):
        if n is not None and (t is None or t.dtype != torch.float32 or tuple(t.shape) != (rows, 2) or t.device != given.device or not t.is_contiguous()):
            raise ValueError("join_backward: the statistics of %s are those that join_forward kept, (%d, 2) in float32" % (what, rows))
    _check_block(given, post, gate, pre, drop, {"ds": ds, "dy": dy, "block": block, "s": s, "the stream": x})
    like = lambda n, name, wanted: getattr(n, name) if wanted and n is not None else None  # noqa: E731
    want = [like(through, "weight", need_pre), like(through, "bias", need_pre), like(post, "weight", need_post), like(post, "bias", need_post), gate if need_gate else None]
    # (a norm that no gradient comes through has zeros)
    silent = [like(pre, name, need_pre) if through is None else None for name in ("weight", "bias")]
    zeros = lambda t: None if t is None else torch.zeros(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    dense = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    if rows == 0:
        pw, pb, qw, qb, dg = (zeros(t) for t in want)
        empty = dense(given)
        return Gradients(empty if need_block else None, empty if need_stream else None, qw, qb, dg, pw if silent[0] is None else zeros(silent[0]),
                         pb if silent[1] is None else zeros(silent[1]))
    if not (need_block or need_stream or any(t is not None for t in want)):
        return Gradients(None, None, None, None, None, zeros(silent[0]), zeros(silent[1]))
    ds, dy, block, s, x, g = (_plain(t) for t in (ds, dy, block, s, x, gate))
    d, kept = _desc(given, post, g, through, drop, stream_scale, block_scale)
    df, dx = (dense(given) if wanted else None for wanted in (need_block, need_stream))
    pw, pb, qw, qb, dg = (None if t is None else dense(t) for t in want)
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    q = _lib.JoinGradients(*(at(t) for t in (ds, dy, block if post is not None or need_gate or again else None,
                                             s if through is not None and not again else None, x, g, post_stats, pre_stats, df, dx, pw, pb, qw, qb, dg)))
    lib, nbytes = _lib.load(), ctypes.c_size_t()
    check(lib.wc_join_backward_workspace_bytes(ctypes.byref(d), ctypes.byref(q), ctypes.byref(nbytes)))
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=given.device)
    with engine._on_device(given):
        check(lib.wc_join_backward(ctypes.byref(d), ctypes.byref(q), engine._ptr(ws), nbytes.value, engine._stream(given)))
    return Gradients(df, dx, qw, qb, dg, zeros(silent[0]) if pw is None else pw, zeros(silent[1]) if pb is None else pb)


def norm_forward(x, norm, keep=False):
    """norm(x) for x (..., C); with keep (y, stats), stats for norm_backward."""
    if engine.USE_EXT:
        out = engine._ext.norm_forward(x, KINDS[norm.kind], norm.eps, norm.weight, norm.bias, keep)
        if out is not None:
            return out
    _, y, stats = _forward(x, None, None, None, norm, None, 1.0, 1.0, False, bool(keep))
    return (y, stats[1]) if keep else y


def norm_backward(dy, x, stats, norm, need_dx=True, need_dw=True, need_db=True):
    """(dx, dw, db) of norm_forward, None for those not asked for or without a parameter."""
    g = join_backward(None, dy, None, x, (None, stats), pre=norm if need_db or norm.bias is None else Norm(norm.kind, norm.weight, None, norm.eps), need_block=need_dx,
                      need_stream=False, need_pre=need_dw or need_db)
    return g.block, g.pre_weight if need_dw else None, g.pre_bias


def dropout_forward(x, drop):
    """drop(x).  Its gradient is the same of dy."""
    return _forward(x, None, None, None, None, drop, 1.0, 1.0, True, False)[0]


def _moved(t, axis):
    return None if t is None else t.movedim(axis, -1)


def _refuse_tangents(*ts):
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError("joins, norms and dropout have no forward-mode derivative: a tangent of their operands would be lost")


class JoinFunction(torch.autograd.Function):
    """join_forward with gradients."""

    @staticmethod
    def forward(ctx, block, stream, gate, post_w, post_b, pre_w, pre_b, conf):
        post, pre, drop, stream_scale, block_scale, need_s = conf
        post = post and Norm(post[0], post_w, post_b, post[1])
        pre = pre and Norm(pre[0], pre_w, pre_b, pre[1])
        s, y, (post_stats, pre_stats) = _forward(block, stream, post, gate, pre, drop, stream_scale, block_scale, need_s, True)
        need = ctx.needs_input_grad
        state = drop.seed if drop is not None and isinstance(drop.seed, torch.Tensor) else None
        # a norm alone keeps what it normalised, a join its s, or block and stream to compute it again; the block is kept for post and the gate too
        ctx.again = need_s and _again(block, pre)
        ctx.save_for_backward(block if post is not None or need[2] or ctx.again else None, None if pre is None or ctx.again else s if need_s else block,
                              stream if ctx.again else None, gate, post_w, post_b, pre_w, pre_b, post_stats, pre_stats, state)
        ctx.conf = conf
        ctx.set_materialize_grads(False)
        return (s, y) if need_s and pre is not None else s if need_s else y

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        block, s, stream, gate, post_w, post_b, pre_w, pre_b, post_stats, pre_stats, state = ctx.saved_tensors
        post, pre, drop, stream_scale, block_scale, need_s = ctx.conf
        need = ctx.needs_input_grad
        ds, dy = grads if need_s and pre else (grads[0], None) if need_s else (None, grads[0])
        if ds is None and dy is None:
            return (None,) * 8
        if state is not None:
            drop = Drop(drop.p, state, 0, drop.per)
        post = post and Norm(post[0], post_w, post_b, post[1])
        pre = pre and Norm(pre[0], pre_w, pre_b, pre[1])
        g = join_backward(ds, dy, block, s, (post_stats, pre_stats) + ((stream,) if ctx.again else ()), post, gate, pre, drop, stream_scale, block_scale, need[0], need[1], need[2],
                          need[3] or need[4], need[5] or need[6])
        return g.block, g.stream, g.gate, g.post_weight, g.post_bias, g.pre_weight, g.pre_bias, None


def _call(block, stream, post, gate, pre, drop, stream_scale, block_scale, need_s):
    parts = [t for n in (post, pre) for t in ((None, None) if n is None else (n.weight, n.bias))]
    given = [block, stream, gate] + parts
    _refuse_tangents(*given)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
        conf = (post and (post.kind, post.eps), pre and (pre.kind, pre.eps), drop, float(stream_scale), float(block_scale), need_s)
        return JoinFunction.apply(*given, conf)
    s, y, _ = _forward(block, stream, post, gate, pre, drop, stream_scale, block_scale, need_s, False)
    return (s, y) if need_s and pre is not None else s if need_s else y


def join(block, stream=None, post=None, gate=None, pre=None, drop=None, stream_scale=1.0, block_scale=1.0, channel_axis=-1):
    """join_forward with gradients: s, or (s, y) with pre.  channel_axis: the axis of the channels in block and stream, so that 1 takes the (N, C, H, W) tensors of
    the convolutions; tensors in channel-last memory are used as they are, and the results are such.  Reverse mode, once."""
    if channel_axis not in (-1, block.dim() - 1):
        if stream is not None and stream.dim() != block.dim():
            raise ValueError("the stream has shape %r, expected that of the block, %r" % (tuple(stream.shape), tuple(block.shape)))
        out = join(_moved(block, channel_axis), _moved(stream, channel_axis), post, gate, pre, drop, stream_scale, block_scale)
        return tuple(t.movedim(-1, channel_axis) for t in out) if isinstance(out, tuple) else out.movedim(-1, channel_axis)
    return _call(block, stream, post, gate, pre, drop, stream_scale, block_scale, True)


def norm(x, norm, channel_axis=-1):
    """norm_forward with gradients; channel_axis as in join."""
    if channel_axis not in (-1, x.dim() - 1):
        return _call(_moved(x, channel_axis), None, None, None, norm, None, 1.0, 1.0, False).movedim(-1, channel_axis)
    return _call(x, None, None, None, norm, None, 1.0, 1.0, False)


def dropout(x, drop, channel_axis=-1):
    """dropout_forward with gradients; channel_axis as in join.  The mask goes by the channels, so it does not hang on how the tensor lies in memory."""
    if channel_axis not in (-1, x.dim() - 1):
        return dropout(_moved(x, channel_axis), drop).movedim(-1, channel_axis)
    return _call(x, None, None, None, None, drop, 1.0, 1.0, True)


class BlockNorm(nn.Module):
    """A norm over channels, beside WinoConv2d and MatrixLinear: "layer" with weight and bias or "rms" with a weight."""

    def __init__(self, channels, kind="layer", eps=1e-5, channel_axis=-1, device=None, dtype=None):
        super().__init__()
        Norm(kind, eps=eps)
        self.channels, self.kind, self.eps, self.channel_axis = channels, kind, eps, channel_axis
        self.weight = nn.Parameter(torch.ones(channels, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(channels, device=device, dtype=dtype)) if kind == "layer" else None

    def as_norm(self):
        return Norm(self.kind, self.weight, self.bias, self.eps)

    def forward(self, x):
        return norm(x, self.as_norm(), self.channel_axis)

    def extra_repr(self):
        return "%d, %r, eps=%g" % (self.channels, self.kind, self.eps)


# Passes that may be run again, of which a module keeps what they drew: 100 bytes each, with counter=True 512 of the GPU's
PASSES_KEPT = 4096


def _in_backward():
    """Whether this is run within a backward pass, as a checkpointed pass is the second time."""
    return torch._C._current_graph_task_id() != -1


def _may_run_again():
    """Whether the pass may be the first run of a checkpointed one, which has no gradients of its own or hooks on the tensors that it saves."""
    return not torch.is_grad_enabled() or torch._C._autograd._top_saved_tensors_default_hooks(True) is not None


class Dropout(nn.Module):
    """Dropout whose mask is never stored.  Each pass in training counts the offset up; the seed is drawn from torch's generator where none is given (and again for a
    copy.deepcopy, whose masks are its own), and both are in the state dict.  counter=True keeps them on the GPU, in the buffer `state`, so that a captured pass draws another
    mask in every replay (two small launches more a pass).

    A pass that torch.utils.checkpoint runs again in the backward pass takes the mask of its first run.  It is known by the state of torch's CPU generator, which checkpoint
    restores (preserve_rng_state) and from which passes without gradients or under saved-tensor hooks draw one number; in a backward pass a mask that is no earlier pass's, or
    that may be several's, is refused, as are those of captured passes with counter=True.  `dropout` and `join` with a Drop of one's own have no such passes."""

    def __init__(self, p=0.5, per="element", seed=None, counter=False, channel_axis=-1, device=None):
        super().__init__()
        self.drawn = seed is None
        seed = self._new_seed() if seed is None else seed
        Drop(p, seed, 0, per)
        self.p, self.per, self.channel_axis = p, per, channel_axis
        self._passes = {}                      # token of a pass: what it drew (None: one of several), whether it was run again
        if counter:
            if seed >= 1 << 63:
                raise ValueError("Dropout: seed %r in a buffer, from 0 to 2^63 - 1" % (seed,))
            self.register_buffer("state", torch.tensor([seed, 0], dtype=torch.int64, device=device))
        else:
            self.state, self.seed, self.calls = None, seed, 0

    @staticmethod
    def _new_seed():
        return int(torch.randint(0, 1 << 62, (1,)).item())

    def draw(self):
        """The Drop of the next pass; None where nothing is dropped."""
        if not self.training or Drop(self.p, 0).level == 0:
            return None
        again = _in_backward()
        # (a second run starts where torch's generator was, so it draws what the first run did)
        token = int(torch.randint(1 << 62, (), device="cpu")) if again or _may_run_again() else None
        if again:
            return self._drawn_by(token)
        if self.state is not None:
            used = self.state.clone()
            self.state[1].add_(1)
            drop = Drop(self.p, used, 0, self.per)
        else:
            self.calls += 1
            drop = Drop(self.p, self.seed, self.calls - 1, self.per)
        # (what a captured pass drew is the graph's)
        if token is not None and not (self.state is not None and self.state.is_cuda and torch.cuda.is_current_stream_capturing()):
            had = self._passes.pop(token, None)
            self._passes[token] = [drop if had is None or had[1] else None, False]
            if len(self._passes) > PASSES_KEPT:
                del self._passes[next(iter(self._passes))]
        return drop

    def _drawn_by(self, token):
        """The Drop of the first run of a pass."""
        found = self._passes.get(token)
        if found is None or found[0] is None:
            raise RuntimeError("Dropout: a pass run again in a backward pass starts at the state that torch's generator had the first time, no other pass's "
                               "(torch.utils.checkpoint with preserve_rng_state, which is its default); else give dropout or join a Drop")
        found[1] = True
        return found[0]

    def __getstate__(self):
        return {**self.__dict__, "_passes": {}}

    def __setstate__(self, state):
        super().__setstate__({"_passes": {}, "drawn": False, **state})

    def __deepcopy__(self, memo):
        made = type(self).__new__(type(self))
        memo[id(self)] = made
        made.__setstate__(copy.deepcopy(self.__getstate__(), memo))
        if made.drawn and made.state is not None:
            made.state[0] = self._new_seed()
        elif made.drawn:
            made.seed = self._new_seed()
        return made

    def get_extra_state(self):
        return None if self.state is not None else torch.tensor([self.seed - (1 << 64) if self.seed >> 63 else self.seed, self.calls])

    def set_extra_state(self, state):
        if state is not None and self.state is None:
            seed, self.calls = (int(v) for v in state)
            self.seed = seed % (1 << 64)

    def forward(self, x):
        drop = self.draw()
        return x if drop is None else dropout(x, drop, self.channel_axis)

    def extra_repr(self):
        return "p=%g, per=%r" % (self.p, self.per)


class ResidualStack(nn.Module):
    """Blocks along a stream: s = stream_scale s + block_scale gate drop(post(block(pre(s)))), and a norm behind the last.  A block is any module from (..., C) to the same
    shape, as matrix_block makes; with channel_axis=1 convolutions may be among them.  Each join, with the next block's norm, is one pass over memory.

    kind: of the norms; post: norms behind the blocks too; gate: the value that a learned gate a channel starts with, or None; drop: probability, a whole sample
    at a time (per="sample") or element by element.  A pass may be captured into a graph (counter=True draws another mask in every replay); as with every torch module, no eager
    autograd graph of the same parameters may be alive while a backward pass is captured."""

    def __init__(self, blocks, channels, kind="layer", eps=1e-5, post=False, gate=None, drop=0.0, per="sample", stream_scale=1.0, block_scale=1.0, counter=False,
                 channel_axis=-1, device=None, dtype=None):
        super().__init__()
        self.blocks = nn.ModuleList(blocks)
        n = len(self.blocks)
        make = lambda: BlockNorm(channels, kind, eps, channel_axis, device, dtype)  # noqa: E731
        self.pre = nn.ModuleList(make() for _ in range(n + 1))
        self.post = nn.ModuleList(make() for _ in range(n)) if post else None
        self.gates = None if gate is None else nn.ParameterList(nn.Parameter(torch.full((channels,), float(gate), device=device, dtype=dtype)) for _ in range(n))
        self.drops = nn.ModuleList(Dropout(drop, per, None, counter, channel_axis, device) for _ in range(n))
        self.stream_scale, self.block_scale, self.channel_axis = float(stream_scale), float(block_scale), channel_axis

    def forward(self, x):
        y = self.pre[0](x)
        for i, block in enumerate(self.blocks):
            x, y = join(block(y), x, self.post and self.post[i].as_norm(), None if self.gates is None else self.gates[i], self.pre[i + 1].as_norm(), self.drops[i].draw(),
                        self.stream_scale, self.block_scale, self.channel_axis)
        return y

    def pack4(self, x4=False):
        """This stack for serving: every MatrixLinear among its blocks and in them becomes a MatrixLinear4, one in several places one (in place; MatrixLinear.pack4)."""
        made = {}
        for parent in list(self.blocks.modules()):
            # (named_children would give a module that stands twice under one parent once)
            for name, child in list(parent._modules.items()):
                if isinstance(child, MatrixLinear):
                    if child not in made:
                        made[child] = child.pack4(x4)
                    setattr(parent, name, made[child])
        return self


def matrix_block(channels, hidden, activation="gelu", channel_axis=-1, checkpoint=None, device=None, dtype=None):
    """An expanding and a contracting layer, the block of a ResidualStack."""
    how = dict(checkpoint=checkpoint, channel_axis=channel_axis, device=device, dtype=dtype)
    return nn.Sequential(MatrixLinear(channels, hidden, activation=activation, **how), MatrixLinear(hidden, channels, **how))
