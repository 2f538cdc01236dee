"""Joins, norms and dropout in 64 bits, by differentiating the definition, with bounds on what fp32 arithmetic and one rounding may be off by
(test infrastructure)."""
import numpy as np
import torch

SUM = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def words(rows, C, seed, offset, first=0):
    """Of rows `first` and on, the eight 16-bit words of Philox4x32-10 for every eight channels, (rows, 8 ceil(C / 8)), in Python's whole numbers by numpy's unsigned ones."""
    width = -(-C // 8)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    x = [np.tile(np.arange(width, dtype=np.uint64), rows), np.repeat(np.arange(first, first + rows, dtype=np.uint64), width), np.full(rows * width, offset & 0xFFFFFFFF, dtype=np.uint64),
         np.full(rows * width, offset >> 32, dtype=np.uint64)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(q >> half) ^ x[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ x[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    out = np.stack([h for v in x for h in (v & np.uint64(0xFFFF), v >> np.uint64(16))], axis=-1)
    return torch.from_numpy(out.astype(np.int64)).view(rows, width * 8)


def mask(shape, p, seed, offset, per):
    """What f of this shape is multiplied by, float64, 0 or 1 / share."""
    level = int(round(p * 65536))
    rows, C = 1, shape[-1]
    for v in shape[:-1]:
        rows *= v
    if per == "sample":
        n = shape[0] if len(shape) > 1 else 1
        kept = (words(n, 1, seed, offset)[:, 0] >= level).view((n,) + (1,) * (len(shape) - 1)) if len(shape) > 1 else words(1, 1, seed, offset)[0, 0] >= level
        kept = kept.expand(shape)
    else:
        kept = (words(rows, C, seed, offset)[:, :C] >= level).view(shape)
    return kept, 65536 / (65536 - level) if level < 65536 else 0.0


def norm(v, kind, w, b, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + eps)
    if w is not None:
        v = v * w
    return v if b is None else v + b


def join(f, x, gate, post, pre, drop, a, b):
    """(s, y) in 64 bits; post, pre: (kind, weight, bias, eps) or None; drop: (p, seed, offset, per) or None."""
    v = f if post is None else norm(f, *post)
    if drop is not None:
        kept, scale = mask(tuple(f.shape), *drop)
        v = torch.where(kept, v * scale, torch.zeros_like(v))
    if gate is not None:
        v = v * (gate if gate.dim() == 1 else gate.view((gate.shape[0],) + (1,) * (f.dim() - 2) + (gate.shape[1],)))
    v = b * v
    if x is not None:
        v = v + a * x
    return v, None if pre is None else norm(v, *pre)


# What an fp32 mean, variance, inverse deviation or product of a row may be off by, relative to the row's values: a thread adds at most 32 values of a vector, a team at
# most 64 lanes and 16 wavefronts in 6 and 16 steps (rows beyond registers: C / 1024 more), each a rounding of SUM; a dozen more roundings, a reciprocal and a
# root.  128 roundings in all, doubled for those of the mean within the variance.
def roundings(C):
    return (256 + C / 512) * SUM


def _hat(v, n):
    """(v^, inverse deviation, how much larger than what is left of them the values are that the mean is taken off)."""
    kind, w, b, eps = n
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    inverse = 1 / torch.sqrt((v - mean).pow(2).mean(-1, keepdim=True) + eps)
    return (v - mean) * inverse, mean, inverse, 1 + v.abs().amax(-1, keepdim=True) * inverse


def forward(f, x, gate, post, pre, drop, a, b):
    """(s, y, bound of s, bound of y, bound of s before its rounding) of CPU tensors of one type, before the roundings of s and y to it, which are added here."""
    t, wide = f.dtype, lambda v: None if v is None else v.double()  # noqa: E731
    u, E = half_step(t), roundings(f.shape[-1])
    F, X, G = wide(f), wide(x), wide(gate)
    post, pre = (None if n is None else (n[0], wide(n[1]), wide(n[2]), n[3]) for n in (post, pre))
    s, _ = join(F, X, G, post, None, drop, a, b)
    # what s is off by before its rounding: of the block's share, and of the stream's
    share = join(F, None, G, post, None, drop, a, b)[0].abs()
    off = 4 * SUM * (s.abs() + share + (0 if X is None else abs(a) * X.abs()))
    if post is not None:
        hat, _, _, large = _hat(F, post)
        scale = torch.ones_like(F) if G is None else G if G.dim() == 1 else G.view((G.shape[0],) + (1,) * (F.dim() - 2) + (G.shape[1],))
        w = 1 if post[1] is None else post[1]
        kept = mask(tuple(F.shape), *drop)[1] if drop is not None else 1.0
        off = off + E * large * (hat.abs() + 1) * (w * scale * b * kept).abs() + 4 * SUM * (0 if post[2] is None else (post[2] * scale * b * kept).abs())
    by_s = off * (1 + u) + u * s.abs() + least(t)
    if pre is None:
        return s, None, by_s, None, off
    hat, _, inverse, large = _hat(s, pre)
    w = torch.ones(s.shape[-1], dtype=torch.float64) if pre[1] is None else pre[1]
    y = hat * w + (0 if pre[2] is None else pre[2])
    # s moves y by its own error, by that of the mean (the largest of the row's) and, times s^, by that of the deviation
    moved = inverse * off.amax(-1, keepdim=True) * (2 + 2 * hat.abs())
    off_y = (moved + E * large * (hat.abs() + 1)) * w.abs() + 4 * SUM * y.abs()
    return s, y, by_s, off_y * (1 + u) + u * y.abs() + least(t), off


def _through(dh, dh_off, n, v, E, v_off=None):
    """(gradient, its bound, dw, db and their bounds) of a norm of v with dh its result's gradient, off by dh_off; v_off: what v is off by."""
    hat, _, inverse, large = _hat(v, n)
    moved = 0 if v_off is None else inverse * v_off.amax(-1, keepdim=True) * (2 + 2 * hat.abs())
    w = torch.ones(v.shape[-1], dtype=torch.float64) if n[1] is None else n[1]
    g = dh * w
    out = g - hat * (g * hat).mean(-1, keepdim=True)
    if n[0] == "layer":
        out = out - g.mean(-1, keepdim=True)
    top = g.abs().amax(-1, keepdim=True) + (dh_off * w.abs()).amax(-1, keepdim=True)
    off = inverse * ((E * large * (2 + 2 * hat.abs()) + (0 if v_off is None else moved + moved.amax(-1, keepdim=True) * (1 + hat.abs()))) * top * 2 + (dh_off * w.abs()).amax(-1, keepdim=True) * (2 + hat.abs()))
    axes = tuple(range(v.dim() - 1))
    rows = v.numel() // v.shape[-1]
    hat_off = E * large * (hat.abs() + 1) + moved
    dw, dw_off = (dh * hat).sum(axes), (dh.abs() * hat_off + dh_off * (hat.abs() + hat_off)).sum(axes) + (rows + 8) * SUM * (dh * hat).abs().sum(axes)
    db, db_off = dh.sum(axes), dh_off.sum(axes) + (rows + 8) * SUM * dh.abs().sum(axes)
    return out * inverse, off, dw, dw_off, db, db_off


def backward(ds, dy, f, s, gate, post, pre, drop, a, b, s_exact=None, s_off=None):
    """{name: (value, bound)} of the gradients in the names of residual.Gradients, from s, off by s_off; its statistics are those of s_exact (of s where it is None)."""
    t, wide = f.dtype, lambda v: None if v is None else v.double()  # noqa: E731
    u, E = half_step(t), roundings(f.shape[-1])
    F, G = wide(f), wide(gate)
    post_like, pre_like = post, pre
    post, pre = (None if n is None else (n[0], wide(n[1]), wide(n[2]), n[3]) for n in (post, pre))
    out = {}

    def put(name, v, off, like):
        if like is None:
            return
        u = half_step(like.dtype)
        out[name] = (v, off * (1 + u) + u * v.abs() + least(like.dtype))
    dr = torch.zeros_like(F) if ds is None else wide(ds)
    off = torch.zeros_like(dr)
    if pre is not None and dy is not None:
        S = wide(s)
        through, off, dw, dw_off, db, db_off = _through(wide(dy), torch.zeros_like(dr), pre, S, E, s_off)
        if s_exact is not None:
            # the rounding moved s^ by u times s, which the statistics did not see
            hat, _, inverse, _ = _hat(s_exact, pre)
            g = wide(dy) * (1 if pre[1] is None else pre[1])
            mine = (S - _hat(s_exact, pre)[1]) * inverse
            through = g - mine * (g * mine).mean(-1, keepdim=True)
            if pre[0] == "layer":
                through = through - g.mean(-1, keepdim=True)
            through = through * inverse
            dw = (wide(dy) * mine).sum(tuple(range(F.dim() - 1)))
        dr = dr + through
        put("pre_weight", dw, dw_off, pre_like[1])
        put("pre_bias", db, db_off, pre_like[2])
    off = off + SUM * dr.abs()
    put("stream", a * dr, abs(a) * off + SUM * (a * dr).abs(), f)
    dd, dd_off = b * dr, abs(b) * off + SUM * (b * dr).abs()
    kept, scale = (torch.ones_like(F, dtype=torch.bool), 1.0) if drop is None else mask(tuple(F.shape), *drop)
    gate_of = None if G is None else G if G.dim() == 1 else G.view((G.shape[0],) + (1,) * (F.dim() - 2) + (G.shape[1],))
    if G is not None:
        n = F if post is None else norm(F, *post)
        n_off = torch.zeros_like(F)
        if post is not None:
            hat, _, _, large = _hat(F, post)
            n_off = E * large * (hat.abs() + 1) * (1 if post[1] is None else post[1].abs()) + 4 * SUM * n.abs()
        d = torch.where(kept, n * scale, torch.zeros_like(n))
        term, term_off = dd * d, dd_off * (d.abs() + n_off * scale) + dd.abs() * (n_off * scale + 4 * SUM * d.abs())
        axes = tuple(range(F.dim() - 1)) if G.dim() == 1 else tuple(range(1, F.dim() - 1))
        rows = F.numel() // F.shape[-1]
        v, v_off = (term.sum(axes), term_off.sum(axes) + (rows + 8) * SUM * term.abs().sum(axes)) if axes else (term, term_off)
        put("gate", v, v_off, gate)
        dd, dd_off = dd * gate_of, dd_off * gate_of.abs() + SUM * (dd * gate_of).abs()
    dv = torch.where(kept, dd * scale, torch.zeros_like(dd))
    dv_off = torch.where(kept, dd_off * scale + 2 * SUM * dv.abs(), torch.zeros_like(dd))
    if post is not None:
        dv, dv_off, dw, dw_off, db, db_off = _through(dv, dv_off, post, F, E)
        put("post_weight", dw, dw_off, post_like[1])
        put("post_bias", db, db_off, post_like[2])
    put("block", dv, dv_off, f)
    return out


def within(got, want, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), "%s: %g over a bound of %g at %r" % (what, float(over.max()), float(bound.flatten()[over.argmax()]), int(over.argmax()))


def of_s(s, want):
    """What `backward` takes for s and after it: s as it was rounded with the statistics of the exact one, or, of 16-bit types, which compute it again, the exact one."""
    return dict(s=s.detach().cpu(), s_exact=want[0]) if s.dtype == torch.float32 else dict(s=want[0], s_off=want[4])
