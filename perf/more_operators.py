"""What stands around and inside the linear layers of a residual block: products with weights (and activations) in microscaled 4-bit floating
point, and the passes that join a block to its stream - norm, dropout, gate, residual, the next block's norm - with their gradients.

A case is a dict of plain values:

  op          "pack": a tensor to 4 bits in groups of 32 channels and back;
              "linear": y = act(x wT + b) (+ r) with w in 4 bits; x as it is, or (x4) put into 4 bits within the call;
              "gradient": dx = (dy act'(z)) w of that layer, whose weight is frozen;
              "norm": y = norm(x), in training dx, dw and db too;
              "join": s = stream_scale x + block_scale gate * drop(post(f)), y = pre(s), in training all of their gradients too.  Without
              stream, norms and gate it is dropout
  dtype       type of the tensors: "float32", "float16", "bfloat16"
  rows, c, k  rows (pixels of all images), input channels, output channels ("linear", "gradient")
  act         "none", "relu", "gelu", "gelu_tanh", "silu"
  bias, residual ("linear"; the residual is added behind the activation)
  kind        "rms" or "layer" ("norm"); post, pre: the same or "none" ("join")
  gate        "none", "channel": (c), "sample": (samples, c)
  samples     images that the rows belong to, in equal shares
  stream      ("join") there is an x
  drop, per   probability; each "element" of its own or each "sample"
  train       gradients come out as well

4 bits (the OCP microscaling formats' MXFP4): the groups of 32 neighbouring channels of a row share a scale 2^e, e = floor(log2(largest magnitude)) - 2
but at least -127; a value is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times that, the nearest, ties to the even code, at most 6.

Dropout: channel c of row i is kept where word c % 8 of eight 16-bit words is at least round(65536 p); the words are the four of Philox4x32-10
with the counter (c / 8, i, offset's low half, its high half) and the key (seed's low half, its high half), low halves first (per "sample": word 0
of counter (0, sample, ...)).  What is kept is divided by the share 1 - round(65536 p) / 65536 that is.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_GROUP = 32
_EPS = 1e-5
_STREAM_SCALE, _BLOCK_SCALE = 0.875, 1.25


def _case(name, op, dtype, rows, c, **more):
    case = {"op": op, "dtype": dtype, "rows": rows, "c": c, "k": 0, "act": "none", "bias": False, "residual": False, "x4": False, "kind": "none",
            "post": "none", "pre": "none", "gate": "none", "samples": 1, "stream": False, "drop": 0.0, "per": "element", "train": False}
    case.update(more)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the weight of a large layer put into 4 bits
        _case("pack_bf16_8192_8192", "pack", "bfloat16", 8192, 8192),
        # a small ragged tensor in single precision
        _case("pack_f32_777_201", "pack", "float32", 777, 201),
        # one row through a 4096-channel layer: what a call costs when all that is read is half a byte a weight
        _case("linear_bf16_1_4096_4096", "linear", "bfloat16", 1, 4096, k=4096, bias=True),
        # the first classifier layer of a VGG-16 over a batch of 8, its weight in 4 bits
        _case("linear_f16_8_25088_4096_relu", "linear", "float16", 8, 25088, k=4096, act="relu", bias=True),
        # the expanding layer of a large batch, both operands in 4 bits: the most work
        _case("linear_bf16_8192_8192_8192_gelu_x4", "linear", "bfloat16", 8192, 8192, k=8192, act="gelu", bias=True, x4=True),
        # odd everything, a residual around the layer
        _case("linear_f16_1001_333_517_silu_residual_x4", "linear", "float16", 1001, 333, k=517, act="silu", residual=True, x4=True),
        # the gradient that passes through a frozen expanding layer
        _case("gradient_bf16_8192_2048_8192_gelu", "gradient", "bfloat16", 8192, 2048, k=8192, act="gelu"),
        # pixels of 56x56 images, N=64, normalised over 256 channels in a training step
        _case("norm_f16_200704_256_layer_train", "norm", "float16", 200704, 256, kind="layer", train=True),
        # one row
        _case("norm_bf16_1_4096_rms", "norm", "bfloat16", 1, 4096, kind="rms"),
        # behind a block of a large training step: its norm, dropout, gate and residual, and the next block's norm
        _case("join_bf16_16384_2048_rms_train", "join", "bfloat16", 16384, 2048, post="rms", pre="rms", gate="channel", stream=True, drop=0.1, train=True),
        # odd sizes in single precision: gated by the sample, whole samples dropped
        _case("join_f32_1001_333_layer_train", "join", "float32", 1001, 333, post="layer", pre="layer", gate="sample", samples=7, stream=True, drop=0.25,
              per="sample", train=True),
        # dropout by itself behind an activation, forward and backward
        _case("dropout_bf16_8192_8192_train", "join", "bfloat16", 8192, 8192, drop=0.1, train=True),
    ]


def _cost(case):
    rows, c, k = case["rows"], case["c"], case["k"]
    if case["op"] in ("linear", "gradient"):
        return 2.0 * rows * c * k / (4 if case["x4"] else 1) + 1000.0 * rows * (c + k)
    return 1000.0 * rows * c


def draw(rng):
    limit = max(_cost(c) for c in listed())

    def size(low, high):
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return v if rng.random() < 0.4 else max(low, (v + 4) // 8 * 8)
    while True:
        op = rng.choice(["pack", "linear", "linear", "linear", "gradient", "norm", "join", "join", "join"])
        dtype = rng.choice(["float32", "float16", "float16", "bfloat16", "bfloat16"])
        if op in ("linear", "gradient"):
            x4 = op == "linear" and rng.random() < 0.5
            case = _case(None, op, dtype, size(1, 16384), size(8, 25088), k=size(8, 8192), act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                         bias=op == "linear" and rng.random() < 0.7, residual=op == "linear" and rng.random() < 0.3, x4=x4)
            # (fp32 runs at a sixteenth of the 16-bit rate)
            if _cost(case) * (16 if dtype == "float32" else 1) <= limit and case["c"] * case["k"] <= 25088 * 4096:
                return case
            continue
        samples = rng.choice([1, size(1, 64)])
        rows = size(1, 200704)
        rows = max(rows // samples, 1) * samples
        c = size(3, 16384)
        if rows * c > 8192 * 8192:
            continue
        if op == "pack":
            return _case(None, op, dtype, rows, c)
        kinds = ["rms", "layer"]
        if op == "norm":
            return _case(None, op, dtype, rows, c, kind=rng.choice(kinds), train=rng.random() < 0.6)
        post, pre, stream = rng.choice(kinds + ["none"]), rng.choice(kinds + ["none"]), rng.random() < 0.8
        case = _case(None, op, dtype, rows, c, post=post, pre=pre, gate=rng.choice(["none", "channel", "sample"]), samples=samples, stream=stream,
                     drop=rng.choice([0.0, 0.1, round(rng.uniform(0.01, 0.9), 3)]), per=rng.choice(["element", "element", "sample"]), train=rng.random() < 0.6)
        if rows * c <= 16384 * 2048:
            return case


def _power(e):
    """2^e in float32 from whole numbers between -149 and 127."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _codes(x):
    """(codes, scales) of x (rows, c) in 4 bits: uint8 (rows, ceil(c / 2)), two codes to a byte, the lower channel in the low half, and uint8
    (rows, groups), e + 127."""
    rows, c = x.shape
    groups = -(-c // _GROUP)
    v = torch.nn.functional.pad(x.float(), (0, groups * _GROUP - c)).view(rows, groups, _GROUP)
    top = v.abs().amax(dim=-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(min=-127)
    a = (v.abs() * _power(-e)[..., None])
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = ((a / step).round() * step).clamp(max=6)
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(rows, groups * _GROUP)
    return (code[:, 0::2] | code[:, 1::2] << 4)[:, :(c + 1) // 2].contiguous(), (e + 127).to(torch.uint8)


def _values(codes, scales, c):
    """The float32 values (rows, c) that codes and scales stand for."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=-1).flatten(1)[:, :c]
    return v * _power(scales.to(torch.int32) - 127).repeat_interleave(_GROUP, dim=1)[:, :c]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    rows, c, k, n = case["rows"], case["c"], case["k"], case["samples"]
    # activations: channels of different ranges, as a network's are
    wide = lambda m: (normal(rows, m) * (0.3 + 1.4 * torch.rand(m, generator=g, device=dev))).to(t)  # noqa: E731
    s = {"case": case}
    if case["op"] in ("pack", "linear"):
        s["x"] = wide(c)
    if case["op"] in ("linear", "gradient"):
        # the weight was put into 4 bits when it was loaded
        w = normal(k, c) * (2.0 / c) ** 0.5
        s["w"] = _codes(w)
        del w
        if own:
            from pytorch_winoconv_amd.packed4 import Packed4
            s["w4"] = Packed4.from_parts(*s["w"], c, t)
        s["b"] = (0.1 * normal(k)).to(t) if case["bias"] else None
        s["r"] = normal(rows, k).to(t) if case["residual"] else None
    if case["op"] == "gradient":
        s["z"] = wide(k)
        s["dy"] = (normal(rows, k) / rows ** 0.5).to(t)
    shape = (n, rows // n, c)

    def parameters(kind):
        if kind == "none":
            return None
        return (1 + 0.2 * normal(c)).to(t), (0.2 * normal(c)).to(t) if kind == "layer" else None
    if case["op"] == "norm":
        s["x"] = (wide(c) + 0.3 * normal(c).to(t)).view(shape)
        s["norm"] = parameters(case["kind"])
        s["dy"] = (normal(*shape) / rows ** 0.5).to(t) if case["train"] else None
    if case["op"] == "join":
        s["f"] = wide(c).view(shape)
        s["x"] = (normal(*shape) + 0.3 * normal(c)).to(t) if case["stream"] else None
        s["post"], s["pre"] = parameters(case["post"]), parameters(case["pre"])
        s["gate"] = None if case["gate"] == "none" else (0.5 + 0.2 * normal(*((n, c) if case["gate"] == "sample" else (c,)))).to(t)
        s["seed"], s["offset"] = (int(v) for v in torch.randint(0, 1 << 62, (2,), generator=g, device=dev).tolist())
        if case["train"]:
            s["ds"] = (normal(*shape) / rows ** 0.5).to(t)
            s["dy"] = (normal(*shape) / rows ** 0.5).to(t) if case["pre"] != "none" else None
    return s


def _act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(z * -math.sqrt(0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    """The derivative of _act."""
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.special.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        th = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * a * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _normalised(x, kind):
    """(x - mean) / deviation and 1 / deviation; "rms": without the mean."""
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    inverse = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS)
    return x * inverse, inverse


def _norm(x, kind, p):
    v = _normalised(x, kind)[0] * p[0].float()
    return v if p[1] is None else v + p[1].float()


def _norm_gradient(dy, x, kind, p):
    """dx, dw and db (None without a bias)."""
    v, inverse = _normalised(x, kind)
    g = dy * p[0].float()
    dx = g - v * (g * v).mean(dim=-1, keepdim=True)
    if kind == "layer":
        dx = dx - g.mean(dim=-1, keepdim=True)
    return dx * inverse, (dy * v).sum(dim=(0, 1)), None if p[1] is None else dy.sum(dim=(0, 1))


def _philox(c0, c1, seed, offset):
    """The four 32-bit words of Philox4x32-10 (Salmon et al., 2011) in int64 tensors."""
    low = 0xFFFFFFFF
    x = [c0, c1, torch.full_like(c0, offset & low), torch.full_like(c0, offset >> 32)]
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p, q = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(q >> 32 & low) ^ x[1] ^ k0, q & low, (p >> 32 & low) ^ x[3] ^ k1, p & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return x


def _kept(case, seed, offset, device):
    """Whether each element is kept, (samples, rows / samples, c) or to be broadcast to it, and what the kept ones are multiplied by."""
    n, rows, c = case["samples"], case["rows"], case["c"]
    level = round(case["drop"] * 65536)
    i = torch.arange(n if case["per"] == "sample" else rows, device=device)
    j = torch.arange(1 if case["per"] == "sample" else -(-c // 8), device=device)
    words = _philox(*(v.contiguous() for v in torch.broadcast_tensors(j[None, :], i[:, None])), seed, offset)
    words = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=-1)
    kept = words >= level
    kept = kept[:, 0, 0].view(n, 1, 1) if case["per"] == "sample" else kept.flatten(1)[:, :c].view(n, rows // n, c)
    return kept, 65536 / (65536 - level) if level < 65536 else 0.0


def _run_plain(s):
    case = s["case"]
    t = _TYPES[case["dtype"]]
    c, act = case["c"], case["act"]
    if case["op"] == "pack":
        return _values(*_codes(s["x"]), c).to(t)
    if case["op"] == "linear":
        x = _values(*_codes(s["x"]), c) if case["x4"] else s["x"].float()
        z = x @ _values(*s["w"], c).t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(z, act)
        return (y if s["r"] is None else y + s["r"].float()).to(t)
    if case["op"] == "gradient":
        dz = s["dy"].float()
        if act != "none":
            dz = dz * _slope(s["z"].float(), act)
        return (dz @ _values(*s["w"], c)).to(t)
    if case["op"] == "norm":
        x = s["x"].float()
        out = {"y": _norm(x, case["kind"], s["norm"]).to(t)}
        if case["train"]:
            out.update(zip(("dx", "dw", "db"), (None if v is None else v.to(t) for v in _norm_gradient(s["dy"].float(), x, case["kind"], s["norm"]))))
        return {name: v for name, v in out.items() if v is not None}
    f = s["f"].float()
    v = f if s["post"] is None else _norm(f, case["post"], s["post"])
    if case["drop"]:
        kept, scale = _kept(case, s["seed"], s["offset"], f.device)
        drop = lambda u: torch.where(kept, u * scale, torch.zeros_like(u))  # noqa: E731
    else:
        drop = lambda u: u  # noqa: E731
    d = drop(v)
    gate = None if s["gate"] is None else s["gate"].float().view(case["samples"] if case["gate"] == "sample" else 1, 1, c)
    r = d if gate is None else gate * d
    if s["x"] is not None or gate is not None or s["post"] is not None or s["pre"] is not None:
        r = _BLOCK_SCALE * r
    if s["x"] is not None:
        r = r + _STREAM_SCALE * s["x"].float()
    out = {"s": r.to(t)}
    if s["pre"] is not None:
        out["y"] = _norm(r, case["pre"], s["pre"]).to(t)
    if not case["train"]:
        return out
    dr = s["ds"].float()
    if s["pre"] is not None:
        through, out["dpre_w"], out["dpre_b"] = _norm_gradient(s["dy"].float(), r, case["pre"], s["pre"])
        dr = dr + through
    if s["x"] is not None:
        out["dx"] = _STREAM_SCALE * dr
    dd = dr
    if s["x"] is not None or gate is not None or s["post"] is not None or s["pre"] is not None:
        dd = _BLOCK_SCALE * dd
    if gate is not None:
        out["dgate"] = (dd * d).sum(dim=1) if case["gate"] == "sample" else (dd * d).sum(dim=(0, 1))
        dd = dd * gate
    dv = drop(dd)
    if s["post"] is not None:
        dv, out["dpost_w"], out["dpost_b"] = _norm_gradient(dv, f, case["post"], s["post"])
    out["df"] = dv
    return {name: v.to(t) for name, v in out.items() if v is not None}


def _run_own(s):
    from pytorch_winoconv_amd import matrix_linear, packed4, residual
    case = s["case"]
    t = _TYPES[case["dtype"]]
    if case["op"] == "pack":
        return packed4.unpack4(packed4.pack4(s["x"]))
    if case["op"] == "linear":
        x = packed4.pack4(s["x"]) if case["x4"] else s["x"]
        return matrix_linear.linear_forward(x, s["w4"], s["b"], s["r"], case["act"], residual_after=True)
    if case["op"] == "gradient":
        return matrix_linear.linear_backward(s["dy"], None, s["w4"], s["z"] if case["act"] != "none" else None, case["act"], need_dw=False, need_db=False)[0]
    norm = lambda kind, p: None if p is None else residual.Norm(kind, p[0], p[1], _EPS)  # noqa: E731
    if case["op"] == "norm":
        n = norm(case["kind"], s["norm"])
        if not case["train"]:
            return {"y": residual.norm_forward(s["x"], n)}
        y, stats = residual.norm_forward(s["x"], n, keep=True)
        out = dict(zip(("dx", "dw", "db"), residual.norm_backward(s["dy"], s["x"], stats, n)), y=y)
        return {name: v for name, v in out.items() if v is not None}
    drop = residual.Drop(case["drop"], s["seed"], s["offset"], case["per"]) if case["drop"] else None
    if s["x"] is None and s["gate"] is None and s["post"] is None and s["pre"] is None:
        out = {"s": residual.dropout_forward(s["f"], drop)} if drop else {"s": s["f"]}
        if case["train"]:
            out["df"] = residual.dropout_forward(s["ds"], drop) if drop else s["ds"]
        return out
    how = dict(post=norm(case["post"], s["post"]), gate=s["gate"], pre=norm(case["pre"], s["pre"]), drop=drop,
               stream_scale=_STREAM_SCALE, block_scale=_BLOCK_SCALE)
    r, y, stats = residual.join_forward(s["f"], s["x"], keep=case["train"], **how)
    out = {"s": r, "y": y}
    if case["train"]:
        grads = residual.join_backward(s["ds"], s["dy"], s["f"], r, stats, need_stream=case["stream"], **how)
        out.update(df=grads.block, dx=grads.stream, dpost_w=grads.post_weight, dpost_b=grads.post_bias, dgate=grads.gate,
                   dpre_w=grads.pre_weight, dpre_b=grads.pre_bias)
    return {name: v for name, v in out.items() if v is not None}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    rows, c, k, size = case["rows"], case["c"], case["k"], 4 if case["dtype"] == "float32" else 2
    packed = lambda n, m: n * (-(-m // 2) + -(-m // _GROUP))  # noqa: E731
    if case["op"] == "pack":
        return {"bytes": 2 * rows * c * size, "flops": 4 * rows * c}
    if case["op"] == "linear":
        return {"bytes": size * (rows * c + rows * k * (1 + case["residual"]) + k * case["bias"]) + packed(k, c), "flops": 2 * rows * c * k + 8 * rows * k}
    if case["op"] == "gradient":
        return {"bytes": size * (rows * c + rows * k * (1 + (case["act"] != "none"))) + packed(k, c), "flops": 2 * rows * c * k + 12 * rows * k}
    parameters = lambda kind: {"none": 0, "rms": 1, "layer": 2}[kind]  # noqa: E731
    if case["op"] == "norm":
        n = parameters(case["kind"])
        return {"bytes": size * (rows * c * (4 if case["train"] else 2) + c * n * (2 if case["train"] else 1)), "flops": rows * c * (20 if case["train"] else 6)}
    pre = case["pre"] != "none"
    gate = {"none": 0, "channel": 1, "sample": case["samples"]}[case["gate"]]
    small = parameters(case["post"]) + parameters(case["pre"]) + gate
    # forward: f, x in, s, y out; backward: ds, dy in (what the forward pass read and wrote is counted there), df, dx out
    planes = 2 + case["stream"] + pre + (2 + pre + case["stream"] if case["train"] else 0)
    return {"bytes": size * (rows * c * planes + c * small * (2 if case["train"] else 1)),
            "flops": rows * c * (10 + 12 * bool(case["drop"])) * (3 if case["train"] else 1)}


_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)      # between one level and the next; the even of the two has it


def _exact_pack(x):
    x = x.to(torch.float64)
    out = torch.empty_like(x)
    for c0 in range(0, x.shape[1], _GROUP):
        part = x[:, c0:c0 + _GROUP]
        top = part.abs().max(dim=1, keepdim=True).values
        e = torch.where(top > 0, torch.floor(torch.log2(top)), torch.full_like(top, -200.0))
        e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e)) - 2
        scale = torch.exp2(e.clamp(min=-127))
        share = part.abs() / scale
        level = torch.zeros_like(share)
        for n, border in enumerate(_BORDERS):
            level = torch.where(share >= border if n % 2 else share > border, _LEVELS[n + 1], level)
        out[:, c0:c0 + _GROUP] = torch.copysign(level, part) * scale
    return out


def _exact_values(codes, scales, c):
    low, high = (torch.tensor(_LEVELS, dtype=torch.float64, device=codes.device)[(codes >> n & 7).long()] * (1.0 - 2.0 * (codes >> n + 3 & 1))
                 for n in (0, 4))
    v = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    v[:, 0::2], v[:, 1::2] = low, high
    scale = torch.exp2(scales.to(torch.float64) - 127)
    return v[:, :c] * scale[:, torch.arange(c, device=codes.device) // _GROUP]


def _exact_kept(case, seed, offset):
    """As _kept, by numpy in unsigned arithmetic."""
    n, rows, c = case["samples"], case["rows"], case["c"]
    sample = case["per"] == "sample"
    count, width = (n, 1) if sample else (rows, -(-c // 8))
    x0 = np.tile(np.arange(width, dtype=np.uint64), count)
    x1 = np.repeat(np.arange(count, dtype=np.uint64), width)
    x2, x3 = (np.full(count * width, (offset >> b) % (1 << 32), dtype=np.uint64) for b in (0, 32))
    half, low = np.uint64(32), np.uint64(0xFFFFFFFF)
    for r in range(10):
        keys = [np.uint64(((seed >> b) + r * w) % (1 << 32)) for b, w in ((0, 0x9E3779B9), (32, 0xBB67AE85))]
        p, q = np.uint64(0xD2511F53) * x0, np.uint64(0xCD9E8D57) * x2
        x0, x1, x2, x3 = (q >> half) ^ x1 ^ keys[0], q & low, (p >> half) ^ x3 ^ keys[1], p & low
    words = np.empty((count, width, 8), dtype=np.uint16)
    for m, x in enumerate((x0, x1, x2, x3)):
        words[:, :, 2 * m] = (x % np.uint64(1 << 16)).reshape(count, width)
        words[:, :, 2 * m + 1] = (x >> np.uint64(16)).reshape(count, width)
    level = round(case["drop"] * 65536)
    share = (65536 - level) / 65536
    kept = torch.from_numpy(words.reshape(count, width * 8).astype(np.int32) >= level)
    kept = kept[:, :1].view(n, 1, 1) if sample else kept[:, :c].view(n, rows // n, c)
    return kept.cuda(), share


def _exact_norm(x, kind, p):
    if kind == "layer":
        return torch.nn.functional.layer_norm(x, x.shape[-1:], p[0], p[1], _EPS)
    return x / torch.sqrt(x.pow(2).mean(dim=-1, keepdim=True) + _EPS) * p[0]


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda v: None if v is None else v.to(torch.float64)  # noqa: E731
    c, act = case["c"], case["act"]
    if case["op"] == "pack":
        return _exact_pack(s["x"])
    if case["op"] == "linear":
        x = _exact_pack(s["x"]) if case["x4"] else wide(s["x"])
        z = torch.nn.functional.linear(x, _exact_values(*s["w"], c), wide(s["b"]))
        y = {"none": lambda v: v, "relu": torch.relu, "gelu": lambda v: v * torch.special.ndtr(v),
             "gelu_tanh": lambda v: v * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3)),
             "silu": lambda v: v * torch.sigmoid(v)}[act](z)
        return y if s["r"] is None else y + wide(s["r"])
    if case["op"] == "gradient":
        z, dz = wide(s["z"]), wide(s["dy"])
        if act == "relu":
            dz = torch.where(z > 0, dz, torch.zeros_like(dz))
        elif act == "gelu":
            dz = dz * (torch.special.ndtr(z) + z * torch.exp(-z ** 2 / 2) / (2 * math.pi) ** 0.5)
        elif act == "gelu_tanh":
            a = 2 * (2 / math.pi) ** 0.5
            g = torch.sigmoid(a * (z + 0.044715 * z ** 3))
            dz = dz * (g + z * g * (1 - g) * a * (1 + 0.134145 * z ** 2))
        elif act == "silu":
            g = torch.sigmoid(z)
            dz = dz * (g + z * g * (1 - g))
        return torch.matmul(dz, _exact_values(*s["w"], c))

    # the gradients by differentiating the definition in 64 bits
    leaves = {}

    def leaf(name, v):
        if v is None:
            return None
        leaves[name] = wide(v).requires_grad_(case["train"])
        return leaves[name]
    if case["op"] == "norm":
        x, p = leaf("dx", s["x"]), (leaf("dw", s["norm"][0]), leaf("db", s["norm"][1]))
        out, given = {"y": _exact_norm(x, case["kind"], p)}, {"y": wide(s["dy"])}
    else:
        f, x, gate = leaf("df", s["f"]), leaf("dx", s["x"]), leaf("dgate", s["gate"])
        v = f
        if s["post"] is not None:
            v = _exact_norm(v, case["post"], (leaf("dpost_w", s["post"][0]), leaf("dpost_b", s["post"][1])))
        if case["drop"]:
            kept, share = _exact_kept(case, s["seed"], s["offset"])
            v = torch.where(kept, v / share, torch.zeros_like(v)) if share else torch.zeros_like(v) * f
        if gate is not None:
            v = v * (gate[:, None, :] if case["gate"] == "sample" else gate)
        if len(leaves) > 1 or s["pre"] is not None:
            v = v * _BLOCK_SCALE
        if x is not None:
            v = v + x * _STREAM_SCALE
        out, given = {"s": v}, {"s": wide(s.get("ds"))}
        if s["pre"] is not None:
            out["y"] = _exact_norm(v, case["pre"], (leaf("dpre_w", s["pre"][0]), leaf("dpre_b", s["pre"][1])))
            given["y"] = wide(s.get("dy"))
    if case["train"]:
        names = sorted(leaves)
        grads = torch.autograd.grad([out[n] for n in sorted(out)], [leaves[n] for n in names], [given[n] for n in sorted(out)])
        out.update(zip(names, grads))
    return {n: v.detach() for n, v in out.items()}
