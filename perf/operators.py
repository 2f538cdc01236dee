"""Matrix products with bias, activation and residual in their epilogue, their gradients, and activations kept in 8 bits for
the backward pass: the layers that stand between, before and behind the convolutions of a network (1x1 convolutions of channel-last
pixels, expanding and contracting layers, classifiers).

A case is a dict of plain values:

  op          "linear": y = act(x wT + b + r), or act(x wT + b) + r;
              "gradient": dx, dw, db (and dz, the gradient of what the activation takes, which is the residual's too) from dy, x, w
              and z = x wT + b + r;
              "pack": a tensor to 8 bits in groups of 32 channels and back
  dtype       type of the tensors: "float32", "float16", "bfloat16"
  rows, c, k  rows (pixels of all images), input channels, output channels ("pack": c alone)
  act         "none", "relu", "gelu", "gelu_tanh", "silu"
  bias        the layer has one
  residual    "none", "before" (added before the activation) or "after" it ("gradient": "before" asks for dz as well)
  keep        (linear) z comes out as well, as a pass that is trained needs it
  bits8       (gradient) x and z were kept in 8 bits

8 bits: the groups of 32 neighbouring channels of a row share a step 2^e, e = floor(log2(largest magnitude)) - 6 but at
least -126; a value is kept as the whole number nearest to its share of the step, ties to even, at most 127 either way.
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_GROUP = 32


def _case(name, op, dtype, rows, c, k=0, act="none", bias=True, residual="none", keep=False, bits8=False):
    case = {"op": op, "dtype": dtype, "rows": rows, "c": c, "k": k, "act": act, "bias": bias, "residual": residual, "keep": keep, "bits8": bits8}
    return dict(case, name=name) if name else case


def listed():
    return [
        # the classifier of one image: what a call costs when the arithmetic is nothing
        _case("linear_bf16_1_4096_1000", "linear", "bfloat16", 1, 4096, 1000),
        # the first classifier layer of a VGG-16 over a batch of 8: a large weight that is read once
        _case("linear_f16_8_25088_4096_relu", "linear", "float16", 8, 25088, 4096, "relu"),
        # the expanding 1x1 convolution of a ResNet bottleneck, N=64 at 56x56, with the block's residual
        _case("linear_f16_200704_64_256_relu_residual", "linear", "float16", 200704, 64, 256, "relu", residual="before"),
        # an expanding layer of a large training step, which keeps what its activation takes
        _case("linear_bf16_8192_2048_8192_gelu", "linear", "bfloat16", 8192, 2048, 8192, "gelu", keep=True),
        # single precision, odd everything, no bias, a residual around the layer
        _case("linear_f32_1001_333_517_silu_residual", "linear", "float32", 1001, 333, 517, "silu", bias=False, residual="after"),
        # a classifier layer's training step over a batch of 8
        _case("gradient_f16_8_4096_4096_relu", "gradient", "float16", 8, 4096, 4096, "relu"),
        # the expanding 1x1 convolution at 28x28 with the gradient of the block's residual
        _case("gradient_f16_50176_128_512_relu_residual", "gradient", "float16", 50176, 128, 512, "relu", residual="before"),
        # the expanding layer of the large training step: the largest case
        _case("gradient_bf16_8192_2048_8192_gelu", "gradient", "bfloat16", 8192, 2048, 8192, "gelu"),
        # a layer at 14x14 whose activations were kept in 8 bits
        _case("gradient_f16_12544_256_1024_silu_8bit", "gradient", "float16", 12544, 256, 1024, "silu", bits8=True),
        # the same, small and ragged
        _case("gradient_bf16_777_201_119_gelu_tanh_8bit", "gradient", "bfloat16", 777, 201, 119, "gelu_tanh", bits8=True),
        # activations of 56x56 pixels, N=64, kept for the backward pass
        _case("pack_f16_200704_256", "pack", "float16", 200704, 256),
        # a small ragged tensor
        _case("pack_bf16_49_77", "pack", "bfloat16", 49, 77),
    ]


def _cost(case):
    return 2.0 * case["rows"] * case["c"] * case["k"] * (2 if case["op"] == "gradient" else 1) + 1000.0 * case["rows"] * (case["c"] + case["k"])


def draw(rng):
    limit = max(_cost(c) for c in listed())

    def size(low, high):
        v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return v if rng.random() < 0.4 else max(low, (v + 4) // 8 * 8)
    while True:
        op = rng.choice(["linear", "linear", "gradient", "gradient", "pack"])
        dtype = rng.choice(["float32", "float16", "float16", "bfloat16", "bfloat16"])
        if op == "pack":
            case = _case(None, op, dtype, size(1, 200704), size(3, 4096))
            if case["rows"] * case["c"] <= 200704 * 256:
                return case
            continue
        act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
        residual = rng.choice(["none", "before", "after"])
        case = _case(None, op, dtype, size(1, 200704), size(8, 25088), size(8, 8192), act, rng.random() < 0.8, residual,
                     op == "linear" and act != "none" and rng.random() < 0.5, op == "gradient" and rng.random() < 0.4)
        # (fp32 runs at a sixteenth of the 16-bit rate)
        cost = _cost(case) * (16 if dtype == "float32" else 1)
        if cost <= limit and max(case["rows"] * case["c"], case["rows"] * case["k"], case["c"] * case["k"]) <= 25088 * 4096:
            return case


def _step(e):
    """2^e in float32 from whole numbers of -126 and more: its exponent's bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(x):
    """(codes, exponents) of x (rows, c) in 8 bits: int8 (rows, c) and (rows, groups)."""
    rows, c = x.shape
    groups = -(-c // _GROUP)
    v = torch.nn.functional.pad(x.float(), (0, groups * _GROUP - c)).view(rows, groups, _GROUP)
    top = v.abs().amax(dim=-1)
    e = ((top.view(torch.int32) >> 23) - 127 - 6).clamp(min=-126)
    q = (v * _step(-e)[..., None]).round().clamp(-127, 127).view(rows, groups * _GROUP)[:, :c]
    return q.to(torch.int8), e.to(torch.int8)


def _values(codes, e):
    """The float32 values that codes and exponents stand for."""
    return codes.float() * _step(e).repeat_interleave(_GROUP, dim=1)[:, :codes.shape[1]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    rows, c, k = case["rows"], case["c"], case["k"]
    # activations: channels of different ranges, as a network's are
    x = (normal(rows, c) * (0.3 + 1.4 * torch.rand(c, generator=g, device=dev))).to(t)
    state = {"case": case, "x": x}
    if case["op"] == "pack":
        return state
    state["w"] = (normal(k, c) * (2.0 / c) ** 0.5).to(t)
    state["b"] = (0.1 * normal(k)).to(t) if case["bias"] else None
    state["r"] = normal(rows, k).to(t) if case["residual"] != "none" else None
    if case["op"] == "gradient":
        z = x.float() @ state["w"].float().t()
        if state["b"] is not None:
            z += state["b"].float()
        if case["residual"] == "before":
            z += state["r"].float()
        state["z"] = z.to(t)
        del z, state["r"]
        state["dy"] = (normal(rows, k) / rows ** 0.5).to(t)
        if case["bits8"]:
            state["x"] = _codes(x)
            state["z"] = _codes(state["z"])
    return state


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


def _run_plain(s):
    case = s["case"]
    t = _TYPES[case["dtype"]]
    if case["op"] == "pack":
        return _values(*_codes(s["x"])).to(t)
    w = s["w"].float()
    if case["op"] == "linear":
        z = s["x"].float() @ w.t()
        if s["b"] is not None:
            z = z + s["b"].float()
        if case["residual"] == "before":
            z = z + s["r"].float()
        y = _act(z, case["act"])
        if case["residual"] == "after":
            y = y + s["r"].float()
        return {"y": y.to(t), "z": z.to(t)} if case["keep"] else y.to(t)
    x = _values(*s["x"]) if case["bits8"] else s["x"].float()
    dz = s["dy"].float()
    if case["act"] != "none":
        dz = dz * _slope(_values(*s["z"]) if case["bits8"] else s["z"].float(), case["act"])
    out = {"dx": (dz @ w).to(t), "dw": (dz.t() @ x).to(t)}
    if case["bias"]:
        out["db"] = dz.sum(dim=0).to(t)
    if case["residual"] == "before":
        out["dz"] = dz.to(t)
    return out


def _run_own(s):
    from pytorch_winoconv_amd import checkpoint8, matrix_linear
    case = s["case"]
    t = _TYPES[case["dtype"]]
    if case["op"] == "pack":
        return checkpoint8.unpack8(checkpoint8.pack8(s["x"]))
    if case["op"] == "linear":
        y = matrix_linear.linear_forward(s["x"], s["w"], s["b"], s["r"], case["act"], residual_after=case["residual"] == "after",
                                         keep_z=case["keep"])
        return {"y": y[0], "z": y[1]} if case["keep"] else y
    x, z = s["x"], s["z"]
    if case["bits8"]:
        x, z = checkpoint8.Packed8(*x, t), checkpoint8.Packed8(*z, t)
    dx, dw, db, dz = matrix_linear.linear_backward(s["dy"], x, s["w"], z if case["act"] != "none" else None, case["act"],
                                                   need_db=case["bias"], need_dz=case["residual"] == "before")
    out = {"dx": dx, "dw": dw}
    if case["bias"]:
        out["db"] = db
    if case["residual"] == "before":
        out["dz"] = dz
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    rows, c, k, s = case["rows"], case["c"], case["k"], 4 if case["dtype"] == "float32" else 2
    if case["op"] == "pack":
        return {"bytes": 2 * rows * c * s, "flops": 4 * rows * c}
    product = 2 * rows * c * k
    if case["op"] == "linear":
        wide = 1 + (case["residual"] != "none") + bool(case["keep"])
        return {"bytes": s * (rows * c + c * k + rows * k * wide + k * case["bias"]), "flops": product + 8 * rows * k}
    packed = (lambda n: rows * n + rows * -(-n // _GROUP)) if case["bits8"] else (lambda n: rows * n * s)
    return {"bytes": packed(c) + (packed(k) if case["act"] != "none" else 0) + s * (rows * k + rows * c + 2 * c * k + k * case["bias"]
                                                                                     + rows * k * (case["residual"] == "before")),
            "flops": 2 * product + 12 * rows * k}


def _exact_values(kept):
    codes, e = kept
    wide = e.to(torch.int64).repeat_interleave(_GROUP, dim=1)[:, :codes.shape[1]]
    return torch.ldexp(codes.to(torch.float64), wide)


def _normal_cdf(z):
    return torch.special.ndtr(z)


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda v: v.to(torch.float64)  # noqa: E731
    if case["op"] == "pack":
        x = wide(s["x"])
        out = torch.empty_like(x)
        for c0 in range(0, case["c"], _GROUP):
            part = x[:, c0:c0 + _GROUP]
            top = part.abs().max(dim=1, keepdim=True).values
            e = torch.where(top > 0, torch.frexp(top).exponent - 7, torch.full_like(top, -126, dtype=torch.int32)).clamp(min=-126)
            share = torch.ldexp(part, -e)
            low = torch.floor(share)
            up = (share - low > 0.5) | ((share - low == 0.5) & (torch.remainder(low, 2) == 1))
            out[:, c0:c0 + _GROUP] = torch.ldexp(torch.where(up, low + 1, low).clamp(-127, 127), e)
        return out
    act, w = case["act"], wide(s["w"])
    if case["op"] == "linear":
        z = torch.nn.functional.linear(wide(s["x"]), w, None if s["b"] is None else wide(s["b"]))
        if case["residual"] == "before":
            z += wide(s["r"])
        y = {"none": lambda v: v.clone(), "relu": torch.relu, "gelu": lambda v: v * _normal_cdf(v),
             "gelu_tanh": lambda v: v * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (v + 0.044715 * v ** 3)),
             "silu": lambda v: v * torch.sigmoid(v)}[act](z)
        if case["residual"] == "after":
            y += wide(s["r"])
        return {"y": y, "z": z} if case["keep"] else y
    x = _exact_values(s["x"]) if case["bits8"] else wide(s["x"])
    dz = wide(s["dy"])
    if act != "none":
        z = _exact_values(s["z"]) if case["bits8"] else wide(s["z"])
        if act == "relu":
            dz = torch.where(z > 0, dz, torch.zeros_like(dz))
        elif act == "gelu":
            dz = dz * (_normal_cdf(z) + z * torch.exp(-z ** 2 / 2) / (2 * math.pi) ** 0.5)
        elif act == "gelu_tanh":
            a = 2 * (2 / math.pi) ** 0.5
            g = torch.sigmoid(a * (z + 0.044715 * z ** 3))
            dz = dz * (g + z * g * (1 - g) * a * (1 + 0.134145 * z ** 2))
        else:
            g = torch.sigmoid(z)
            dz = dz * (g + z * g * (1 - g))
    out = {"dx": torch.matmul(dz, w), "dw": torch.matmul(dz.t(), x)}
    if case["bias"]:
        out["db"] = dz.sum(0)
    if case["residual"] == "before":
        out["dz"] = dz
    return out
