"""Cases of the 8-bit linear layers: quantising activations by token, the product of 8-bit integers with scales for each token
and channel, and the norms around a block with its gate and residual scale.  ``run`` computes a case either in plain torch
operations or through the package."""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_LEAST = 2.0 ** -100           # smallest absolute maximum that a row's scale is made of
_TOP = 127.0


# ---------------------------------------------------------------------------------------------------------------- cases

def _quantize(name, rows, width, dtype, rotate):
    return {"name": name, "op": "quantize", "rows": rows, "width": width, "dtype": dtype, "rotate": rotate}


def _linear(name, rows, width, out, dtype, rotate=False, bias=False):
    return {"name": name, "op": "linear", "rows": rows, "width": width, "out": out, "dtype": dtype, "rotate": rotate, "bias": bias}


def _norm(name, groups, each, width, dtype, kind="rms", residual="", post=False, gate="", scale=1.0, bias=False):
    """`groups` sequences or images of `each` tokens; `residual`: the type of the residual stream, "" for the block's."""
    return {"name": name, "op": "norm", "groups": groups, "each": each, "width": width, "dtype": dtype, "kind": kind,
            "residual": residual or dtype, "post": post, "gate": gate, "scale": scale, "bias": bias}


def _block(name, rows, width, out, small, dtype, rotate=False, post=False):
    return {"name": name, "op": "block", "rows": rows, "width": width, "out": out, "small": small, "dtype": dtype, "rotate": rotate,
            "post": post}


def listed():
    return [
        # activations of a serving batch's decode step, quantised once for several products; latency counts
        _quantize("quantize_step", 64, 8192, "bf16", False),
        # what goes into the down projection of a batch of prompts, rotated
        _quantize("quantize_prompt", 8191, 11008, "bf16", True),
        # one user's single token through one matrix; latency counts
        _linear("linear_one", 1, 4096, 11008, "bf16"),
        # a decode step of 48 sequences through a large matrix: reading the weights
        _linear("linear_batch", 48, 8192, 28672, "bf16"),
        # a prompt of 2048 tokens, rotated
        _linear("linear_prompt", 2048, 4096, 11008, "bf16", rotate=True),
        # prompts of a batch through a large matrix
        _linear("linear_large", 8192, 8192, 28672, "bf16"),
        # the first layer of a small network over a test set of 10000 images, fp32 in and out
        _linear("linear_images", 10000, 784, 300, "fp32", bias=True),
        # odd sizes everywhere
        _linear("linear_odd", 1003, 4100, 1003, "fp16", bias=True),
        # between two blocks of a decode step: the residual sum and the next block's norm; latency counts
        _norm("norm_step", 64, 1, 8192, "bf16"),
        # prompts, a norm on each side of the block, a residual stream of 32 bits that grows by a part of each block
        _norm("norm_prompt", 1, 8191, 4096, "bf16", residual="fp32", post=True, scale=0.25),
        # images as 197 patches, gated by a vector for each image
        _norm("norm_images", 256, 197, 768, "fp16", kind="layer", gate="group", bias=True),
        # the way into a block's attention: norm, codes, and the three products that read them
        _block("block_chunk", 512, 4096, 4096, 1024, "bf16"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "linear", "norm", "norm", "norm", "block"])
    dtype = rng.choice(["bf16", "bf16", "fp16"] + ["fp32"] * (op != "block"))
    rotate = rng.random() < 0.3 and dtype != "fp32"

    def width(low, high):
        n = _log_int(rng, low, high)
        return max(128, n // 128 * 128) if rotate or rng.random() < 0.5 else n

    if op == "quantize":
        k = width(100, 28672)
        case = _quantize("", _log_int(rng, 1, max(1, min(16384, 90000000 // k))), k, dtype, rotate)
    elif op == "linear":
        k, n = width(100, 28672), _log_int(rng, 10, 32000)
        rows = _log_int(rng, 1, max(1, min(16384, 1900000000000 // (k * n), 235000000 // n)))
        case = _linear("", rows, k, n, dtype, rotate, rng.random() < 0.3)
    elif op == "norm":
        d = width(64, 16384)
        each = rng.choice([1, 1, 197, _log_int(rng, 2, 4096)])
        groups = _log_int(rng, 1, max(1, min(16384, 33000000 // (d * each))))
        case = _norm("", groups, each, d, dtype, rng.choice(["rms", "rms", "layer"]),
                     rng.choice(["", "", "fp32"]), rng.random() < 0.4, rng.choice(["", "", "channel", "group", "token"]),
                     rng.choice([1.0, 1.0, 0.25, 0.7071]), rng.random() < 0.3)
    else:
        k, n = width(256, 8192), _log_int(rng, 128, 8192)
        case = _block("", _log_int(rng, 1, 4096), k, n, max(16, n // rng.choice([1, 2, 4, 8])), dtype, rotate, rng.random() < 0.4)
    del case["name"]
    return case


def work(case):
    op, size = case["op"], _SIZES[case["dtype"]]
    if op == "norm":
        n = case["groups"] * case["each"] * case["width"]
        gate = {"": 0, "channel": case["width"], "group": case["groups"] * case["width"],
                "token": case["groups"] * case["each"]}[case["gate"]]
        vectors = (1 + case["post"]) * (1 + case["bias"]) * case["width"]
        return {"bytes": n * 2 * (size + _SIZES[case["residual"]]) + (gate + vectors) * size, "flops": (6 + 4 * case["post"]) * n}
    rows, k = case["rows"], case["width"]
    if op == "quantize":
        return {"bytes": rows * k * 2 * size + rows * k, "flops": rows * k * (2 + 7 * case["rotate"])}
    n = case["out"] + (2 * case["small"] if op == "block" else 0)
    moved = rows * k * size + n * k + 4 * n * (1 + case.get("bias", False)) + rows * n * size
    if op == "block":
        moved += rows * k * 2 * size + k * size
    return {"bytes": moved, "flops": 2 * rows * n * k}


# --------------------------------------------------------------------------------------------------------------- inputs

def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _stride(k):
    """Codes of a weight row: a multiple of 32, zeros behind the last."""
    return (k + 31) // 32 * 32


def _weight(n, k, gen, dev):
    """A layer's weights quantised by channel: what a program keeps of them."""
    w = torch.randn(n, k, generator=gen, device=dev).mul_(k ** -0.5)
    w *= torch.rand(n, 1, generator=gen, device=dev) + 0.5
    scales = w.abs().amax(1).clamp_(min=_LEAST) / torch.full((n,), _TOP, device=dev)
    codes = torch.zeros(n, _stride(k), dtype=torch.int8, device=dev)
    codes[:, :k] = torch.round(w.div_(scales[:, None])).to(torch.int8)
    return {"codes": codes, "scales": scales}


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)                                    # noqa: E731
    dtype, state = _DTYPES[case["dtype"]], {"case": dict(case)}
    if case["op"] == "norm":
        G, T, D = case["groups"], case["each"], case["width"]
        state["x"] = normal(G, T, D).mul_(0.5).to(dtype)
        state["residual"] = normal(G, T, D).mul_(2.0).to(_DTYPES[case["residual"]])
        state["weight"] = (normal(D) * 0.1 + 1).to(dtype)
        state["bias"] = (normal(D) * 0.1).to(dtype) if case["bias"] else None
        state["post_weight"] = (normal(D) * 0.1 + 1).to(dtype) if case["post"] else None
        state["post_bias"] = (normal(D) * 0.1).to(dtype) if case["post"] and case["bias"] else None
        shape = {"": None, "channel": (D,), "group": (G, 1, D), "token": (G, T, 1)}[case["gate"]]
        state["gate"] = normal(*shape).to(dtype) if shape else None
        return state
    # activations have a few channels that are much stronger than the others, and tokens of different sizes
    rows, k = case["rows"], case["width"]
    x = normal(rows, k)
    x[:, ::97] *= 8.0
    x *= torch.rand(rows, 1, generator=gen, device=dev) + 0.5
    state["x"] = x.to(dtype)
    if case["op"] == "block":
        state["residual"] = normal(rows, k).mul_(2.0).to(dtype)
        state["weight"] = (normal(k) * 0.1 + 1).to(dtype)
        state["post_weight"] = (normal(k) * 0.1 + 1).to(dtype) if case["post"] else None
        state["q"], state["k"], state["v"] = (_weight(n, k, gen, dev) for n in (case["out"], case["small"], case["small"]))
    elif case["op"] == "linear":
        state["w"] = _weight(case["out"], k, gen, dev)
        state["bias"] = normal(case["out"]) if case["bias"] else None
    return state


# ------------------------------------------------------------------------------------------------------- the plain forms

def _stage(x, stride):
    """One stage of the rotation's butterfly over blocks of 128: sums in the lower places, differences in the upper ones."""
    y = x.reshape(*x.shape[:-1], -1, 2, stride)
    a, b = y[..., 0, :], y[..., 1, :]
    return torch.stack([a + b, a - b], -2).reshape(x.shape)


def _rotated(x):
    x = _stage(_stage(_stage(_stage(x, 1), 2), 4), 8)
    return _stage(_stage(_stage(x, 16), 32), 64) * 128 ** -0.5


def _plain_quantize(x, rotate):
    """(codes as fp32, scales [rows, 1]) of fp32 rows."""
    if rotate:
        x = _rotated(x)
    size = x.abs().amax(-1, keepdim=True).clamp(min=_LEAST)
    scales = size / torch.full_like(size, _TOP)
    return torch.round(x / scales), scales


def _plain_product(codes, scales, w, bias, dtype):
    k = codes.shape[-1]
    y = (codes @ w["codes"][:, :k].float().T).mul_(w["scales"]).mul_(scales)
    return (y if bias is None else y.add_(bias)).to(dtype)


def _plain_normed(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    return v if bias is None else v + bias.float()


def _plain_sum(s, kind, scale, gate):
    """The residual stream behind the block, in fp32."""
    u = s["x"].float()
    if s["post_weight"] is not None:
        u = _plain_normed(u, kind, s["post_weight"], s.get("post_bias"))
    if gate is not None:
        u = u * gate.float()
    return s["residual"].float() + u * scale


def _plain(s):
    c = s["case"]
    dtype = _DTYPES[c["dtype"]]
    if c["op"] == "quantize":
        codes, scales = _plain_quantize(s["x"].float(), c["rotate"])
        return (codes * scales).to(dtype)
    if c["op"] == "linear":
        return _plain_product(*_plain_quantize(s["x"].float(), c["rotate"]), s["w"], s["bias"], dtype)
    if c["op"] == "norm":
        r = _plain_sum(s, c["kind"], c["scale"], s["gate"])
        return {"r": r.to(s["residual"].dtype), "h": _plain_normed(r, c["kind"], s["weight"], s["bias"]).to(dtype)}
    r = _plain_sum(s, "rms", 1.0, None)
    codes, scales = _plain_quantize(_plain_normed(r, "rms", s["weight"], None), c["rotate"])
    out = {name: _plain_product(codes, scales, s[name], None, dtype) for name in ("q", "k", "v")}
    return {"r": r.to(dtype), **out}


# ------------------------------------------------------------------------------------------------------------------ runs

def _packed(state, name):
    """The layer's packed weight, which a program makes once."""
    if name + "_packed" not in state:
        from if_i_could_turn_back_time_b200 import PackedWeight, QuantSpec
        c, w = state["case"], state[name]
        spec = QuantSpec("int8", 0, 128 if c["rotate"] else 0)
        state[name + "_packed"] = PackedWeight(spec, w["codes"].shape[0], c["width"], w["codes"], w["scales"], None)
    return state[name + "_packed"]


def run(state):
    if not own:
        return _plain(state)
    from if_i_could_turn_back_time_b200 import ops
    c = state["case"]
    if c["op"] == "quantize":
        rows = ops.quantize_rows(state["x"], had_block=128 if c["rotate"] else 0)
        return rows.dequantize(_DTYPES[c["dtype"]])
    if c["op"] == "linear":
        return ops.linear(state["x"], _packed(state, "w"), state["bias"])
    if c["op"] == "norm":
        h, r = ops.residual_norm(state["x"], state["residual"], state["weight"], state["bias"], post_weight=state["post_weight"],
                                 post_bias=state["post_bias"], gate=state["gate"], scale=c["scale"], kind=c["kind"])
        return {"r": r, "h": h}
    h, r = ops.residual_norm(state["x"], state["residual"], state["weight"], post_weight=state["post_weight"], quantize=True,
                             had_block=128 if c["rotate"] else 0)
    return {"r": r, **{name: ops.linear(h, _packed(state, name)) for name in ("q", "k", "v")}}


# --------------------------------------------------------------------------------------------------- the answer in 64 bits

def _hadamard(dev):
    """H / sqrt(128), by its definition: the sign of an entry is the parity of the bits that its row and column share."""
    both = torch.arange(128, device=dev)[:, None] & torch.arange(128, device=dev)
    odd = sum((both >> b) & 1 for b in range(7)) % 2
    return (1 - 2 * odd).double() / math.sqrt(128)


def _exact_codes(v, rotate):
    """(codes, scales) of rows in 64 bits; by the operator's definition a scale and the quotients that are rounded to codes are
    numbers of 32 bits."""
    if rotate:
        v = (v.reshape(-1, 128) @ _hadamard(v.device)).reshape(v.shape)
    s = (v.abs().amax(-1, keepdim=True).clamp(min=_LEAST) / _TOP).float().double()
    return torch.round((v / s).float()).double(), s


def _exact_linear(codes, s, w, bias):
    rows, k = codes.shape
    if 2 * rows * k * len(w["scales"]) > 2e13:
        return None
    w64 = w["codes"][:, :k].double() * w["scales"].double()[:, None]
    y = torch.cat([(codes[at:at + 2048] * s[at:at + 2048]) @ w64.T for at in range(0, rows, 2048)])
    return y if bias is None else y + bias.double()


def _exact_norm(v, kind, weight, bias):
    if kind == "layer":
        mean = v.mean(-1, keepdim=True)
        v = (v - mean) / ((v - mean) ** 2).mean(-1, keepdim=True).add(1e-6).sqrt()
    else:
        v = v / (v * v).mean(-1, keepdim=True).add(1e-6).sqrt()
    return v * weight.double() + (0 if bias is None else bias.double())


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "quantize":
        codes, scales = _exact_codes(x, case["rotate"])
        return codes * scales
    if case["op"] == "linear":
        return _exact_linear(*_exact_codes(x, case["rotate"]), s["w"], s["bias"])
    kind = case.get("kind", "rms")
    if s["post_weight"] is not None:
        x = _exact_norm(x, kind, s["post_weight"], s.get("post_bias"))
    if s.get("gate") is not None:
        x = x * s["gate"].double()
    r = s["residual"].double() + case.get("scale", 1.0) * x
    h = _exact_norm(r, kind, s["weight"], s.get("bias"))
    if case["op"] == "norm":
        return {"r": r, "h": h}
    codes, scales = _exact_codes(h, case["rotate"])
    return {"r": r, **{name: _exact_linear(codes, scales, s[name], None) for name in ("q", "k", "v")}}
