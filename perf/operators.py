"""Cases of the framework's channels-last operators, for timing and checking.

group_norm_act: group norm over [samples, positions, channels] with an
activation (s2b200.group_norm_act); linear_act: y = act(x W^T + b) + residual
(s2b200.linear_act). Each case runs in a plain form (torch, 32 bits) or, with
`own` set, as the framework's call.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "seedvr2-ncnn-valkan_b200")
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
_ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")

# What a drawn case may cost at most: the elements of the largest listed norm
# and the products of the largest listed matrix product.
_MAX_ELEMENTS = 21 * 720 * 1280 * 128
_MAX_PRODUCTS = 21600 * 2560 * 10240


def _norm(name, samples, positions, channels, groups, dtype, out, act, pad=0):
    return {"name": name} | _norm_case(samples, positions, channels, groups, dtype, out, act, pad)


def _norm_case(samples, positions, channels, groups, dtype, out, act, pad):
    return {"op": "group_norm_act", "samples": samples, "positions": positions, "channels": channels,
            "groups": groups, "dtype": dtype, "out": out, "act": act, "pad": pad}


def _linear(name, m, n, k, dtype, act, bias, residual, pad=0):
    return {"name": name} | _linear_case(m, n, k, dtype, act, bias, residual, pad)


def _linear_case(m, n, k, dtype, act, bias, residual, pad):
    return {"op": "linear_act", "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "pad": pad}


def listed():
    return [
        # a residual block's first norm at the 5-frame 480 x 256 clip's latent (2 x 32 x 60): one short launch
        _norm("norm_latent_480x256", 2, 1920, 512, 32, "fp16", "fp16", "silu"),
        # a ragged crop's fp32 features, read from a wider row and handed on in 16 bits (3 channels a group)
        _norm("norm_ragged_fp32", 3, 7973, 96, 32, "fp32", "fp16", "gelu", 5),
        # the norm in front of the mid-block attention, 6 latent frames of 90 x 160
        _norm("norm_mid_720p", 6, 14400, 512, 32, "fp16", "fp16", "none"),
        # after the decoder's first space-time upsampling: 11 frames of 180 x 320
        _norm("norm_up_720p", 11, 57600, 512, 32, "bf16", "bf16", "silu"),
        # the decoder's last residual block, 21 full 720p frames
        _norm("norm_pixels_720p", 21, 921600, 128, 32, "bf16", "bf16", "silu"),
        # the timestep MLP: one row through 2560 -> 2560 with SiLU, then 2560 -> 15360
        _linear("linear_time_hidden", 1, 2560, 2560, "bf16", "silu", True, False),
        _linear("linear_time_out", 1, 15360, 2560, "fp16", "none", True, False),
        # the text projection, 58 tokens of 5120 channels
        _linear("linear_text", 58, 2560, 5120, "fp16", "none", True, False),
        # odd in every extent: a cropped batch with a head of 777 outputs, rows of odd pitch
        _linear("linear_ragged", 1237, 777, 1001, "bf16", "gelu_tanh", True, True, 2),
        # the mid block's output projection with its residual, 6 frames of 14400 tokens
        _linear("linear_vae_out", 86400, 512, 512, "fp16", "none", True, True),
        # the MLP of a DiT block over 21600 tokens: GELU up to 10240, and 6912 back down onto the stream
        _linear("linear_mlp_up", 21600, 10240, 2560, "bf16", "gelu", True, False),
        _linear("linear_mlp_down", 21600, 2560, 6912, "fp16", "none", True, True),
    ]


def _log(rng, lo, hi):
    return int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))


def draw(rng):
    if rng.random() < 0.5:
        groups = rng.choice((8, 10, 16, 32, 32))
        channels = groups * rng.choice((1, 2, 3, 4, 7, 8, 13, 16, 16))
        samples = rng.randint(1, 24)
        positions = min(_log(rng, 1, 1000000), _MAX_ELEMENTS // (samples * channels))
        dtype, out = rng.choice((("fp16", "fp16"), ("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "fp16"),
                                 ("fp32", "bf16")))
        if dtype == "fp32":
            positions = max(1, positions // 2)
        return _norm_case(samples, positions, channels, groups, dtype, out, rng.choice(_ACTS),
                          rng.choice((0, 0, 8, rng.randint(1, 40))))
    m, n, k = _log(rng, 1, 90000), _log(rng, 4, 15360), _log(rng, 8, 10240)
    if rng.random() < 0.5:  # channel counts are mostly round
        n, k = max(16, n // 16 * 16), max(16, k // 16 * 16)
    m = max(1, min(m, _MAX_PRODUCTS // (n * k)))
    return _linear_case(m, n, k, rng.choice(("fp16", "bf16")), rng.choice(_ACTS), rng.random() < 0.8,
                        rng.random() < 0.5, rng.choice((0, 0, 8, rng.randint(1, 40))))


def _round8(v):
    return (v + 7) // 8 * 8


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    dtype = _DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "group_norm_act":
        c = case["channels"]
        # features with a scale and an offset of each channel's own, in rows of channels + pad values
        x = normal(case["samples"], case["positions"], c + case["pad"], dtype=dtype)[..., :c]
        x.mul_(torch.exp(0.5 * normal(c)).to(dtype)).add_((2.0 * normal(c)).to(dtype))
        return state | {"x": x, "weight": 1.0 + 0.1 * normal(c), "offset": 0.1 * normal(c)}
    m, n, k = case["m"], case["n"], case["k"]
    x = normal(m, k + case["pad"], dtype=dtype)[:, :k]
    # a program keeps its weights in rows that start on 16 bytes
    w = normal(n, _round8(k), dtype=dtype).mul_(0.02)[:, :k]
    return state | {"x": x, "w": w, "offset": 0.1 * normal(n) if case["bias"] else None,
                    "stream": normal(m, n, dtype=dtype) if case["residual"] else None}


def _activate(v, act):
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    return v


def run(state):
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import s2b200
        if state["op"] == "group_norm_act":
            return s2b200.group_norm_act(state["x"], state["groups"], state["weight"], state["offset"], eps=1e-6,
                                         activation=state["act"], out_dtype=_DTYPES[state["out"]])
        return s2b200.linear_act(state["x"], state["w"], bias=state["offset"], activation=state["act"],
                                 residual=state["stream"])
    x = state["x"].float()
    if state["op"] == "group_norm_act":
        s, p, c = x.shape
        g = state["groups"]
        v = x.reshape(s, p, g, c // g)
        mean = v.mean(dim=(1, 3), keepdim=True)
        v = v - mean
        var = (v * v).mean(dim=(1, 3), keepdim=True)
        v = (v * torch.rsqrt(var + 1e-6)).reshape(s, p, c) * state["weight"] + state["offset"]
        return _activate(v, state["act"]).to(_DTYPES[state["out"]])
    v = torch.matmul(x, state["w"].float().t())
    if state["offset"] is not None:
        v = v + state["offset"]
    v = _activate(v, state["act"])
    if state["stream"] is not None:
        v = v + state["stream"].float()
    return v.to(state["w"].dtype)


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "group_norm_act":
        elements = case["samples"] * case["positions"] * case["channels"]
        return {"bytes": elements * (size + _BYTES[case["out"]]) + 8 * case["channels"], "flops": 10 * elements}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": size * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0),
            "flops": 2 * m * n * k}


def exact(case, seed):
    norm = case["op"] == "group_norm_act"
    if norm and case["samples"] * case["positions"] * case["channels"] > 1_000_000_000:
        return None
    state = prepare(case, seed)
    act = case["act"]
    sigmoid, root = torch.sigmoid, torch.sqrt
    if norm:
        g, c = case["groups"], case["channels"]
        weight, offset = state["weight"].double(), state["offset"].double()
        parts = []
        for sample in state["x"]:
            columns = sample.double().t().reshape(g, -1)
            variance, mean = torch.var_mean(columns, dim=1, correction=0, keepdim=True)
            columns = ((columns - mean) / root(variance + 1e-6)).reshape(c, -1).t()
            parts.append(torch.addcmul(offset, columns, weight))
        y = torch.stack(parts)
        del parts
    else:
        y = torch.nn.functional.linear(state["x"].double(), state["w"].double())
        if case["bias"]:
            y += state["offset"].double()
    if act == "relu":
        y = y.clamp(min=0)
    elif act == "silu":
        y = y * sigmoid(y)
    elif act == "gelu":
        y = y * torch.special.ndtr(y)
    elif act == "gelu_tanh":
        y = y * sigmoid(1.5957691216057308 * (y + 0.044715 * y ** 3))
    if not norm and case["residual"]:
        y = y + state["stream"].double()
    return y
