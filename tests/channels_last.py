"""Plain 64-bit forms and error bounds of the channels-last operators, for their tests.

Bounds count roundings. An output is rounded once: at most half a step, torch.finfo(t).eps / 2
relative to its value. In front of that stand the fp32 roundings, 2^-24 relative each.

Group norm, z = (x - m) / sigma * w + b. The mean is joined from runs, threads and blocks; each
join rounds it by 2^-24 |m|, and at most 24 of them lie on the way of any value (8 runs of a thread
as a rule, 5 + 5 shuffles, the rest averaged down), so z is off by at most 24 * 2^-24 |m| / sigma |w|
from the mean, by as many 2^-24 |z| from sigma (sums of squares of runs of at most 64 values each
round to 64 * 2^-24, halved by the square root), and by a few more from the last steps: 64 * 2^-24 =
2^-18 of |w| (|x - m| / sigma + |m| / sigma) + |b| holds all of it. The activations' slopes are at
most 1.13, and the hardware's exponential and division add a few 2^-23: 2^-17 in all.

Matrix product, S = sum |x w|. The tensor cores add 16 products at a time to an fp32 sum and cut it
off (a whole step 2^-23 at most): (K / 16 + 16) 2^-23 S, with the slope 1.13 and the last steps
another 2^-17 of the value.
"""
from __future__ import annotations

import torch

ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def activate(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)))
    return v


def norm_exact(x, groups, weight, bias, eps, act):
    """(y, bound on the fp32 part of its error) in 64 bits, x [S, ..., C]."""
    S, C = x.shape[0], x.shape[-1]
    v = x.double().reshape(S, -1, groups, C // groups)
    mean = v.mean(dim=(1, 3), keepdim=True)
    d = v - mean
    sigma = ((d * d).mean(dim=(1, 3), keepdim=True) + eps).sqrt()
    w = torch.ones(C, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    z = (d / sigma).reshape(S, -1, C) * w + b
    room = ((d.abs() + mean.abs()) / sigma).reshape(S, -1, C) * w.abs() + b.abs()
    return activate(z, act).reshape(x.shape), 2.0 ** -17 * room.reshape(x.shape)


def linear_exact(x, w, bias, act, residual):
    """(y, bound on the fp32 part of its error) in 64 bits."""
    K = x.shape[-1]
    v = x.double() @ w.double().t()
    room = x.double().abs() @ w.double().abs().t() * (K / 16 + 16) * 2.0 ** -23
    if bias is not None:
        v = v + bias.double()
    y = activate(v, act)
    room = 1.13 * room + 2.0 ** -17 * v.abs()
    if residual is not None:
        y = y + residual.double()
        room = room + 2.0 ** -23 * y.abs()
    return y, room


def check(got, want, room, what=""):
    """Every value of `got` within its rounding and `room` of `want`."""
    info = torch.finfo(got.dtype)
    half = info.eps / 2
    limit = room * (1 + half) + half * want.abs() + info.smallest_normal * half
    off = (got.double() - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst by "
                           f"{(off / limit).nan_to_num(9e9).max().item():.3g} times its bound")


def activation_exact(v, act):
    """(act(v), bound on its error in fp32) for fp32 values v, in 64 bits, every tail relatively exact.

    Roundings, in units of u = 2^-23 (two fp32 half steps, one ulp of the hardware's reciprocal; its 2^x is within
    2 u): silu, v / (1 + e^-v): 2^x, +, 1 / x, * are 2 + 1 + 1 + 1 with one to spare, and the exponent's product with
    a rounded log2 e is off by |v| u at most in the exponent. gelu, v h: the fit of h 0.8 u, seven fmas of which the
    last ones count (2), t 2, products 1.5, 2^x 2: 8, and v^2 / 2 u from the exponent's two products and its constant.
    gelu_tanh like silu, its exponent w from three roundings and two rounded constants: 2 w u. Above 0 the exponentials
    weigh at most 0.37 of these last terms; the bound keeps them whole below 0 and drops them above, where 2 u more
    cover them. Below 2^-119 a result may be 0."""
    v = v.double()
    a, u = v.abs(), 2.0 ** -23
    w = 2 * (2 / torch.pi) ** 0.5 * (a + 0.044715 * a ** 3)
    if act == "gelu_tanh":
        y = v * torch.sigmoid(torch.sign(v) * w)
    elif act == "gelu":
        y = v * 0.5 * torch.erfc(v * -0.5 ** 0.5)  # special.ndtr is exact absolutely only
    else:
        y = activate(v, act)
    base, slope = {"none": (0, 0 * a), "relu": (0, 0 * a), "silu": (6, a), "gelu": (8, a * a / 2),
                   "gelu_tanh": (6, 2 * w)}[act]
    units = torch.where(v < 0, base + slope, (base + 2.0 if base else 0.0) + 0 * a)
    return y, y.abs() * units * u + (2.0 ** -119 if base else 0.0)
