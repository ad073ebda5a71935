"""Gate, experts and dense products in 64 bits, each value with a bound of how far a kernel with fp32 sums may be from it.

Bounds. u: half a step of the rounded type, relative (bf16 2^-8 ... as finfo.eps / 2), and half its smallest subnormal. A sum of K products on
the tensor cores rounds once for every 16 of them, each time by at most 2^-22 of the sum of magnitudes S that has come together (fp32 sums
whose addends are aligned and cut): S * (K / 16 + 8) * 2^-22, where the 8 covers sums over warps and parts, the bias and the residual.
Functions of an argument that is off by d are off by at most their steepest slope times d (gelu 1.13, silu 1.1) and 2^-20 of their value.
"""
import math

import torch

SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(value, bound, dtype):
    """The bound of a value that is rounded to `dtype` after all."""
    info = torch.finfo(dtype)
    return bound + half_step(dtype) * (value.abs() + bound) + info.smallest_normal * info.eps / 2


def product(x, w, bias=None):
    x, w = x.double(), w.double()
    value, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        value, size = value + bias.double(), size + bias.double().abs()
    return value, size * (math.ceil(x.shape[-1] / 16) + 8) * 2.0 ** -22


def swiglu(value, bound):
    (gate, up), (dg, du) = value.chunk(2, dim=-1), bound.chunk(2, dim=-1)
    s = gate * torch.sigmoid(gate)
    out = s * up
    return out, 1.1 * dg * (up.abs() + du) + s.abs() * du + 2.0 ** -20 * out.abs()


def linear(x, w, bias, activation, residual, out_dtype):
    value, bound = product(x, w, bias)
    if activation == "swiglu":
        value, bound = swiglu(value, bound)
    else:
        f = {"none": lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[activation]
        value, bound = f(value), bound * SLOPE[activation]
        bound = bound + (0 if activation == "none" else 2.0 ** -20) * value.abs()
    if residual is not None:
        value = value + residual.double()
        bound = bound + 2.0 ** -23 * (value.abs() + residual.double().abs())
    return value, rounded(value, bound, out_dtype)


def expert(x, gate_up, down, dtype):
    """One expert on rows: values and bounds before the last rounding."""
    h, dh = swiglu(*product(x, gate_up))
    dh = rounded(h, dh, dtype)
    value, bound = product(h, down)
    return value, bound * 1.01 + dh @ down.double().abs().t()


def layer(x, indices, weights, gate_up, down, residual):
    tokens, k = indices.shape
    value, bound, size = (torch.zeros(x.shape, dtype=torch.float64) for _ in range(3))
    for e in range(gate_up.shape[0]):
        t, j = (indices == e).nonzero(as_tuple=True)
        if t.numel():
            v, d = expert(x[t], gate_up[e], down[e], x.dtype)
            w = weights[t, j, None].double()
            value.index_add_(0, t, w * v)
            bound.index_add_(0, t, w.abs() * d)
            size.index_add_(0, t, (w * v).abs())
    if residual is not None:
        value, size = value + residual.double(), size + residual.double().abs()
    return value, rounded(value, bound + (k + 2) * 2.0 ** -23 * size, x.dtype)


def gate(logits, k, score, bias, renormalize, scale):
    l = logits.double()
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    indices = torch.sort(l if bias is None else s + bias.double(), dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, indices)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    return indices.to(torch.int32), w * scale


def assert_within(got, value, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (got.shape, value.shape)
    off = (got - value).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert bool((off <= bound).all()), f"{what}: {worst:.3g} times the bound"
