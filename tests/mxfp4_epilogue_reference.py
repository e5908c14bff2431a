"""Epilogues of the MXFP4 products in 64 bits, from their definitions, and how far a kernel that
follows its documented roundings may be from them (tests only).

The kernels' sigmoid comes from an exponential and a reciprocal within 2^-22 each; its argument z
is off by a few halves of a step, so by at most 2^-21 |z|, which goes into the sigmoid as it is."""
import math

import torch

import mxfp4_reference as ref

HALF = {torch.float32: ref.HALF_F32, torch.bfloat16: ref.HALF_BF16}
GELU = 2 * math.sqrt(2 / math.pi)


def inner(v, act):
    """z of v sigmoid(z), and its derivative."""
    if act == "silu":
        return v, torch.ones_like(v)
    return GELU * (v + 0.044715 * v ** 3), GELU * (1 + 3 * 0.044715 * v ** 2)


def near(z):
    return 2.0 ** -20 + 2.0 ** -21 * z.abs()


def lost(z, size):
    """Where exp(-z) overflows fp32 the kernels' sigmoid is 0 instead of at most 2^-115."""
    return torch.where(z < -80, size, torch.zeros_like(size))


def activated(v, err, act):
    """act(v) and its bound, v being within err: |silu'| <= 1.1, |gelu'| <= 1.13."""
    if act is None:
        return v, err
    z, _ = inner(v, act)
    y = v * torch.sigmoid(z)
    return y, 1.13 * err + (y.abs() + 1.13 * err) * near(z) + lost(z, y.abs())


def slope(v, act):
    """act'(v) and the bound of its computation."""
    z, dz = inner(v, act)
    s = torch.sigmoid(z)
    d = s + v * s * (1 - s) * dz
    # (1 - s is off by what s is, and the rest is at most s)
    return d, s * near(z) * (1 + 3 * (v * dz).abs()) + lost(z, d.abs())


def pre_activation(x, w, bias=None):
    v, err = ref.sum_bound(x, w)
    if bias is not None:
        v = v + bias
        err = err + (v.abs() + err) * ref.HALF_F32
    return v, err


def linear(x, w, bias, act, residual, dtype):
    """(pre, its bound), (y, its bound) with y as dtype."""
    pre, err = pre_activation(x, w, bias)
    y, bound = activated(pre, err, act)
    if residual is not None:
        y = y + residual
        bound = bound + (y.abs() + bound) * ref.HALF_F32
    return (pre, err), (y, rounded(y, bound, dtype))


def rounded(y, bound, dtype):
    return bound + (y.abs() + bound) * (HALF[dtype] if dtype == torch.bfloat16 else 0) + ref.TINY


def clamped(g, u):
    """(h, dh/dg, dh/du) of the clamped gate."""
    c, v = g.clamp(max=7), u.clamp(-7, 7)
    s = torch.sigmoid(1.702 * c)
    zero = torch.zeros_like(g)
    return (c * s * (v + 1), torch.where(g <= 7, (v + 1) * s * (1 + 1.702 * c * (1 - s)), zero),
            torch.where(u.abs() <= 7, c * s, zero))


def gate(g, u, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s * u, u * s * (1 + g * (1 - s)), g * s
    return clamped(g, u)


def gated(g, dg, u, du, act):
    """h and its bound as bf16, g and u being within dg and du: the gate's slopes are at most
    1.13 (|u| + 1) in g and |silu-like of g| in u."""
    h, _, by_u = gate(g, u, act)
    z = g if act == "silu" else 1.702 * g.clamp(max=7)
    room = (u.abs() + du + (0 if act == "silu" else 1))
    bound = 1.13 * dg * room + (by_u.abs() + 1.13 * dg + (
        0 if act == "silu" else torch.where(u.abs() > 7 - du, g.abs().clamp(max=7), 0 * g))) * du
    size = torch.maximum(h.abs(), by_u.abs()) + bound  # (u' + 1 may cancel)
    return h, rounded(h, bound + size * near(z) + lost(z, h.abs() + by_u.abs()), torch.bfloat16)


def gate_gradients(dh, g, u, act):
    """[dg | du] in 64 bits and its bound as bf16."""
    if act == "silu":
        return ref.gate_gradients(dh, g, u)
    _, by_g, by_u = gate(g, u, act)
    c = g.clamp(max=7)
    z = 1.702 * c
    s = torch.sigmoid(z)
    e1 = dh.abs() * (u.abs().clamp(max=7) + 1) * s * (2 + 3 * z.abs()) * near(z)
    e2 = (dh * by_u).abs() * near(z)
    exact = torch.cat([dh * by_g, dh * by_u], 1)
    err = torch.cat([e1 + lost(z, (dh * by_g).abs()), e2 + lost(z, (dh * by_u).abs())], 1)
    return exact, rounded(exact, err, torch.bfloat16)


def by_expert(f, offsets, *rows):
    """f(expert, its rows of each) for every expert that has some: [(first, end, result)]."""
    out = []
    for e in range(len(offsets) - 1):
        first, end = offsets[e], offsets[e + 1]
        if end > first:
            out.append((first, end, f(e, *[r[first:end] for r in rows])))
    return out
