"""MXFP4 dense operators in 64 bits, from their definitions, and how far a kernel that
follows its documented roundings may be from them (tests only)."""
import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
HALF_BF16 = 2.0 ** -8     # half a step of bf16 (torch.finfo.eps / 2), relative
HALF_F32 = 2.0 ** -24
TINY = 2.0 ** -126        # below this, types run out of exponents


def quantize(x):
    """float64 [rows, cols] -> (blocks, scales) by comparing every value with every level."""
    rows, cols = x.shape
    b = x.reshape(-1, 32)
    top = np.abs(b).max(1)
    with np.errstate(divide="ignore"):
        byte = np.where(top > 0, np.floor(np.log2(top)) - 2 + 127, 0)
    byte = np.maximum(byte, 0).astype(np.int64)
    a = np.abs(b) / np.exp2(byte - 127.0)[:, None]
    off = np.abs(a[..., None] - LEVELS)
    nearest = off.min(-1, keepdims=True)
    near = off == nearest
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = (code | (np.signbit(b) << 3)).astype(np.uint8).reshape(rows, cols)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte.astype(np.uint8).reshape(rows, -1)


def decode(blocks, scales):
    """uint8 tensors -> float64 [rows, cols] on their device (byte 255 as 2^128)."""
    table = torch.tensor(np.concatenate([LEVELS, -LEVELS]), device=blocks.device)
    codes = torch.stack([blocks & 15, blocks >> 4], -1).reshape(blocks.shape[0], -1)
    powers = torch.tensor(np.exp2(np.arange(256) - 127.0), device=blocks.device)  # exact
    return table[codes.long()] * powers[scales.long()].repeat_interleave(32, 1)


def matrix(g, rows, cols, low=118, high=125):
    """Random codes and scale bytes on the device of g."""
    dev = g.device
    blocks = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8, device=dev)
    scales = torch.randint(low, high, (rows, cols // 32), generator=g, dtype=torch.uint8,
                           device=dev)
    return blocks, scales


def sum_bound(x, w):
    """x [m, k] W^T in 64 bits and the largest distance of an fp32 sum of its exact products:
    k - 1 additions, each off by at most half a step of a partial sum, which is at most the
    sum of magnitudes."""
    y = x @ w.T
    return y, x.shape[1] * HALF_F32 * (x.abs() @ w.abs().T) + TINY


def gated(x, wg, wu):
    """(g, u, h) and the bounds of each (h as bf16): |silu'| <= 1.1; the exponential and the
    reciprocal are within 2^-22 and the exponent's argument within 2^-24 of |g| log2(e)."""
    g, dg = sum_bound(x, wg)
    u, du = sum_bound(x, wu)
    s = g * torch.sigmoid(g)
    h = s * u
    inner = 1.1 * dg * (u.abs() + du) + (s.abs() + 1.1 * dg) * du + h.abs() * (
        2.0 ** -20 + 2.0 ** -23 * g.abs())
    # (silu underflows in fp32 where exp(-g) overflows: below -88 it is at most 2^-120)
    inner = inner + torch.where(g < -80, s.abs() * u.abs(), torch.zeros_like(s))
    return (g, dg), (u, du), (h, inner + (h.abs() + inner) * HALF_BF16 + TINY)


def gate_gradients(dh, g, u):
    """[dg | du] in 64 bits and its bound as bf16: each factor of dg = dh u (s (1 + g (1 - s)))
    is within 2^-20 of the terms it sums, du = dh g s within 2^-20 of itself."""
    s = torch.sigmoid(g)
    dg, du = dh * u * (s * (1 + g * (1 - s))), dh * g * s
    eps = 2.0 ** -20 + 2.0 ** -23 * g.abs()
    e1 = (dh * u).abs() * s * (2 + 2 * g.abs()) * eps
    e2 = du.abs() * eps
    # (where exp(-g) overflows fp32 s is zero instead of at most 2^-120)
    low = torch.where(g < -80, torch.ones_like(g), torch.zeros_like(g))
    e1, e2 = e1 + low * dg.abs(), e2 + low * du.abs()
    exact = torch.cat([dg, du], 1)
    err = torch.cat([e1, e2], 1)
    return exact, err + (exact.abs() + err) * HALF_BF16 + TINY


def within(got, want, bound, what=""):
    """Every value within its bound (NaN in none of them)."""
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(
            f"{what}: {int(bad.sum())} of {bad.numel()} outside, the first at {i}: got "
            f"{float(got.reshape(-1)[i])}, want {float(want.reshape(-1)[i])} within "
            f"{float(bound.reshape(-1)[i])}")
