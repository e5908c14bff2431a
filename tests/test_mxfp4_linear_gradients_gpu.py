"""The backward passes of the MXFP4 products with an epilogue and of the experts' gated projection
against their whole formula in 64 bits (dx from dy and the kept pre-activations, with no rounding in
between) and against differences of the forward formula.

dx is a sum of products of dpre (dg, du) rounded to bf16, each off by at most half a step, 2^-8 of
itself.  Those errors add up to 2^-8 |dpre| |W| where all have the worst size and sign; having any
sign and a rounding's spread, below a third of their squares, their root mean square over the results
is below 2^-8 times that of sqrt(dpre^2 W^2)."""
import pytest
import torch

from kadan_amd import ops

import mxfp4_epilogue_reference as epi
import mxfp4_reference as ref

pytestmark = pytest.mark.gpu

HALF, BF16 = ref.HALF_BF16, torch.bfloat16


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(808)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def near(dx, exact, bound, w, what):
    """dx against exact @ w, exact being within bound before it is rounded to bf16."""
    bound = bound + (exact.abs() + bound) * HALF + ref.TINY
    want, sums = ref.sum_bound(exact, w.T)
    ref.within(dx, want, epi.rounded(want, 1.01 * sums + bound @ w.abs(), BF16), what)
    spread = ((exact ** 2) @ (w ** 2)).mean().sqrt()
    off = (dx.double() - want).square().mean().sqrt()
    assert float(off) <= HALF * float(spread + want.square().mean().sqrt()), what


def products(g, m, experts, n, k):
    """Matrices of each expert in 64 bits, their backward form, offsets (None: dense)."""
    blocks, scales = ref.matrix(g, max(experts, 1) * n, k)
    w = ref.decode(blocks, scales).view(max(experts, 1), n, k)
    if not experts:
        return w, ops.mxfp4_pack(blocks, scales, transposed=True), None
    turned = ops.mxfp4_pack(blocks.view(experts, n, -1), scales.view(experts, n, -1),
                            transposed=True)
    ends = torch.sort(torch.randint(0, m + 1, (experts - 1,), generator=g, device=g.device))[0]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=g.device)
    offsets[1:-1], offsets[-1] = ends, m
    return w, turned, offsets


# m, experts (0: dense), n, k: single rows, every tile, K slices
SIZES = [(1, 0, 64, 96), (33, 0, 1600, 160), (300, 0, 1032, 288), (910, 0, 4152, 544),
         (1025, 0, 520, 2048), (5, 4, 96, 64), (40, 3, 2912, 416), (700, 5, 512, 608),
         (2048, 32, 544, 352)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,experts,n,k", SIZES)
def test_linear(gen, m, experts, n, k, act):
    w, turned, offsets = products(gen, m, experts, n, k)
    dy, saved = normal(gen, m, n).bfloat16(), (normal(gen, m, n) * 2).bfloat16()
    dx, _ = ops.mxfp4_linear_backward(dy, turned, k, saved=saved, activation=act, offsets=offsets)
    slope, err = epi.slope(saved.double(), act)
    exact = dy.double() * slope
    bound = dy.double().abs() * err + exact.abs() * 2.0 ** -22
    epi.by_expert(lambda e, *rows: near(*rows, w[e], f"expert {e}"),
                  [0, m] if offsets is None else offsets.tolist(), dx, exact, bound)


@pytest.mark.parametrize("act", ["silu", "clamped"])
@pytest.mark.parametrize("m,experts,n,k", [s for s in SIZES if s[1]])
def test_experts_gated(gen, m, experts, n, k, act):
    n = n // 32 * 32
    gate, gate_turned, offsets = products(gen, m, experts, n, k)
    up, up_turned, _ = products(gen, m, experts, n, k)
    dh, saved = normal(gen, m, n).bfloat16(), (normal(gen, m, 2 * n) * 3).bfloat16()
    dx, _ = ops.mxfp4_experts_gated_backward(dh, offsets, saved, gate_turned, up_turned, k,
                                             activation=act)
    g, u = saved.double()[:, :n], saved.double()[:, n:]
    exact, _ = epi.gate_gradients(dh.double(), g, u, act)
    # (what dg and du are off by ahead of their rounding: an exponential, a reciprocal and the
    # sums of a few terms of the size of |dh| (|u| + 1) (1 + |z|) or of |dh g|)
    z = g if act == "silu" else 1.702 * g.clamp(max=7)
    size = dh.double().abs() * epi.near(z)
    bound = torch.cat([size * (u.abs() + 1) * (2 + 3 * z.abs()), size * g.abs()], 1)
    epi.by_expert(lambda e, *rows: near(*rows, torch.cat([gate[e], up[e]]), f"expert {e}"),
                  offsets.tolist(), dx, exact, bound)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_linear_against_differences(gen, act):
    m, n, k = 40, 64, 96
    w, turned, _ = products(gen, m, 0, n, k)
    dy, saved = normal(gen, m, n).bfloat16(), (normal(gen, m, n) * 2).bfloat16()
    dx, dpre = ops.mxfp4_linear_backward(dy, turned, k, saved=saved, activation=act)

    def y(at):  # the activation at the kept values and beside them
        return at * torch.sigmoid(epi.inner(at, act)[0])

    step, kept = 2.0 ** -14, saved.double()
    differences = dy.double() * (y(kept + step) - y(kept - step)) / (2 * step)
    # a central difference is off by step^2 / 6 of the third derivative, which is at most 3
    slack = dy.double().abs() * (step * step + 2.0 ** -18 * (1 + kept.abs() ** 2)) + ref.TINY
    ref.within(dpre, differences, slack + (differences.abs() + slack) * HALF, "dpre")
    near(dx, differences, slack, w[0], "dx")


@pytest.mark.parametrize("act", ["silu", "clamped"])
def test_experts_gated_against_differences(gen, act):
    m, experts, n, k = 40, 3, 64, 96
    gate, gate_turned, offsets = products(gen, m, experts, n, k)
    up, up_turned, _ = products(gen, m, experts, n, k)
    dh, saved = normal(gen, m, n).bfloat16(), (normal(gen, m, 2 * n) * 4).bfloat16()
    kept = saved.double()
    kept[(kept.abs() - 7).abs() < 0.01] = 6.5  # (away from the clamps, where there is no slope)
    saved = kept.bfloat16()
    dx, dgu = ops.mxfp4_experts_gated_backward(dh, offsets, saved, gate_turned, up_turned, k,
                                               activation=act)
    g, u, step = kept[:, :n], kept[:, n:], 2.0 ** -14

    def h(g, u):
        return epi.gate(g, u, act)[0] * dh.double()

    differences = torch.cat([h(g + step, u) - h(g - step, u), h(g, u + step) - h(g, u - step)],
                            1) / (2 * step)
    # third derivatives are at most 3 (|u| + 1) (1.702^2) in g and 0 in u
    size = dh.double().abs()
    slack = torch.cat([size * (u.abs() + 1) * (3 * step * step + 2.0 ** -18 * (1 + g.abs())),
                       size * 2.0 ** -18 * (1 + g.abs()) ** 2], 1) + ref.TINY
    ref.within(dgu, differences, slack + (differences.abs() + slack) * HALF, "dgu")
    epi.by_expert(lambda e, *rows: near(*rows, torch.cat([gate[e], up[e]]), f"expert {e}"),
                  offsets.tolist(), dx, differences, slack)
