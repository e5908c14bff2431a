"""MXFP4 products with an epilogue, dense and of a mixture's experts, and the experts' gated
projection, with their backward passes (kdq_mxfp4_linear, _linear_backward, _experts_gated,
_experts_gated_backward, _experts_pack), against their definitions in 64 bits."""
import pytest
import torch

import kadan_amd
from kadan_amd import ops

import mxfp4_epilogue_reference as epi
import mxfp4_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(4321)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def stack(g, experts, rows, cols):
    blocks, scales = ref.matrix(g, experts * rows, cols)
    return blocks.view(experts, rows, -1), scales.view(experts, rows, -1)


def decoded(matrices, e):
    return ref.decode(matrices[0][e], matrices[1][e])


def counts_of(g, m, experts, kind):
    """Rows of each expert, m in all."""
    if kind == "even":
        of = torch.arange(m, device=g.device) % experts
    elif kind == "one":
        of = torch.full((m,), experts // 2, device=g.device)
    else:  # some popular, some with none
        odds = torch.rand(experts, generator=g, device=g.device) ** 4 + 1e-4
        odds[::3] = 0 if experts > 2 else 1
        of = torch.multinomial(odds, m, replacement=True, generator=g)
    return torch.bincount(of, minlength=experts)


def offsets_of(counts):
    out = torch.zeros(counts.numel() + 1, dtype=torch.int32, device=counts.device)
    out[1:] = torch.cumsum(counts, 0)
    return out


# ---------------------------------------------------------------- dense

LINEAR = [  # m, n, k: decode and larger tiles, K slices, ragged in each direction
    (1, 1, 32), (1, 16, 64), (2, 33, 96), (3, 8, 14336), (9, 2880, 2880), (16, 70, 128),
    (17, 65, 256), (31, 100, 288), (32, 8192, 672), (1, 8161, 32), (33, 70, 96), (65, 257, 544),
    (77, 4096, 1440), (127, 130, 1056), (129, 63, 4128), (257, 1030, 288), (2933, 525, 544),
    (833, 4756, 544), (2083, 2856, 1632), (65, 11414, 12448), (520, 2048, 608),
    (16, 8412, 544), (2872, 3, 12608), (3017, 525, 10528)]
EPILOGUES = [(None, True, False), ("silu", False, True), ("gelu", True, True),
             ("gelu", False, False), (None, False, True)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act,with_bias,with_residual", EPILOGUES)
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(gen, m, n, k, act, with_bias, with_residual, dtype):
    w, x = ref.matrix(gen, n, k), normal(gen, m, k).bfloat16()
    bias = normal(gen, n) if with_bias else None
    residual = normal(gen, m, n).to(dtype) if with_residual else None
    y = ops.mxfp4_linear(x, ops.mxfp4_pack(*w), n, bias=bias, activation=act, residual=residual,
                         dtype=dtype, save=act is not None)
    (pre, err), (want, bound) = epi.linear(x.double(), ref.decode(*w),
                                           None if bias is None else bias.double(), act,
                                           None if residual is None else residual.double(), dtype)
    if act:
        y, saved = y
        ref.within(saved, pre, epi.rounded(pre, err, BF16), "saved")
    ref.within(y, want, bound, f"{m}x{n}x{k}")


def test_linear_of_nothing_is_the_product(gen):
    """No bias, activation or residual: mxfp4_product's results, bit for bit."""
    for m, n, k in [(1, 100, 288), (20, 300, 2048), (300, 257, 544), (64, 4096, 4096)]:
        w, x = ops.mxfp4_pack(*ref.matrix(gen, n, k)), normal(gen, m, k).bfloat16()
        for dtype in (F32, BF16):
            assert torch.equal(ops.mxfp4_linear(x, w, n, dtype=dtype),
                               ops.mxfp4_product(x, w, n, dtype))


# m, n, k of dy [m, n] and dx [m, k]
BACKWARD = [(1, 8, 32), (2, 40, 64), (7, 2880, 2880), (33, 72, 96), (65, 264, 544),
            (77, 4096, 1440), (129, 64, 4128), (300, 1032, 288), (1025, 520, 2048),
            (2083, 1632, 2848), (64, 14336, 1024), (520, 608, 5024),
            (3272, 8, 1056), (2846, 16584, 64), (2832, 14744, 32), (2739, 15568, 32)]


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("m,n,k", BACKWARD)
def test_linear_backward(gen, m, n, k, act):
    w = ref.matrix(gen, n, k)
    dy, saved = normal(gen, m, n).bfloat16(), normal(gen, m, n).bfloat16() * 3
    dx, dpre = ops.mxfp4_linear_backward(dy, ops.mxfp4_pack(*w, transposed=True), k,
                                         saved=saved if act else None, activation=act)
    if act:
        d, err = epi.slope(saved.double(), act)
        want = dy.double() * d
        ref.within(dpre, want, epi.rounded(want, dy.double().abs() * err + want.abs() * 2.0 ** -22,
                                           BF16), "dpre")
    else:
        assert dpre is dy
    want, bound = ref.sum_bound(dpre.double(), ref.decode(*w).T)
    ref.within(dx, want, epi.rounded(want, bound, BF16), f"{m}x{n}x{k}")


# ---------------------------------------------------------------- experts

EXPERTS = [  # m, experts, n, k, rows: every kernel, one and no row, odd and long ones
    (1, 1, 1, 32, "even"), (1, 32, 96, 64, "even"), (4, 32, 2880, 2880, "even"),
    (4, 128, 2048, 768, "odd"), (5, 5, 33, 96, "even"), (16, 3, 100, 288, "odd"),
    (16, 128, 2048, 768, "even"), (14, 64, 2030, 800, "odd"),
    (16, 16, 8192, 96, "odd"), (24, 4, 300, 1056, "odd"), (32, 256, 640, 512, "even"),
    (40, 7, 257, 2080, "one"), (64, 32, 2880, 2880, "odd"), (100, 256, 130, 160, "odd"),
    (129, 2, 64, 4128, "even"), (256, 8, 777, 544, "odd"), (333, 32, 1030, 288, "odd"),
    (400, 12, 320, 1440, "even"), (513, 5, 500, 224, "odd"), (700, 3, 2100, 608, "even"),
    (1000, 9, 96, 2912, "one"), (2048, 32, 520, 352, "odd"), (2000, 16, 4096, 96, "even"),
    (5000, 255, 288, 128, "odd"), (27, 7, 385, 2912, "odd"), (90, 2, 72, 8192, "odd"),
    (330, 3, 257, 3968, "odd")]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act,with_bias,with_residual", EPILOGUES[:3])
@pytest.mark.parametrize("m,experts,n,k,kind", EXPERTS)
def test_experts_linear(gen, m, experts, n, k, kind, act, with_bias, with_residual, dtype):
    w, x = stack(gen, experts, n, k), normal(gen, m, k).bfloat16()
    offsets = offsets_of(counts_of(gen, m, experts, kind))
    bias = normal(gen, experts, n) if with_bias else None
    residual = normal(gen, m, n).to(dtype) if with_residual else None
    y = ops.mxfp4_linear(x, ops.mxfp4_pack(*w), n, bias=bias, activation=act, residual=residual,
                         dtype=dtype, offsets=offsets, save=act is not None)
    y, saved = y if act else (y, None)

    def check(e, rows, got, kept, add):
        (pre, err), (want, bound) = epi.linear(rows.double(), decoded(w, e),
                                               None if bias is None else bias[e].double(), act,
                                               add.double() if with_residual else None, dtype)
        ref.within(got, want, bound, f"expert {e}")
        if act:
            ref.within(kept, pre, epi.rounded(pre, err, BF16), "saved")

    epi.by_expert(check, offsets.tolist(), x, y, saved if act else y,
                  residual if with_residual else y)


GATED = [(1, 1, 32, 32, "even"), (4, 32, 2880, 2880, "even"), (4, 128, 768, 2048, "odd"),
         (5, 5, 64, 96, "even"), (16, 16, 4128, 96, "odd"), (16, 3, 96, 288, "odd"),
         (40, 7, 256, 2080, "one"), (64, 32, 2880, 1440, "odd"), (100, 256, 160, 160, "odd"),
         (129, 2, 64, 4128, "even"), (256, 8, 768, 544, "odd"), (400, 12, 320, 1440, "even"),
         (513, 5, 512, 224, "odd"), (700, 3, 2112, 608, "even"), (2048, 32, 544, 352, "odd"),
         (5000, 255, 288, 128, "odd"), (1, 3, 96, 4160, "odd"), (27, 7, 384, 2912, "odd"),
         (90, 2, 64, 8192, "odd"), (330, 3, 288, 3968, "odd")]


@pytest.mark.parametrize("save", [None, "bf16", "q8"])
@pytest.mark.parametrize("act,with_bias", [("silu", False), ("silu", True), ("clamped", True),
                                           ("clamped", False)])
@pytest.mark.parametrize("m,experts,n,k,kind", GATED)
def test_experts_gated(gen, m, experts, n, k, kind, act, with_bias, save):
    gate, up = stack(gen, experts, n, k), stack(gen, experts, n, k)
    x = (normal(gen, m, k) * (3 if act == "clamped" else 1)).bfloat16()
    offsets = offsets_of(counts_of(gen, m, experts, kind))
    bg, bu = (normal(gen, experts, n) * 2, normal(gen, experts, n)) if with_bias else (None, None)
    h = ops.mxfp4_experts_gated(x, offsets, ops.mxfp4_pack(*gate), ops.mxfp4_pack(*up), n,
                                gate_bias=bg, up_bias=bu, activation=act, save=save)
    h, saved = h if save else (h, None)
    if save == "q8":
        saved = (saved[0].view(m, -1, 32).double() * saved[1].double().unsqueeze(2)).flatten(1)

    def check(e, rows, got, kept):
        g, dg = epi.pre_activation(rows.double(), decoded(gate, e),
                                   bg[e].double() if with_bias else None)
        u, du = epi.pre_activation(rows.double(), decoded(up, e),
                                   bu[e].double() if with_bias else None)
        want, bound = epi.gated(g, dg, u, du, act)
        ref.within(got, want, bound, f"expert {e}")
        if save:
            both, err = torch.cat([g, u], 1), torch.cat([dg, du], 1)
            if save == "bf16":
                bound = epi.rounded(both, err, BF16)
            else:  # codes of amax / 127: half a step, and what amax and the quotient are off by
                top = (both.abs() + err).view(both.shape[0], -1, 32).amax(2, keepdim=True)
                bound = err + (top * (0.5 / 127 + 2.0 ** -20)).expand(-1, -1, 32).flatten(1)
            ref.within(kept, both, bound, "saved")

    epi.by_expert(check, offsets.tolist(), x, h, saved if save else h)


EXPERTS_BACKWARD = [
    (1, 1, 8, 32, "even"), (4, 32, 96, 64, "even"), (16, 3, 104, 288, "odd"),
    (64, 32, 2880, 1440, "odd"), (100, 256, 136, 160, "odd"), (129, 2, 64, 4128, "even"),
    (256, 8, 776, 544, "odd"), (400, 12, 320, 1440, "even"), (513, 5, 504, 224, "odd"),
    (700, 3, 2104, 608, "even"), (1000, 9, 96, 2912, "one"), (5000, 255, 288, 128, "odd"),
    (1, 3, 2600, 32, "odd"), (27, 7, 2904, 416, "odd"), (330, 3, 3960, 288, "odd")]


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("m,experts,n,k,kind", EXPERTS_BACKWARD)
def test_experts_linear_backward(gen, m, experts, n, k, kind, act):
    w = stack(gen, experts, n, k)
    offsets = offsets_of(counts_of(gen, m, experts, kind))
    dy, saved = normal(gen, m, n).bfloat16(), normal(gen, m, n).bfloat16() * 3
    dx, dpre = ops.mxfp4_linear_backward(dy, ops.mxfp4_pack(*w, transposed=True), k,
                                         saved=saved if act else None, activation=act,
                                         offsets=offsets)

    def check(e, d, got):
        want, bound = ref.sum_bound(d.double(), decoded(w, e).T)
        ref.within(got, want, epi.rounded(want, bound, BF16), f"expert {e}")

    epi.by_expert(check, offsets.tolist(), dpre, dx)
    if act:
        d, err = epi.slope(saved.double(), act)
        want = dy.double() * d
        ref.within(dpre, want, epi.rounded(want, dy.double().abs() * err + want.abs() * 2.0 ** -22,
                                           BF16), "dpre")


GATED_BACKWARD = [
    (1, 1, 32, 32, "even"), (4, 32, 96, 64, "even"), (16, 3, 96, 288, "odd"),
    (64, 32, 2880, 1440, "odd"), (100, 256, 160, 160, "odd"), (129, 2, 64, 4128, "even"),
    (256, 8, 768, 544, "odd"), (400, 12, 320, 1440, "even"), (513, 5, 512, 224, "odd"),
    (700, 3, 2112, 608, "even"), (5000, 255, 288, 128, "odd"), (4, 28, 3392, 96, "odd"),
    (27, 7, 2912, 416, "odd"), (330, 3, 3968, 288, "odd")]


@pytest.mark.parametrize("save", ["bf16", "q8"])
@pytest.mark.parametrize("act", ["silu", "clamped"])
@pytest.mark.parametrize("m,experts,n,k,kind", GATED_BACKWARD)
def test_experts_gated_backward(gen, m, experts, n, k, kind, act, save):
    gate, up = stack(gen, experts, n, k), stack(gen, experts, n, k)
    offsets = offsets_of(counts_of(gen, m, experts, kind))
    dh = normal(gen, m, n).bfloat16()
    if save == "bf16":
        saved = (normal(gen, m, 2 * n) * 4).bfloat16()
        saved[0, ::5], saved[0, 1::5], saved[0, 2::5] = 7.0, -7.0, 7.03125  # the clamps' borders
        kept = saved.double()
    else:
        saved = (torch.randint(-127, 128, (m, 2 * n), generator=gen, dtype=torch.int8,
                               device=gen.device),
                 torch.rand(m, n // 16, generator=gen, device=gen.device) / 8)
        kept = (saved[0].view(m, -1, 32).float() * saved[1].unsqueeze(2)).flatten(1).double()
    dx, dgu = ops.mxfp4_experts_gated_backward(
        dh, offsets, saved, ops.mxfp4_pack(*gate, transposed=True),
        ops.mxfp4_pack(*up, transposed=True), k, activation=act)
    want, bound = epi.gate_gradients(dh.double(), kept[:, :n], kept[:, n:], act)
    ref.within(dgu, want, bound, "dgu")

    def check(e, d, got):
        both = torch.cat([decoded(gate, e), decoded(up, e)])
        want, bound = ref.sum_bound(d.double(), both.T)
        ref.within(got, want, epi.rounded(want, bound, BF16), f"expert {e}")

    epi.by_expert(check, offsets.tolist(), dgu, dx)


# ---------------------------------------------------------------- forms, rows and places

def test_packed_stack_is_the_mixture_layers(gen):
    blocks, scales = stack(gen, 3, 96, 320)
    assert torch.equal(ops.mxfp4_pack(blocks, scales),
                       ops.moe_mxfp4_pack(blocks, scales, 3, 96, 320))
    one = ops.mxfp4_pack(blocks[:1], scales[:1])
    assert torch.equal(one, ops.mxfp4_pack(blocks[0], scales[0]))
    turned = ops.mxfp4_pack(blocks[:1], scales[:1], transposed=True)
    assert torch.equal(turned[0], ops.mxfp4_pack(blocks[0], scales[0], transposed=True))


@pytest.mark.parametrize("m,experts,n,k", [(9, 4, 70, 96), (600, 4, 160, 96),
                                           (60, 4, 96, 4160), (60, 4, 4160, 96)])
def test_rows_that_no_expert_has_stay(gen, m, experts, n, k):
    """Rows before the first offset and behind the last."""
    n = n // 32 * 32
    w, v = stack(gen, experts, n, k), stack(gen, experts, n, k)
    x = normal(gen, m, k).bfloat16()
    offsets = torch.tensor([2, 4, 4, m // 2, m - 3], dtype=torch.int32, device=gen.device)
    inside = torch.arange(m, device=gen.device)
    inside = (inside >= 2) & (inside < m - 3)
    for dtype in (F32, BF16):
        y = torch.full((m, n), 5.0, dtype=dtype, device=gen.device)
        ops.mxfp4_linear(x, ops.mxfp4_pack(*w), n, dtype=dtype, offsets=offsets, out=y)
        assert bool((y[~inside] == 5).all())
        whole = ops.mxfp4_linear(x[2:m - 3].contiguous(), ops.mxfp4_pack(*w), n, dtype=dtype,
                                 offsets=offsets - 2)
        ref.within(y[inside], whole.double(), (whole.double().abs() + 1) * 2.0 ** -7, "inside")
    h = torch.full((m, n), 5.0, dtype=BF16, device=gen.device)
    ops.mxfp4_experts_gated(x, offsets, ops.mxfp4_pack(*w), ops.mxfp4_pack(*v), n, out=h)
    assert bool((h[~inside] == 5).all()) and not bool((h[inside] == 5).all())
    dx = torch.full((m, k), 5.0, dtype=BF16, device=gen.device)
    turned = [ops.mxfp4_pack(*s, transposed=True) for s in (w, v)]
    ops.mxfp4_linear_backward(h, turned[0], k, offsets=offsets, out=dx)
    assert bool((dx[~inside] == 5).all())
    saved = normal(gen, m, 2 * n).bfloat16()
    ops.mxfp4_experts_gated_backward(h, offsets, saved, *turned, k, out=dx)
    assert bool((dx[~inside] == 5).all())


@pytest.mark.parametrize("m", [9, 600])
def test_offsets_outside_of_the_rows_are_the_nearer_end(gen, m):
    experts, n, k = 3, 64, 96
    w, x = ops.mxfp4_pack(*stack(gen, experts, n, k)), normal(gen, m, k).bfloat16()
    inside = torch.tensor([0, 5, 5, m], dtype=torch.int32, device=gen.device)
    outside = torch.tensor([-7, 5, 5, 2 ** 31 - 1], dtype=torch.int32, device=gen.device)
    assert torch.equal(ops.mxfp4_linear(x, w, n, offsets=inside),
                       ops.mxfp4_linear(x, w, n, offsets=outside))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_strided_rows_and_given_outputs(gen, m):
    n, k = 96, 160
    w = ref.matrix(gen, n, k)
    packed = ops.mxfp4_pack(*w)
    wide = normal(gen, m, 2 * k).bfloat16()
    x = wide[:, 8:8 + k]
    for dtype in (F32, BF16):
        around = normal(gen, m, n + 7).to(dtype)
        before, y = around.clone(), around[:, 3:3 + n]
        residual = normal(gen, m, n + 5).to(dtype)[:, 1:1 + n]
        bias = normal(gen, n + 1)[1:]  # from any element on
        got = ops.mxfp4_linear(x, packed, n, bias=bias, residual=residual, activation="silu",
                               dtype=dtype, out=y)
        assert got is y
        want = ops.mxfp4_linear(x.contiguous(), packed, n, bias=bias.clone(),
                                residual=residual.contiguous(), activation="silu", dtype=dtype)
        assert torch.equal(y, want)
        assert torch.equal(around[:, :3], before[:, :3])
        assert torch.equal(around[:, 3 + n:], before[:, 3 + n:])
        # onto the residual itself
        same = residual.contiguous()
        assert ops.mxfp4_linear(x, packed, n, bias=bias, residual=same, activation="silu",
                                dtype=dtype, out=same) is same
        assert torch.equal(same, want)
    dy = normal(gen, m, 2 * n).bfloat16()[:, 16:16 + n]
    turned, saved = ops.mxfp4_pack(*w, transposed=True), normal(gen, m, n).bfloat16()
    for act, kept in ((None, None), ("gelu", saved)):
        out = normal(gen, m, k + 9).bfloat16()
        dx, dpre = ops.mxfp4_linear_backward(dy, turned, k, saved=kept, activation=act,
                                             out=out[:, 5:5 + k])
        want, dwant = ops.mxfp4_linear_backward(dy.contiguous(), turned, k, saved=kept,
                                                activation=act)
        assert torch.equal(dx, want) and torch.equal(dpre, dwant)


@pytest.mark.parametrize("m", [6, 100, 700])
@pytest.mark.parametrize("n,k", [(96, 160), (96, 4160), (4160, 160)])  # (K slices of the long ones)
def test_strided_rows_of_experts(gen, m, n, k):
    experts = 4
    gate, up, down = stack(gen, experts, n, k), stack(gen, experts, n, k), stack(gen, experts, k, n)
    fwd = [ops.mxfp4_pack(*s) for s in (gate, up, down)]
    back = [ops.mxfp4_pack(*s, transposed=True) for s in (gate, up, down)]
    padded = torch.zeros(experts + 2, dtype=torch.int32, device=gen.device)
    padded[1:] = offsets_of(counts_of(gen, m, experts, "odd"))
    offsets = padded[1:]  # from any element on
    x = normal(gen, m, 2 * k).bfloat16()[:, 24:24 + k]
    around = normal(gen, m, n + 9).bfloat16()
    before, h = around.clone(), around[:, 5:5 + n]
    ops.mxfp4_experts_gated(x, offsets, fwd[0], fwd[1], n, out=h)
    want = ops.mxfp4_experts_gated(x.contiguous(), offsets.clone(), fwd[0], fwd[1], n)
    assert torch.equal(h, want)
    assert torch.equal(around[:, :5], before[:, :5])
    assert torch.equal(around[:, 5 + n:], before[:, 5 + n:])
    for dtype in (F32, BF16):
        residual = normal(gen, m, k + 3).to(dtype)[:, 2:2 + k]
        y = normal(gen, m, k + 5).to(dtype)[:, 1:1 + k]
        ops.mxfp4_linear(want, fwd[2], k, residual=residual, dtype=dtype, offsets=offsets, out=y)
        plain = ops.mxfp4_linear(want, fwd[2], k, residual=residual.contiguous(), dtype=dtype,
                                 offsets=offsets)
        assert torch.equal(y, plain)
        same = residual.contiguous()
        ops.mxfp4_linear(want, fwd[2], k, residual=same, dtype=dtype, offsets=offsets, out=same)
        assert torch.equal(same, plain)
    dy = normal(gen, m, 2 * k).bfloat16()[:, 8:8 + k]
    dh = normal(gen, m, n + 11).bfloat16()[:, 3:3 + n]
    ops.mxfp4_linear_backward(dy, back[2], n, offsets=offsets, out=dh)
    plain, _ = ops.mxfp4_linear_backward(dy.contiguous(), back[2], n, offsets=offsets)
    assert torch.equal(dh, plain)
    saved = normal(gen, m, 2 * n).bfloat16()
    wide = normal(gen, m, n + 8).bfloat16()
    wide[:, 8:] = plain
    dx = normal(gen, m, k + 1).bfloat16()[:, 1:]
    ops.mxfp4_experts_gated_backward(wide[:, 8:], offsets, saved, back[0], back[1], k, out=dx)
    plain, _ = ops.mxfp4_experts_gated_backward(plain, offsets, saved, back[0], back[1], k)
    assert torch.equal(dx, plain)


@pytest.mark.parametrize("m", [4, 500])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_values_that_are_not_finite_stay_in_their_rows(gen, m, bad):
    """An infinite or NaN row of x reaches its own results only, its neighbours' in a tile and the
    next expert's not."""
    experts, n, k = 3, 64, 416
    w, v = ops.mxfp4_pack(*stack(gen, experts, n, k)), ops.mxfp4_pack(*stack(gen, experts, n, k))
    offsets = torch.tensor([0, m // 2, m // 2, m], dtype=torch.int32, device=gen.device)
    x = normal(gen, m, k).bfloat16()
    clean = (ops.mxfp4_linear(x, w, n, offsets=offsets),
             ops.mxfp4_experts_gated(x, offsets, w, v, n))
    row = m // 2 - 1
    x[row] = bad
    spoilt = (ops.mxfp4_linear(x, w, n, offsets=offsets),
              ops.mxfp4_experts_gated(x, offsets, w, v, n))
    for a, b in zip(clean, spoilt):
        keep = torch.arange(m, device=gen.device) != row
        assert torch.equal(a[keep], b[keep])
        assert not bool(torch.isfinite(b[row].float()).all())


@pytest.mark.parametrize("m", [4, 40, 500])
@pytest.mark.parametrize("k", [352, 768, 2080])
def test_a_block_without_a_scale_reaches_its_own_results_only(gen, m, k):
    """Scale byte 255 (NaN) in one row of one expert's matrix."""
    experts, n = 3, 96
    (blocks, scales), other = stack(gen, experts, n, k), ops.mxfp4_pack(*stack(gen, experts, n, k))
    offsets = torch.tensor([0, m // 4, m // 2, m], dtype=torch.int32, device=gen.device)
    x = normal(gen, m, k).bfloat16()
    for block in (0, k // 64, k // 32 - 1):
        w = ops.mxfp4_pack(blocks, scales)
        bad = scales.clone()
        bad[1, 37, block] = 255
        v = ops.mxfp4_pack(blocks, bad)
        hit = torch.zeros(m, n, dtype=torch.bool, device=gen.device)
        hit[m // 4:m // 2, 37] = True
        for f in (lambda p: ops.mxfp4_linear(x, p, n, offsets=offsets),
                  lambda p: ops.mxfp4_experts_gated(x, offsets, p, other, n),
                  lambda p: ops.mxfp4_experts_gated(x, offsets, other, p, n)):
            want, got = f(w), f(v)
            assert torch.equal(got[~hit], want[~hit]) and bool(torch.isnan(got[hit]).all())


@pytest.mark.parametrize("n,k", [(160, 288), (160, 4160), (4160, 288)])
def test_two_calls_at_once(gen, n, k):
    """Calls on two streams share nothing."""
    experts, top_k = 8, 2
    w = ops.mxfp4_pack(*stack(gen, experts, n, k))
    turned = ops.mxfp4_pack(*stack(gen, experts, n, k), transposed=True)
    batches = []
    for tokens in (7, 300):
        x = normal(gen, tokens, k).bfloat16()
        _, weights, offsets, perm = ops.moe_route(normal(gen, tokens, experts), top_k)
        batches.append((x, weights, offsets, perm))

    def chain(x, weights, offsets, perm):
        rows, place = ops.moe_sort(x, perm, top_k)
        y = ops.mxfp4_linear(rows, w, n, activation="gelu", dtype=BF16, offsets=offsets)
        d, dw = ops.moe_combine_backward(ops.moe_combine(y, weights, place), y, weights, place)
        return y, d, dw, ops.mxfp4_linear_backward(d, turned, k, offsets=offsets)[0]

    want = [chain(*b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(chain(*batches[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


@pytest.mark.parametrize("m", [4, 64, 700])
@pytest.mark.parametrize("n,k", [(96, 160), (96, 4160), (4160, 160)])
def test_on_another_stream_and_captured(gen, m, n, k):
    """A graph of the experts' projections and their gradients, replayed with other inputs, and
    other rows for each expert, between eager work."""
    experts = 6
    gate, up, down = stack(gen, experts, n, k), stack(gen, experts, n, k), stack(gen, experts, k, n)
    fwd = [ops.mxfp4_pack(*s) for s in (gate, up, down)]
    back = [ops.mxfp4_pack(*s, transposed=True) for s in (gate, up, down)]
    x, dy = normal(gen, m, k).bfloat16(), normal(gen, m, k).bfloat16()
    bias = normal(gen, experts, k)
    offsets = offsets_of(counts_of(gen, m, experts, "even"))

    def chain():
        h, saved = ops.mxfp4_experts_gated(x, offsets, fwd[0], fwd[1], n, save="bf16")
        y = ops.mxfp4_linear(h, fwd[2], k, bias=bias, dtype=BF16, offsets=offsets)
        dh, _ = ops.mxfp4_linear_backward(dy, back[2], n, offsets=offsets)
        dx, dgu = ops.mxfp4_experts_gated_backward(dh, offsets, saved, back[0], back[1], k)
        return h, saved, y, dh, dx, dgu

    eager = chain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    for kind in ("odd", "one", "even"):
        x.copy_(normal(gen, m, k))
        dy.copy_(normal(gen, m, k))
        offsets.copy_(offsets_of(counts_of(gen, m, experts, kind)))
        eager = chain()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))


# ---------------------------------------------------------------- a whole layer

class Mixture(torch.autograd.Function):
    """A mixture layer over frozen MXFP4 experts: the way the pieces are used together."""

    @staticmethod
    def forward(ctx, x, logits, stream, fwd, back, biases, top_k, n):
        idx, w, offsets, perm = ops.moe_route(logits, top_k)
        rows, place = ops.moe_sort(x, perm, top_k)
        h, saved = ops.mxfp4_experts_gated(rows, offsets, fwd[0], fwd[1], n, biases[0], biases[1],
                                           activation="clamped", save="bf16")
        out = ops.mxfp4_linear(h, fwd[2], x.shape[1], bias=biases[2], dtype=BF16, offsets=offsets)
        ctx.save_for_backward(idx, w, offsets, place, saved, out)
        ctx.back, ctx.k, ctx.n, ctx.experts = back, x.shape[1], n, logits.shape[1]
        return ops.moe_combine(out, w, place, residual=stream, dtype=stream.dtype)

    @staticmethod
    def backward(ctx, dy):
        idx, w, offsets, place, saved, out = ctx.saved_tensors
        dout, dw = ops.moe_combine_backward(dy.contiguous(), out, w, place)
        dh, _ = ops.mxfp4_linear_backward(dout, ctx.back[2], ctx.n, offsets=offsets)
        drows, _ = ops.mxfp4_experts_gated_backward(dh, offsets, saved, ctx.back[0], ctx.back[1],
                                                    ctx.k, activation="clamped")
        return (ops.moe_sort_backward(drows, place, w.shape[1]),
                ops.moe_route_backward(idx, w, dw, ctx.experts), dy, None, None, None, None, None)


@pytest.mark.parametrize("tokens,experts,top_k,k,n", [(1, 8, 2, 96, 64), (37, 16, 4, 160, 96),
                                                      (400, 8, 3, 288, 160)])
def test_mixture_layer_and_its_gradients(gen, tokens, experts, top_k, k, n):
    gate, up, down = stack(gen, experts, n, k), stack(gen, experts, n, k), stack(gen, experts, k, n)
    biases = [0.3 * normal(gen, experts, n), 0.3 * normal(gen, experts, n),
              0.3 * normal(gen, experts, k)]
    fwd = [ops.mxfp4_pack(*s) for s in (gate, up, down)]
    back = [ops.mxfp4_pack(*s, transposed=True) for s in (gate, up, down)]
    x = normal(gen, tokens, k).bfloat16().requires_grad_(True)
    logits = normal(gen, tokens, experts).requires_grad_(True)
    stream = normal(gen, tokens, k).requires_grad_(True)
    y = Mixture.apply(x, logits, stream, fwd, back, biases, top_k, n)
    dy = normal(gen, tokens, k)
    y.backward(dy)
    # the same layer in 64 bits, by autograd
    leaves = [t.detach().double().requires_grad_(True) for t in (x, logits, stream)]
    p = torch.softmax(leaves[1], 1)
    idx = ops.moe_route(logits.detach(), top_k)[0].long()
    w = p.gather(1, idx)
    w = w / w.sum(1, keepdim=True)
    want = leaves[2]
    for e in range(experts):
        g = leaves[0] @ decoded(gate, e).T + biases[0][e].double()
        u = leaves[0] @ decoded(up, e).T + biases[1][e].double()
        h = epi.clamped(g, u)[0]
        out = h @ decoded(down, e).T + biases[2][e].double()
        want = want + out * (w * (idx == e)).sum(1, keepdim=True)
    want.backward(dy.double())
    # bf16 in between: rows, h, out, dout, dh, dgu, drows, each half a step of its values, so of
    # independent sign: together below 8 halves of a step of the whole's root mean square
    for got, exact, steps in ((y, want, 8), (x.grad, leaves[0].grad, 8),
                              (logits.grad, leaves[1].grad, 8), (stream.grad, leaves[2].grad, 1)):
        off, size = (got.detach().double() - exact.detach()), exact.detach()
        assert float(off.square().mean()) ** 0.5 <= (
            steps * ref.HALF_BF16 * float(size.square().mean()) ** 0.5)


def test_serving_forward_agrees_with_the_mixture_layer(gen):
    """Route, sort, gate, down and combine against kdq_moe_mxfp4_packed, one resident copy of the
    weights for both."""
    experts, top_k, k, n = 32, 4, 320, 192
    gate, up, down = stack(gen, experts, n, k), stack(gen, experts, n, k), stack(gen, experts, k, n)
    packed = [ops.mxfp4_pack(*s) for s in (gate, up, down)]
    for tokens in (1, 6, 200):
        x, logits = normal(gen, tokens, k).bfloat16(), normal(gen, tokens, experts)
        want = ops.moe_mxfp4_packed(x, logits, top_k, n, *packed)
        _, w, offsets, perm = ops.moe_route(logits, top_k)
        rows, place = ops.moe_sort(x, perm, top_k)
        h = ops.mxfp4_experts_gated(rows, offsets, packed[0], packed[1], n)
        out = ops.mxfp4_linear(h, packed[2], k, offsets=offsets)
        y = ops.moe_combine(out, w, place)
        # h is rounded to bf16 here and to about 12 bits there
        off = float((y - want).double().square().mean().sqrt())
        assert off <= 2 * ref.HALF_BF16 * float(want.double().square().mean().sqrt())


def test_wrapper_refusals(gen):
    n, k, m, experts = 64, 96, 8, 4
    one, many = ref.matrix(gen, n, k), stack(gen, experts, n, k)
    w, ws = ops.mxfp4_pack(*one), ops.mxfp4_pack(*many)
    t, ts = ops.mxfp4_pack(*one, transposed=True), ops.mxfp4_pack(*many, transposed=True)
    x, dy = normal(gen, m, k).bfloat16(), normal(gen, m, n).bfloat16()
    bias, biases = normal(gen, n), normal(gen, experts, n)
    offsets = offsets_of(counts_of(gen, m, experts, "even"))
    saved = normal(gen, m, 2 * n).bfloat16()
    refused = [
        lambda: ops.mxfp4_linear(x.float(), w, n), lambda: ops.mxfp4_linear(x, w, n + 32),
        lambda: ops.mxfp4_linear(x, t, n), lambda: ops.mxfp4_linear(x, ws, n),
        lambda: ops.mxfp4_linear(x, w, n, offsets=offsets),
        lambda: ops.mxfp4_linear(x, ts, n, offsets=offsets),
        lambda: ops.mxfp4_linear(x, ws, n, offsets=offsets.long()),
        lambda: ops.mxfp4_linear(x, ws, n, offsets=offsets[:1]),
        lambda: ops.mxfp4_linear(x, ws, n, offsets=offsets.cpu()),
        lambda: ops.mxfp4_linear(x, w, n, bias=biases),
        lambda: ops.mxfp4_linear(x, w, n, bias=bias.bfloat16()),
        lambda: ops.mxfp4_linear(x, w, n, bias=bias[:-1]),
        lambda: ops.mxfp4_linear(x, ws, n, bias=bias, offsets=offsets),
        lambda: ops.mxfp4_linear(x, w, n, activation="clamped"),
        lambda: ops.mxfp4_linear(x, w, n, activation="relu"),
        lambda: ops.mxfp4_linear(x, w, n, residual=dy),
        lambda: ops.mxfp4_linear(x, w, n, save=True),
        lambda: ops.mxfp4_linear(x, w, n, dtype=torch.float16),
        lambda: ops.mxfp4_linear(x, w, n, bias=bias.requires_grad_(True)),
        lambda: ops.mxfp4_linear(x.float().requires_grad_(True).bfloat16(), w, n),
        lambda: ops.mxfp4_linear_backward(dy, w, k), lambda: ops.mxfp4_linear_backward(dy, ts, k),
        lambda: ops.mxfp4_linear_backward(dy, t, k, offsets=offsets),
        lambda: ops.mxfp4_linear_backward(dy, t, k, saved=dy),
        lambda: ops.mxfp4_linear_backward(dy, t, k, activation="silu"),
        lambda: ops.mxfp4_linear_backward(dy, t, k, saved=dy[:4], activation="silu"),
        lambda: ops.mxfp4_linear_backward(dy[:, :63], t, k),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, w, n),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, ws, n, gate_bias=biases),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, ws, n, biases, biases[:2]),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, ws, n, activation="gelu"),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, ws, n, activation=None),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, ws, n, save="f32"),
        lambda: ops.mxfp4_experts_gated(x, offsets, ws, ws, n - 1),
        lambda: ops.mxfp4_experts_gated_backward(dy, offsets, saved, ts, ws, k),
        lambda: ops.mxfp4_experts_gated_backward(dy, offsets, dy, ts, ts, k),
        lambda: ops.mxfp4_experts_gated_backward(dy, offsets, saved, ts, ts, k, activation="gelu"),
        lambda: ops.mxfp4_pack(many[0], many[1][:2]),
        lambda: ops.mxfp4_pack(many[0][:, :, :8], many[1]),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((ValueError, kadan_amd.KdqError)):
            call()
            raise AssertionError(f"call {i} was not refused")
