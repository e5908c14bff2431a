"""A mixture layer whose experts take a limited number of rows: what does not fit is dropped, so the
permutation ends in entries that are no slot and rows that no expert has, and no value of theirs may
reach a result or a gradient."""
import pytest
import torch

from kadan_amd import ops

import mxfp4_epilogue_reference as epi
import mxfp4_reference as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(404)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def poison(device, megabytes=256):
    """Leaves NaN and valid positions in the memory that the next tensors get."""
    for size in (1 << 10, 1 << 13, 1 << 16, 1 << 19, megabytes << 18):
        for _ in range(4):
            held = [torch.full((size,), float("nan"), device=device),
                    torch.zeros(size, dtype=torch.int32, device=device)]
    del held


@pytest.mark.parametrize("tokens,experts,top_k,room,k,n", [
    (6, 4, 2, 2, 96, 64), (37, 16, 4, 6, 160, 96), (400, 8, 3, 100, 288, 160),
    (600, 8, 8, 500, 96, 64), (5000, 4, 4, 3000, 64, 64)])
def test_layer_of_limited_experts(gen, tokens, experts, top_k, room, k, n):
    slots = tokens * top_k
    stacks = []
    for rows, cols in ((n, k), (n, k), (k, n)):
        blocks, scales = ref.matrix(gen, experts * rows, cols)
        stacks.append((blocks.view(experts, rows, -1), scales.view(experts, rows, -1)))
    fwd = [ops.mxfp4_pack(*s) for s in stacks]
    back = [ops.mxfp4_pack(*s, transposed=True) for s in stacks]
    bias = 0.3 * normal(gen, experts, k)
    logits = normal(gen, tokens, experts) + normal(gen, experts)
    idx, weights, offsets, perm = ops.moe_route(logits, top_k)
    # an expert keeps its first `room` rows; the rest leave the permutation, which is closed up
    counts = (offsets[1:] - offsets[:-1]).clamp(max=room)
    within = torch.arange(slots, device=gen.device) - offsets[:-1].long().repeat_interleave(
        (offsets[1:] - offsets[:-1]).long())
    kept = perm[within < room]
    assert kept.numel() < slots
    limited = torch.full_like(perm, -1)
    limited[:kept.numel()] = kept
    ends = torch.zeros_like(offsets)
    ends[1:] = torch.cumsum(counts, 0)
    there = torch.zeros(slots, dtype=torch.bool, device=gen.device)
    there[kept.long()] = True
    there = there.view(tokens, top_k)

    x, stream = normal(gen, tokens, k).bfloat16(), normal(gen, tokens, k)
    dy = normal(gen, tokens, k)
    torch.cuda.synchronize()
    poison(gen.device)
    rows, place = ops.moe_sort(x, limited, top_k)
    h, saved = ops.mxfp4_experts_gated(rows, ends, fwd[0], fwd[1], n, activation="clamped",
                                       save="bf16")
    out = ops.mxfp4_linear(h, fwd[2], k, bias=bias, dtype=BF16, offsets=ends)
    y = ops.moe_combine(out, weights, place, residual=stream, dtype=torch.float32)
    dout, dw = ops.moe_combine_backward(dy, out, weights, place)
    dh, _ = ops.mxfp4_linear_backward(dout, back[2], n, offsets=ends)
    drows, _ = ops.mxfp4_experts_gated_backward(dh, ends, saved, back[0], back[1], k,
                                                activation="clamped")
    dx = ops.moe_sort_backward(drows, place, top_k)

    assert bool((place.view(tokens, top_k)[~there] == -1).all()) and not bool(dw[~there].any())
    assert not bool(dout[kept.numel():].any())
    # the bias's gradient: the rows' of each expert, and of all experts all rows'
    within_experts = [dout[a:b].double().sum(0) for a, b in zip(ends.tolist(), ends.tolist()[1:])]
    assert torch.allclose(torch.stack(within_experts).sum(0), dout.double().sum(0))
    leaves = [t.double().requires_grad_(True) for t in (x, stream, weights)]
    want = leaves[1]
    mask = leaves[2] * there
    for e in range(experts):
        g, u = (leaves[0] @ ref.decode(s[0][e], s[1][e]).T for s in stacks[:2])
        o = epi.clamped(g, u)[0] @ ref.decode(stacks[2][0][e], stacks[2][1][e]).T + bias[e].double()
        want = want + o * (mask * (idx == e)).sum(1, keepdim=True)
    want.backward(dy.double())
    # bf16 in between: rows, h, out, dout, dh, dgu, drows, each half a step of its values, so of
    # independent sign: together below 8 halves of a step of the whole's root mean square
    for got, exact in ((y, want.detach()), (dx, leaves[0].grad), (dw, leaves[2].grad)):
        off = float((got.double() - exact).square().mean().sqrt())
        assert off <= 8 * ref.HALF_BF16 * float(exact.square().mean().sqrt())
