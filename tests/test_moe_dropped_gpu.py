"""Selections that are dropped: entries of a mixture's permutation that are no slot, so that as many
slots have no place.  Outputs are handed over full of what an earlier call might have left there."""
import pytest
import torch

import kadan_amd
from kadan_amd import ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
KIND = {F32: 0, F16: 1, BF16: 30}  # KDQ_F32, KDQ_F16, KDQ_BF16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step, relative
LEAST = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}

# tokens, top_k, cols: one slot, a few, as many as one workgroup writes the places of and one more,
# the most whose places the rows' launch writes and one more, 32 MB of rows and more
SIZES = [(1, 1, 1), (1, 4, 2880), (5, 3, 77), (64, 8, 65), (300, 5, 129), (512, 8, 333),
         (1024, 4, 64), (4097, 1, 40), (2389, 5, 33), (4096, 8, 12), (32769, 1, 3), (30000, 3, 9),
         (1100, 8, 2050), (4100, 2, 4101)]


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(77)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def dropped(g, slots, share):
    """A permutation of the slots with a share of its entries, one at least, replaced by numbers
    that are none, and which positions those are."""
    perm = torch.randperm(slots, generator=g, device=g.device).int()
    gone = torch.rand(slots, generator=g, device=g.device) < share
    gone[torch.randint(slots, (1,), generator=g, device=g.device)] = True
    none = torch.tensor([-1, slots, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32, device=g.device)
    bad = none[torch.arange(slots, device=g.device) % 4]
    return torch.where(gone, bad, perm), gone


def sort(x, perm, top_k):
    """kdq_moe_sort into rows of NaN and places that are positions."""
    slots, cols = perm.numel(), x.shape[1]
    rows = torch.full((slots, cols), float("nan"), dtype=x.dtype, device=x.device)
    place = torch.arange(slots, dtype=torch.int32, device=x.device).flip(0).contiguous()
    kadan_amd.call("kdq_moe_sort", KIND[x.dtype], x.data_ptr(), cols, x.shape[0], cols, top_k,
                   perm.data_ptr(), rows.data_ptr(), cols, place.data_ptr(),
                   torch.cuda.current_stream().cuda_stream)
    return rows, place


def places(perm):
    """The inverse of the permutation, -1 where there is none."""
    slots = perm.numel()
    there = (perm >= 0) & (perm < slots)
    want = torch.full((slots,), -1, dtype=torch.int32, device=perm.device)
    want[perm[there].long()] = torch.arange(slots, dtype=torch.int32, device=perm.device)[there]
    return want


@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,top_k,cols", SIZES)
def test_a_slot_that_the_permutation_does_not_name_has_no_place(gen, tokens, top_k, cols, dtype,
                                                                share):
    slots = tokens * top_k
    perm, gone = dropped(gen, slots, share)
    x = normal(gen, tokens, cols).to(dtype)
    rows, place = sort(x, perm, top_k)
    want = x[perm.where(~gone, torch.zeros_like(perm)).long() // top_k]
    want[gone] = 0
    assert torch.equal(rows, want)
    assert torch.equal(place, places(perm))
    # (and through the wrapper)
    again, at = ops.moe_sort(x, perm, top_k)
    assert torch.equal(again, want) and torch.equal(at, place)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,top_k,cols", SIZES)
def test_dropped_selections_on_their_way_back(gen, tokens, top_k, cols, dtype):
    """moe_sort's own places, of a permutation that drops some, in the sums and their gradients."""
    slots = tokens * top_k
    perm, gone = dropped(gen, slots, 0.25)
    _, place = sort(normal(gen, tokens, cols).to(dtype), perm, top_k)
    rows, dy = normal(gen, slots, cols).to(dtype), normal(gen, tokens, cols).to(dtype)
    weights = torch.rand(tokens, top_k, generator=gen, device=gen.device)
    there = (place >= 0).reshape(tokens, top_k)
    each = rows.double()[place.clamp(min=0).long()].reshape(tokens, top_k, cols)
    each = each * there.unsqueeze(2)

    def within(got, want, bound):
        bound = bound + (want.abs() + bound) * HALF[got.dtype] + LEAST[got.dtype]
        assert bool(((got.double() - want).abs() <= bound).all())

    y = ops.moe_combine(rows, weights, place)
    within(y, (each * weights.double().unsqueeze(2)).sum(1),
           top_k * HALF[F32] * (each.abs() * weights.double().unsqueeze(2)).sum(1))
    within(ops.moe_sort_backward(rows, place, top_k), each.sum(1),
           top_k * HALF[F32] * each.abs().sum(1))
    drows, dweights = ops.moe_combine_backward(dy, rows, weights, place)
    terms = dy.double().unsqueeze(1) * each
    within(dweights, terms.sum(2), (cols + 1) * HALF[F32] * terms.abs().sum(2))
    assert not bool(dweights[~there].any())
    slot = perm[~gone].long()
    want = dy.double()[slot // top_k] * weights.double().reshape(-1, 1)[slot]
    within(drows[~gone], want, HALF[F32] * want.abs())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,top_k,cols", SIZES + [(512, 8, 500), (513, 8, 500),
                                                       (700, 6, 1400), (2048, 8, 1600),
                                                       (10923, 3, 1537)])
def test_rows_that_no_place_names_have_a_gradient_of_zero(gen, tokens, top_k, cols, dtype):
    """Into rows of NaN, some values apart; the values between them stay."""
    slots = tokens * top_k
    perm, gone = dropped(gen, slots, 0.25)
    place = places(perm)
    place[place < 0] = torch.tensor([-1, slots, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32,
                                    device=gen.device).repeat(slots)[:int((place < 0).sum())]
    rows, dy = normal(gen, slots, cols).to(dtype), normal(gen, tokens, cols).to(dtype)
    weights = torch.rand(tokens, top_k, generator=gen, device=gen.device)
    drows = torch.full((slots, cols + 3), float("nan"), dtype=dtype, device=gen.device)
    dweights = torch.full((tokens, top_k), float("nan"), device=gen.device)
    kadan_amd.call("kdq_moe_combine_backward", KIND[dtype], rows.data_ptr(), cols, place.data_ptr(),
                   weights.data_ptr(), tokens, cols, top_k, KIND[dtype], dy.data_ptr(), cols,
                   drows.data_ptr(), cols + 3, dweights.data_ptr(),
                   torch.cuda.current_stream().cuda_stream)
    assert bool(drows[:, cols:].isnan().all())
    assert not bool(drows[gone, :cols].any())
    slot = perm[~gone].long()
    want = dy.double()[slot // top_k] * weights.double().reshape(-1, 1)[slot]
    off = (drows[~gone, :cols].double() - want).abs()
    bound = HALF[F32] * want.abs()
    assert bool((off <= bound + (want.abs() + bound) * HALF[dtype] + LEAST[dtype]).all())
    again, dw = ops.moe_combine_backward(dy, rows, weights, place)
    assert torch.equal(again, drows[:, :cols]) and torch.equal(dw, dweights)


@pytest.mark.parametrize("way", ["sort", "back"])
@pytest.mark.parametrize("tokens,top_k,cols", [(4096, 8, 2048), (600, 8, 16384), (500, 8, 16384)])
def test_dropped_selections_cost_no_more_than_the_others(gen, tokens, top_k, cols, way):
    """Rows of zeros are written by as many lanes as rows of tokens: a permutation of which half is
    dropped takes no twice as long as one of which nothing is."""
    slots = tokens * top_k
    x = normal(gen, tokens, cols).bfloat16()
    rows, weights = normal(gen, slots, cols).bfloat16(), normal(gen, tokens, top_k)
    took = []
    for share in (None, 0.5):
        perm = (dropped(gen, slots, share)[0] if share else
                torch.randperm(slots, generator=gen, device=gen.device).int())
        place = places(perm)
        times = []
        for _ in range(7):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            for _ in range(5):
                if way == "sort":
                    ops.moe_sort(x, perm, top_k)
                else:
                    ops.moe_combine_backward(x, rows, weights, place)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        took.append(sorted(times)[len(times) // 2])
    assert took[1] <= 2 * took[0]


@pytest.mark.parametrize("tokens,top_k,cols", [(64, 4, 72), (4097, 4, 40), (9000, 4, 40),
                                               (2100, 8, 1100)])
def test_captured_with_other_drops_at_every_replay(gen, tokens, top_k, cols):
    slots = tokens * top_k
    x, dy = normal(gen, tokens, cols).bfloat16(), normal(gen, tokens, cols).bfloat16()
    weights = torch.rand(tokens, top_k, generator=gen, device=gen.device)
    perm, _ = dropped(gen, slots, 0.2)

    def chain():
        rows, place = ops.moe_sort(x, perm, top_k)
        y = ops.moe_combine(rows, weights, place, residual=x)
        drows, dweights = ops.moe_combine_backward(dy, rows, weights, place)
        return rows, place, y, drows, dweights, ops.moe_sort_backward(drows, place, top_k)

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    for share in (0.5, 0.0, 1.0, 0.1):
        other, gone = dropped(gen, slots, share)
        perm.copy_(other)
        x.copy_(normal(gen, tokens, cols))
        eager = chain()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))
        assert not bool(captured[0][gone].any()) and not bool(captured[3][gone].any())
        assert torch.equal(captured[1], places(perm))
