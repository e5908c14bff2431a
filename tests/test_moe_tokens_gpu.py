"""Tokens sorted by expert and back, and the router's gradient (kdq_moe_sort, _sort_backward,
_combine, _combine_backward, _route_backward), against their definitions in 64 bits."""
import pytest
import torch

from kadan_amd import ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
# half a step, relative, and of the least exponent, absolute
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
LEAST = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}
BITS = {F32: torch.int32, F16: torch.int16, BF16: torch.int16}

# tokens, experts, top_k, cols: one of each, odd rows, every way rows share a workgroup, rows of
# several workgroups
SIZES = [(1, 1, 1, 1), (1, 4, 4, 2880), (3, 5, 2, 7), (5, 32, 4, 2880), (17, 8, 3, 8),
         (33, 16, 8, 9), (64, 128, 8, 65), (7, 256, 5, 1023), (100, 12, 6, 511), (257, 9, 7, 128),
         (1000, 64, 4, 333), (6, 4, 4, 2049), (2, 3, 3, 8192), (513, 128, 8, 2048)]


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(99)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def routed(g, tokens, experts, top_k):
    return ops.moe_route(normal(g, tokens, experts) + normal(g, experts), top_k)


def within(got, want, bound, dtype, what):
    """want within bound of got, once want is rounded to dtype."""
    off = (got.double() - want).abs()
    bound = bound + (want.abs() + bound) * HALF[dtype] + LEAST[dtype]
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(off[bad].max()))


def same(a, b):
    return torch.equal(a.contiguous().view(BITS[a.dtype]), b.contiguous().view(BITS[b.dtype]))


def combined(rows, weights, place, residual=None):
    """y and the sum of its terms' magnitudes, in 64 bits."""
    tokens, top_k = weights.shape
    terms = rows.double()[place.long()].reshape(tokens, top_k, -1) * weights.double().unsqueeze(2)
    y, size = terms.sum(1), terms.abs().sum(1)
    return (y, size) if residual is None else (y + residual.double(),
                                               size + residual.double().abs())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top_k,cols", SIZES)
def test_sort_is_a_copy_and_back_a_sum(gen, tokens, experts, top_k, cols, dtype):
    _, _, offsets, perm = routed(gen, tokens, experts, top_k)
    x = normal(gen, tokens, cols).to(dtype)
    x[0, 0], x[-1, -1] = float("nan"), float("inf")
    rows, place = ops.moe_sort(x, perm, top_k)
    assert same(rows, x[perm.long() // top_k])
    assert torch.equal(place[perm.long()].long(), torch.arange(tokens * top_k, device=x.device))
    drows = normal(gen, tokens * top_k, cols).to(dtype)
    dx = ops.moe_sort_backward(drows, place, top_k)
    ones = torch.ones(tokens, top_k, device=x.device)
    want, size = combined(drows, ones, place)
    within(dx, want, top_k * HALF[F32] * size, dtype, "dx")


@pytest.mark.parametrize("dtype,out", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16),
                                       (BF16, F32)])
@pytest.mark.parametrize("tokens,experts,top_k,cols", SIZES)
def test_combine_and_its_gradients(gen, tokens, experts, top_k, cols, dtype, out):
    _, weights, _, perm = routed(gen, tokens, experts, top_k)
    x = normal(gen, tokens, cols).to(dtype)
    _, place = ops.moe_sort(x, perm, top_k)
    rows = normal(gen, tokens * top_k, cols).to(dtype)
    residual = normal(gen, tokens, cols).to(out)
    for add in (None, residual):
        y = ops.moe_combine(rows, weights, place, residual=add, dtype=out)
        assert y.dtype == out and y.shape == (tokens, cols)
        want, size = combined(rows, weights, place, add)
        within(y, want, top_k * HALF[F32] * size, out, "y")
    dy = normal(gen, tokens, cols).to(out)
    drows, dweights = ops.moe_combine_backward(dy, rows, weights, place)
    of = torch.empty(tokens * top_k, dtype=torch.long, device=x.device)
    of[place.long()] = torch.arange(tokens * top_k, device=x.device)
    spread = dy.double()[of // top_k]
    within(drows, spread * weights.double().reshape(-1, 1)[of],
           HALF[F32] * spread.abs() + LEAST[F32], dtype, "drows")
    terms = dy.double().unsqueeze(1) * rows.double()[place.long()].reshape(tokens, top_k, cols)
    within(dweights, terms.sum(2), (cols + 1) * HALF[F32] * terms.abs().sum(2), F32, "dweights")


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_given_outputs(gen, dtype):
    tokens, top_k, cols = 19, 4, 77
    _, weights, _, perm = routed(gen, tokens, 8, top_k)
    wide = normal(gen, tokens, 2 * cols + 3).to(dtype)
    x = wide[:, 5:5 + cols]  # odd rows from an odd element on
    rows, place = ops.moe_sort(x, perm, top_k)
    assert same(rows, x[perm.long() // top_k])
    big = normal(gen, tokens * top_k, 3 * cols).to(dtype)
    part = big[:, cols + 1:2 * cols + 1]
    assert same(ops.moe_sort_backward(part, place, top_k),
                ops.moe_sort_backward(part.contiguous(), place, top_k))
    around = normal(gen, tokens, cols + 6).to(dtype)
    before = around.clone()
    y = around[:, 3:3 + cols]
    assert ops.moe_combine(part, weights, place, residual=x, out=y) is y
    assert same(y, ops.moe_combine(part.contiguous(), weights, place, residual=x.contiguous()))
    assert same(around[:, :3], before[:, :3]) and same(around[:, 3 + cols:], before[:, 3 + cols:])
    got = ops.moe_combine_backward(x, part, weights, place)
    for a, b in zip(got, ops.moe_combine_backward(x.contiguous(), part.contiguous(), weights,
                                                  place)):
        assert same(a, b)


@pytest.mark.parametrize("dtype,tokens,top_k,cols", [
    (BF16, 1100, 8, 2050), (F16, 4100, 2, 2047), (F32, 900, 3, 4101), (F32, 140, 8, 8200)])
def test_sort_of_many_rows_by_tokens(gen, dtype, tokens, top_k, cols):
    """32 MB of rows and more: odd rows apart, and entries that are no slot or a slot again."""
    wide = normal(gen, tokens, cols + 5).to(dtype)
    x = wide[:, 3:3 + cols]
    _, _, _, perm = routed(gen, tokens, 32, top_k)
    rows, place = ops.moe_sort(x, perm, top_k)
    assert rows.numel() * rows.element_size() >= 32 << 20
    assert same(rows, x[perm.long() // top_k])
    assert torch.equal(place[perm.long()].long(), torch.arange(tokens * top_k, device=x.device))
    bad = perm.clone()
    bad[5], bad[77], bad[-1] = -1, tokens * top_k, 2 ** 31 - 1
    got, _ = ops.moe_sort(x, bad, top_k)
    want = x[perm.long() // top_k]
    want[[5, 77, tokens * top_k - 1]] = 0
    assert same(got, want)


def test_combine_onto_the_residual_itself(gen):
    _, weights, _, perm = routed(gen, 31, 16, 4)
    rows, place = ops.moe_sort(normal(gen, 31, 300).bfloat16(), perm, 4)
    stream = normal(gen, 31, 300)
    want = ops.moe_combine(rows, weights, place, residual=stream, dtype=F32)
    assert ops.moe_combine(rows, weights, place, residual=stream, dtype=F32, out=stream) is stream
    assert torch.equal(stream, want)


def test_places_that_are_no_positions_contribute_nothing(gen):
    """A selection whose place is negative or past the rows: nothing is read or written for it."""
    tokens, top_k, cols = 6, 3, 40
    _, weights, _, perm = routed(gen, tokens, 5, top_k)
    rows, place = ops.moe_sort(normal(gen, tokens, cols), perm, top_k)
    drop = place.clone()
    drop[4], drop[9], drop[10], drop[11] = -1, tokens * top_k, 2 ** 31 - 1, -(2 ** 31)
    kept = weights.clone()
    kept.view(-1)[[4, 9, 10, 11]] = 0
    assert torch.equal(ops.moe_combine(rows, weights, drop), ops.moe_combine(rows, kept, place))
    assert not bool(ops.moe_combine(rows, weights, drop)[3].any())  # (none of its three is left)
    drows, dweights = ops.moe_combine_backward(rows[:tokens].clone(), rows, weights, drop)
    want, full = ops.moe_combine_backward(rows[:tokens].clone(), rows, weights, place)
    there = [i for i in range(tokens * top_k) if i not in (4, 9, 10, 11)]
    assert torch.equal(drows[place[there].long()], want[place[there].long()])
    full.view(-1)[[4, 9, 10, 11]] = 0
    assert torch.equal(dweights, full)
    # and a permutation's entry that is no slot: a row of zeros
    bad = perm.clone()
    bad[2], bad[7] = -5, tokens * top_k
    x = normal(gen, tokens, cols)
    got, _ = ops.moe_sort(x, bad, top_k)
    want = x[perm.long() // top_k]
    want[[2, 7]] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 32, 4), (3, 5, 5), (37, 32, 4),
                                                  (64, 64, 8), (65, 65, 1), (130, 128, 8),
                                                  (9, 256, 8), (1000, 255, 3)])
def test_route_gradient(gen, tokens, experts, top_k):
    logits = normal(gen, tokens, experts) * 3
    idx, weights, _, _ = ops.moe_route(logits, top_k)
    dweights = normal(gen, tokens, top_k)
    got = ops.moe_route_backward(idx, weights, dweights, experts)
    # the whole router in 64 bits: softmax over the experts, the chosen renormalised
    leaf = logits.double().requires_grad_(True)
    p = torch.softmax(leaf, 1).gather(1, idx.long())
    w = p / p.sum(1, keepdim=True).clamp(min=2.0 ** -14)
    w.backward(dweights.double())
    # the weights come as fp32 ones: each off by 2^-20 of itself (softmax and quotient in fp32)
    terms = weights.double() * dweights.double().abs()
    size = terms + weights.double() * terms.sum(1, keepdim=True)
    bound = torch.zeros_like(leaf).scatter(1, idx.long(), size * 2.0 ** -18)
    # (an unchosen expert's gradient cancels: what is left of it in 64 bits is the rounding, 2^-53
    # each, of fewer than 2^9 operations on numbers up to the largest |dw| over the sum of p)
    bound = bound + 2.0 ** -44 * (dweights.abs().amax(1) / p.sum(1)).unsqueeze(1).detach()
    within(got, leaf.grad, bound, F32, "dlogits")
    assert int((got != 0).sum()) <= tokens * top_k


def test_route_gradient_against_differences(gen):
    tokens, experts, top_k = 4, 12, 3
    logits = normal(gen, tokens, experts) * 2
    idx, weights, _, _ = ops.moe_route(logits, top_k)
    dweights = normal(gen, tokens, top_k)
    got = ops.moe_route_backward(idx, weights, dweights, experts).double()

    def loss(v):  # of the chosen experts, in 64 bits
        return float((torch.softmax(v.gather(1, idx.long()), 1) * dweights.double()).sum())

    step = 2.0 ** -16
    for t in range(tokens):
        for e in range(experts):
            up, down = logits.double(), logits.double()
            up[t, e] += step
            down[t, e] -= step
            # a central difference is off by step^2 / 6 of the third derivative, which is at most
            # 6 of the largest |dweights|; fp32 weights and sums by 2^-18 of it
            size = float(dweights.abs().max())
            assert abs((loss(up) - loss(down)) / (2 * step) - float(got[t, e])) <= (
                step * step + 2.0 ** -18 + 2.0 ** -34) * size


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_values_that_are_not_finite_stay_in_their_token(gen, bad):
    _, weights, _, perm = routed(gen, 9, 4, 2)
    rows, place = ops.moe_sort(normal(gen, 9, 24).bfloat16(), perm, 2)
    clean = ops.moe_combine(rows, weights, place, dtype=F32)
    rows[place[5].long(), 7] = bad  # of token 2
    y = ops.moe_combine(rows, weights, place, dtype=F32)
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[2, 7] = False
    assert torch.equal(y[keep], clean[keep]) and not bool(torch.isfinite(y[2, 7]))
    _, dweights = ops.moe_combine_backward(clean, rows, weights, place)
    assert int((~torch.isfinite(dweights)).sum()) == 1


def test_on_another_stream_and_captured(gen):
    """A graph of the whole chain, replayed with new inputs between eager work."""
    tokens, experts, top_k, cols = 40, 16, 4, 264
    logits, x = normal(gen, tokens, experts), normal(gen, tokens, cols).bfloat16()
    dy = normal(gen, tokens, cols).bfloat16()
    idx, weights, _, perm = ops.moe_route(logits, top_k)

    def chain():
        rows, place = ops.moe_sort(x, perm, top_k)
        y = ops.moe_combine(rows, weights, place, residual=x)
        drows, dweights = ops.moe_combine_backward(dy, rows, weights, place)
        return (rows, place, y, drows, dweights, ops.moe_sort_backward(drows, place, top_k),
                ops.moe_route_backward(idx, weights, dweights, experts))

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
    for seed in range(3):
        g = torch.Generator(device=x.device).manual_seed(seed)
        x.copy_(normal(g, tokens, cols))
        dy.copy_(normal(g, tokens, cols))
        eager = chain()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))


def test_far_rows(device):
    """Rows past 2^32 bytes."""
    tokens, top_k, cols = 32800, 8, 8192  # 262400 rows of 16 KB
    perm = torch.arange(tokens * top_k, dtype=torch.int32, device=device)
    x = torch.arange(tokens, device=device, dtype=torch.float32).fmod(251).bfloat16()
    x = x.unsqueeze(1).expand(tokens, cols).contiguous()
    rows, place = ops.moe_sort(x, perm, top_k)
    assert torch.equal(rows.view(tokens, top_k, cols)[-3:], x[-3:, None].expand(3, top_k, cols))
    weights = torch.full((tokens, top_k), 0.125, device=device)
    assert torch.equal(ops.moe_combine(rows, weights, place), x)
    drows, dweights = ops.moe_combine_backward(x, rows, weights, place)
    assert torch.equal(drows.view(tokens, top_k, cols)[-1], x[-1:].expand(top_k, cols) * 0.125)
    assert torch.equal(ops.moe_sort_backward(drows, place, top_k), x)
    want = (x.float() ** 2).sum(1, keepdim=True)
    assert torch.allclose(dweights, want.expand(tokens, top_k), rtol=2.0 ** -10)


def test_wrapper_refusals(gen):
    x = normal(gen, 4, 16).bfloat16()
    perm = torch.arange(8, dtype=torch.int32, device=x.device)
    weights = torch.ones(4, 2, device=x.device)
    rows, place = ops.moe_sort(x, perm, 2)
    refused = [
        lambda: ops.moe_sort(x, perm, 3), lambda: ops.moe_sort(x, perm.long(), 2),
        lambda: ops.moe_sort(x.double(), perm, 2), lambda: ops.moe_sort(x.t(), perm, 2),
        lambda: ops.moe_sort(x, perm.cpu(), 2), lambda: ops.moe_sort(x.cpu(), perm, 2),
        lambda: ops.moe_sort(x.float().requires_grad_(True), perm, 2),
        lambda: ops.moe_sort_backward(rows, place, 3),
        lambda: ops.moe_sort_backward(rows[:7], place, 2),
        lambda: ops.moe_sort_backward(rows, place, 0),
        lambda: ops.moe_combine(rows[:6], weights, place),
        lambda: ops.moe_combine(rows, weights.double(), place),
        lambda: ops.moe_combine(rows, weights.reshape(-1), place),
        lambda: ops.moe_combine(rows, weights, place, dtype=F16),
        lambda: ops.moe_combine(rows, weights, place, residual=x.float()),
        lambda: ops.moe_combine(rows, weights, place, residual=x[:3]),
        lambda: ops.moe_combine(rows, weights, place, out=x.float()),
        lambda: ops.moe_combine(rows, weights.requires_grad_(True), place),
        lambda: ops.moe_combine_backward(x.half(), rows, weights, place),
        lambda: ops.moe_combine_backward(x[:, :8], rows, weights, place),
        lambda: ops.moe_combine_backward(x[:1].expand(4, 16), rows, weights, place),
        lambda: ops.moe_route_backward(perm.reshape(4, 2).long(), weights.detach(),
                                       weights.detach(), 4),
        lambda: ops.moe_route_backward(perm.reshape(4, 2), weights.detach(),
                                       weights.detach()[:, :1], 4),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")
