"""The dense MXFP4 product with an epilogue and its backward pass in every kernel variant: strided
and unaligned rows, y in place of the residual, rows and blocks that are not finite, captures and
calls on two streams."""
import pytest
import torch

from kadan_amd import ops

import mxfp4_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16

# m, n, k: decode of 16 and 32 rows, staged and not, and the GEMM's tiles of 32, 64, 96 and 128 rows,
# in K slices too (test_mxfp4_linear_variants.py checks that they are all there)
LINEAR = [(1, 16, 64), (3, 8, 14336), (9, 2880, 2880), (17, 65, 256), (32, 8192, 672),
          (1, 8161, 32), (11, 8632, 768), (17, 8736, 32), (33, 70, 96), (33, 70, 1984),
          (77, 1030, 4128), (2733, 565, 32), (2758, 1, 12320), (2746, 1314, 32),
          (2853, 636, 9024), (2838, 2124, 1664), (101, 17043, 8736)]
# m, n, k of dy [m, n] and dx [m, k]
BACKWARD = [(17, 8, 32), (18, 1608, 32), (64, 4096, 544), (2926, 8, 576), (2940, 12624, 32),
            (1641, 8, 2336), (195, 4768, 9440), (777, 8, 7232), (910, 4152, 2272)]
SLICED = [(33, 70, 1984), (77, 1030, 4128), (2758, 1, 12320), (2853, 636, 9024),
          (101, 17043, 8736)]
SLICED_BACKWARD = [(18, 1608, 32), (64, 4096, 544), (2940, 12624, 32), (195, 4768, 9440),
                   (910, 4152, 2272)]


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(2024)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_strided_rows_and_the_residual_itself(gen, m, n, k, dtype, act):
    packed = ops.mxfp4_pack(*ref.matrix(gen, n, k))
    x = normal(gen, m, k + 24).bfloat16()[:, 16:16 + k]
    bias = normal(gen, n + 1)[1:]  # from any element on
    residual = normal(gen, m, n + 5).to(dtype)[:, 1:1 + n]
    around = normal(gen, m, n + 7).to(dtype)
    before, y = around.clone(), around[:, 3:3 + n]
    save = act is not None
    more = dict(bias=bias, activation=act, dtype=dtype, save=save)
    got = ops.mxfp4_linear(x, packed, n, residual=residual, out=y, **more)
    want = ops.mxfp4_linear(x.contiguous(), packed, n, bias=bias.clone(), activation=act,
                            residual=residual.contiguous(), dtype=dtype, save=save)
    if save:
        (got, kept), (want, saved) = got, want
        assert torch.equal(kept, saved)
    assert got is y and torch.equal(y, want)
    assert torch.equal(around[:, :3], before[:, :3])
    assert torch.equal(around[:, 3 + n:], before[:, 3 + n:])
    # onto the residual itself, side by side and some values apart
    for same in (residual.contiguous(), around[:, 3:3 + n].copy_(residual)):
        ops.mxfp4_linear(x, packed, n, residual=same, out=same, **more)
        assert torch.equal(same, want)
    assert torch.equal(around[:, :3], before[:, :3])
    assert torch.equal(around[:, 3 + n:], before[:, 3 + n:])


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("m,n,k", BACKWARD)
def test_strided_gradients(gen, m, n, k, act):
    turned = ops.mxfp4_pack(*ref.matrix(gen, n, k), transposed=True)
    dy = normal(gen, m, n + 24).bfloat16()[:, 8:8 + n]
    saved = normal(gen, m, n).bfloat16() if act else None
    around = normal(gen, m, k + 9).bfloat16()
    before = around.clone()
    dx, dpre = ops.mxfp4_linear_backward(dy, turned, k, saved=saved, activation=act,
                                         out=around[:, 5:5 + k])
    want, dwant = ops.mxfp4_linear_backward(dy.contiguous(), turned, k, saved=saved,
                                            activation=act)
    assert torch.equal(dx, want) and torch.equal(dpre, dwant)
    assert torch.equal(around[:, :5], before[:, :5])
    assert torch.equal(around[:, 5 + k:], before[:, 5 + k:])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_a_row_that_is_not_finite_stays_in_its_row(gen, m, n, k, bad):
    packed, x = ops.mxfp4_pack(*ref.matrix(gen, n, k)), normal(gen, m, k).bfloat16()
    bias, residual = normal(gen, n), normal(gen, m, n)
    more = dict(bias=bias, residual=residual)
    clean = ops.mxfp4_linear(x, packed, n, **more)
    for row in {0, m // 2, m - 1}:
        spoilt = x.clone()
        spoilt[row] = bad
        y = ops.mxfp4_linear(spoilt, packed, n, **more)
        keep = torch.arange(m, device=gen.device) != row
        assert torch.equal(y[keep], clean[keep])
        assert not bool(torch.isfinite(y[row]).all())


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("m,n,k", BACKWARD)
def test_a_gradient_that_is_not_finite_stays_in_its_row(gen, m, n, k, bad):
    turned = ops.mxfp4_pack(*ref.matrix(gen, n, k), transposed=True)
    dy = normal(gen, m, n).bfloat16()
    clean, _ = ops.mxfp4_linear_backward(dy, turned, k)
    for row in {0, m // 2, m - 1}:
        spoilt = dy.clone()
        spoilt[row] = bad
        dx, _ = ops.mxfp4_linear_backward(spoilt, turned, k)
        keep = torch.arange(m, device=gen.device) != row
        assert torch.equal(dx[keep], clean[keep])
        assert not bool(torch.isfinite(dx[row].float()).all())


@pytest.mark.parametrize("m,n,k", LINEAR)
def test_a_block_without_a_scale_reaches_its_own_results_only(gen, m, n, k):
    """Scale byte 255 (NaN) in one row of the matrix."""
    blocks, scales = ref.matrix(gen, n, k)
    x, row = normal(gen, m, k).bfloat16(), n // 2
    want = ops.mxfp4_linear(x, ops.mxfp4_pack(blocks, scales), n)
    keep = torch.arange(n, device=gen.device) != row
    for block in {0, k // 64, k // 32 - 1}:
        bad = scales.clone()
        bad[row, block] = 255
        got = ops.mxfp4_linear(x, ops.mxfp4_pack(blocks, bad), n)
        assert torch.equal(got[:, keep], want[:, keep]) and bool(torch.isnan(got[:, row]).all())


@pytest.mark.parametrize("m,n,k", SLICED + [(9, 2880, 2880), (2838, 2124, 1664)])
def test_captured(gen, m, n, k):
    """A graph of a product with everything, replayed with other inputs between eager work."""
    packed, bias = ops.mxfp4_pack(*ref.matrix(gen, n, k)), normal(gen, n)
    x, residual = normal(gen, m, k).bfloat16(), normal(gen, m, n)

    def call():
        return ops.mxfp4_linear(x, packed, n, bias=bias, activation="gelu", residual=residual,
                                save=True)

    replayed_as_eager(gen, call, x, residual)


@pytest.mark.parametrize("m,n,k", SLICED_BACKWARD + [(777, 8, 7232)])
def test_captured_gradients(gen, m, n, k):
    turned = ops.mxfp4_pack(*ref.matrix(gen, n, k), transposed=True)
    dy, saved = normal(gen, m, n).bfloat16(), normal(gen, m, n).bfloat16()

    def call():
        return ops.mxfp4_linear_backward(dy, turned, k, saved=saved, activation="silu")

    replayed_as_eager(gen, call, dy, saved)


def replayed_as_eager(gen, call, *inputs):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    for _ in range(3):
        for t in inputs:
            t.copy_(normal(gen, *t.shape))
        eager = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))


@pytest.mark.parametrize("m,n,k", SLICED)
def test_two_calls_at_once(gen, m, n, k):
    """Sliced calls on two streams share no partial sums."""
    packed = ops.mxfp4_pack(*ref.matrix(gen, n, k))
    at_once(lambda x, y: ops.mxfp4_linear(x, packed, n, residual=y, activation="silu"),
            [(normal(gen, m, k).bfloat16(), normal(gen, m, n)) for _ in range(2)])


@pytest.mark.parametrize("m,n,k", SLICED_BACKWARD)
def test_two_gradients_at_once(gen, m, n, k):
    turned = ops.mxfp4_pack(*ref.matrix(gen, n, k), transposed=True)
    at_once(lambda dy, saved: ops.mxfp4_linear_backward(dy, turned, k, saved=saved,
                                                        activation="gelu")[0],
            [(normal(gen, m, n).bfloat16(), normal(gen, m, n).bfloat16()) for _ in range(2)])


def at_once(call, batches):
    want = [call(*b) for b in batches]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in batches], [[] for _ in batches]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(call(*batches[i]))
    torch.cuda.synchronize()
    for i, runs in enumerate(got):
        assert all(torch.equal(run, want[i]) for run in runs)
