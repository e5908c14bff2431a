"""A matrix row without a scale (byte 255, NaN) where K leaves a wavefront group, or the last K slice's
second part, nothing to multiply: K of one to four chunks of 64 values, and slices that end early."""
import pytest
import torch

from kadan_amd import ops

import mxfp4_reference as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SHORT = [32, 64, 96, 128, 160, 192, 224, 256, 288, 544, 2080, 4128, 5920]


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(31)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def spoilt(scales, row, block):
    out = scales.clone()
    out[..., row, block] = 255
    return out


def only_there(got, want, columns):
    keep = torch.ones(want.shape[1], dtype=torch.bool, device=want.device)
    keep[columns] = False
    assert torch.equal(got[:, keep], want[:, keep])
    assert bool(torch.isnan(got[:, columns].float()).all())


@pytest.mark.parametrize("m", [5, 40, 300, 2100])
@pytest.mark.parametrize("k", SHORT)
def test_dense(gen, m, k):
    n = 160
    blocks, scales = ref.matrix(gen, n, k)
    x, other = normal(gen, m, k).bfloat16(), ops.mxfp4_pack(*ref.matrix(gen, n, k))
    good = ops.mxfp4_pack(blocks, scales)
    for row in (0, 37, 58, 159):  # (halves of 16 rows, and of 32)
        for block in {0, k // 64, k // 32 - 1}:
            bad = ops.mxfp4_pack(blocks, spoilt(scales, row, block))
            for f in (lambda w: ops.mxfp4_linear(x, w, n), lambda w: ops.mxfp4_product(x, w, n),
                      lambda w: ops.mxfp4_product_quantized(*ops.mxfp4_quantize(x), w, n),
                      lambda w: ops.mxfp4_gated(x, w, other, n),
                      lambda w: ops.mxfp4_gated(x, other, w, n)):
                only_there(f(bad), f(good), [row])


@pytest.mark.parametrize("m", [3, 40, 500])
@pytest.mark.parametrize("k", SHORT)
def test_experts(gen, m, k):
    experts, n = 3, 96
    blocks, scales = ref.matrix(gen, experts * n, k)
    blocks, scales = blocks.view(experts, n, -1), scales.view(experts, n, -1)
    other = ops.mxfp4_pack(blocks.flip(0).contiguous(), scales.flip(0).contiguous())
    good, x = ops.mxfp4_pack(blocks, scales), normal(gen, m, k).bfloat16()
    offsets = torch.tensor([0, m // 3, m // 3, m], dtype=torch.int32, device=gen.device)
    for row in (0, 37, 58, 95):
        for block in {0, k // 64, k // 32 - 1}:
            bad = ops.mxfp4_pack(blocks, spoilt(scales, row, block))
            for f in (lambda w: ops.mxfp4_linear(x, w, n, offsets=offsets),
                      lambda w: ops.mxfp4_experts_gated(x, offsets, w, other, n),
                      lambda w: ops.mxfp4_experts_gated(x, offsets, other, w, n)):
                only_there(f(bad), f(good), [row])


@pytest.mark.parametrize("m", [5, 40, 300])
@pytest.mark.parametrize("n", SHORT)
def test_gradients(gen, m, n):
    """Sums over the matrix's rows: a block's 32 columns."""
    k = 160
    blocks, scales = ref.matrix(gen, n, k)
    turned = [ops.mxfp4_pack(blocks, s, transposed=True)
              for s in (scales, spoilt(scales, n // 2, 3))]
    dy, saved = normal(gen, m, n).bfloat16(), normal(gen, m, 2 * n).bfloat16()
    columns = list(range(96, 128))
    want, got = (ops.mxfp4_linear_backward(dy, t, k)[0] for t in turned)
    only_there(got, want, columns)
    for pair in ((0, 1), (1, 0)):
        got = ops.mxfp4_gated_backward(dy, saved, turned[pair[0]], turned[pair[1]], k)[0]
        want = ops.mxfp4_gated_backward(dy, saved, turned[0], turned[0], k)[0]
        only_there(got, want, columns)
    offsets = torch.tensor([0, m // 3, m], dtype=torch.int32, device=gen.device)
    both = torch.stack([blocks, blocks])
    turned = [ops.mxfp4_pack(both, torch.stack([s, s]), transposed=True)
              for s in (scales, spoilt(scales, n // 2, 3))]
    want, got = (ops.mxfp4_linear_backward(dy, t, k, offsets=offsets)[0] for t in turned)
    only_there(got, want, columns)
    for pair in ((0, 1), (1, 0)):
        got = ops.mxfp4_experts_gated_backward(dy, offsets, saved, turned[pair[0]],
                                               turned[pair[1]], k)[0]
        want = ops.mxfp4_experts_gated_backward(dy, offsets, saved, turned[0], turned[0], k)[0]
        only_there(got, want, columns)
