"""The MXFP4 dense operators (kdq_mxfp4_quantize, _pack, _product, _product_quantized,
_gated, _gated_backward) against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import kadan_amd
from kadan_amd import ops

import mxfp4_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def gen(device):
    return torch.Generator(device=device).manual_seed(1234)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def rounded(y, bound, dtype):
    """The bound of y's fp32 sum once it is rounded to dtype."""
    return bound + (y.abs() + bound) * (ref.HALF_BF16 if dtype == BF16 else 0)


# ---------------------------------------------------------------- quantising

def quantize_cases():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((37, 96)).astype(np.float32)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.0, -0.0, 6.0, 4.0])
    t = np.zeros((30, 64), np.float32)
    for r in range(30):  # every tie, and its neighbours, at scales from the least to the largest
        v = np.resize(ties, 64).astype(np.float32)
        v[1::3] = np.nextafter(v[1::3], np.float32(0))
        v[2::3] = np.nextafter(v[2::3], np.float32(9))
        v[0] = v[32] = 7.0
        t[r] = np.ldexp(v * np.where(rng.random(64) < 0.5, -1, 1).astype(np.float32),
                        int(np.linspace(-126, 124, 30)[r]))
    small = np.zeros((4, 32), np.float32)
    small[0, 3] = 2.0 ** -149
    small[1] = np.float32(2.0 ** -128)
    small[2, 7] = -(2.0 ** -126)
    return {"normal": x, "ties": t, "small": small, "one row": x[:1, :32].copy()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", list(quantize_cases()))
def test_quantize_exact(device, name, dtype):
    x = torch.from_numpy(quantize_cases()[name]).to(dtype)
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    blocks, scales = ref.quantize(x.double().numpy())
    status = torch.zeros(1, dtype=torch.int32, device=device)
    got = ops.mxfp4_quantize(x.to(device), status)
    assert np.array_equal(got[1].cpu().numpy(), scales)
    assert np.array_equal(got[0].cpu().numpy(), blocks)
    assert int(status) == 0
    values = ops.mxfp4_dequantize(*got, *x.shape)
    assert torch.equal(values.double(), ref.decode(*got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_strided_rows(device, gen, dtype):
    wide = normal(gen, 19, 200).to(dtype)
    for x in (wide[:, 8:168], wide[:, :32], wide[2:3, 40:104], wide[::3, 64:192]):
        want = ref.quantize(x.double().cpu().numpy())
        got = ops.mxfp4_quantize(x)
        assert np.array_equal(got[0].cpu().numpy(), want[0])
        assert np.array_equal(got[1].cpu().numpy(), want[1])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quantize_marks_blocks_that_are_not_finite(device, gen, dtype, bad):
    x = normal(gen, 3, 96).to(dtype)
    clean = ops.mxfp4_quantize(x)
    x[1, 40] = bad
    status = torch.zeros(1, dtype=torch.int32, device=device)
    blocks, scales = ops.mxfp4_quantize(x, status)
    assert int(status) == 1 and int(scales[1, 1]) == 255
    assert not bool(blocks[1, 16:32].any())
    keep = torch.ones(3, 3, dtype=torch.bool, device=device)
    keep[1, 1] = False
    assert torch.equal(scales[keep], clean[1][keep])
    assert torch.equal(blocks.view(3, 3, 16)[keep], clean[0].view(3, 3, 16)[keep])


def test_packed_form_is_the_mixture_layers(device, gen):
    blocks, scales = ref.matrix(gen, 96, 320)
    assert torch.equal(ops.mxfp4_pack(blocks, scales),
                       ops.moe_mxfp4_pack(blocks, scales, 1, 96, 320))


# ---------------------------------------------------------------- products

SIZES = [  # m, n, k: each side of every tile, block, part and slice
    (1, 1, 32), (1, 16, 64), (2, 33, 96), (15, 17, 160), (16, 64, 128), (17, 65, 256),
    (31, 100, 288), (32, 48, 2048), (1, 300, 4096), (3, 96, 14336), (9, 2880, 2880),
    (33, 70, 96), (64, 256, 512), (65, 257, 544), (127, 130, 1056), (128, 512, 2048),
    (129, 63, 4128), (200, 600, 2880), (255, 31, 64), (257, 1030, 288), (300, 14336, 96),
    (77, 4096, 1440), (520, 5000, 608), (1025, 2100, 320),
]
# and sizes that reach every tile of the larger kernel (64, 96 and 128 rows; MXFP4 x: 256),
# with and without K slices, ragged in each direction
TILES = [(2933, 525, 544), (833, 4756, 544), (2083, 2856, 1632), (3219, 17, 12704),
         (65, 11414, 12448), (2167, 770, 10272)]
TILES_MXFP4 = [(2821, 531, 1312), (2049, 1867, 1312), (843, 9332, 1248), (2401, 2423, 1248),
               (399, 13133, 32), (75, 30, 3872)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", SIZES + TILES)
def test_product(device, gen, m, n, k, dtype):
    w = ref.matrix(gen, n, k)
    x = normal(gen, m, k).bfloat16()
    y = ops.mxfp4_product(x, ops.mxfp4_pack(*w), n, dtype)
    want, bound = ref.sum_bound(x.double(), ref.decode(*w))
    ref.within(y, want, rounded(want, bound, dtype), f"{m}x{n}x{k}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", SIZES + TILES_MXFP4)
def test_product_quantized(device, gen, m, n, k, dtype):
    w, x = ref.matrix(gen, n, k), ref.matrix(gen, m, k)
    y = ops.mxfp4_product_quantized(*x, ops.mxfp4_pack(*w), n, dtype)
    want, bound = ref.sum_bound(ref.decode(*x), ref.decode(*w))
    ref.within(y, want, rounded(want, bound, dtype), f"{m}x{n}x{k}")


# a few rows of matrices whose 32-row blocks fill the compute units, and MXFP4 rows too long for
# LDS: n on both sides of whole blocks, K on both sides of whole units
WIDE = [(1, 8161, 32), (7, 8224, 1056), (11, 8163, 768), (16, 9001, 4128), (17, 8335, 32),
        (32, 8192, 672)]
WIDE_MXFP4 = [(14, 1, 4672), (16, 130, 5408), (1, 8360, 32), (8, 8192, 4128), (9, 8531, 7264),
              (17, 8839, 32), (32, 8200, 672)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("quantized,m,n,k", [(False, *size) for size in WIDE] +
                         [(True, *size) for size in WIDE_MXFP4])
def test_few_rows_of_a_wide_matrix(device, gen, quantized, m, n, k, dtype):
    w = ref.matrix(gen, n, k)
    packed = ops.mxfp4_pack(*w)
    if quantized:
        x = ref.matrix(gen, m, k)
        y, x = ops.mxfp4_product_quantized(*x, packed, n, dtype), ref.decode(*x)
    else:
        x = normal(gen, m, k).bfloat16()
        y, x = ops.mxfp4_product(x, packed, n, dtype), x.double()
    want, bound = ref.sum_bound(x, ref.decode(*w))
    ref.within(y, want, rounded(want, bound, dtype), f"{m}x{n}x{k}")


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_product_scales_over_the_whole_range(device, gen, m):
    """Scale bytes from 0 to 252 in one matrix, against x whose size makes up for them."""
    n, k = 80, 32
    blocks, _ = ref.matrix(gen, n, k)
    byte = torch.linspace(0, 252, n, device=device).round().to(torch.uint8)
    x = normal(gen, m, k).bfloat16()
    packed = ops.mxfp4_pack(blocks, byte[:, None].contiguous())
    y = ops.mxfp4_product(x, packed, n)
    w = ref.decode(blocks, byte[:, None])
    want, bound = ref.sum_bound(x.double(), w)
    # (terms of 0.5 * 2^-127 times x may fall below fp32's normal numbers: each is then off by
    # at most 2^-149 or, flushed, 2^-126; sum_bound's TINY counts one of them)
    # (an fp32 sum may overflow on the way where the terms' magnitudes add up to 2^128)
    inside = x.double().abs() @ w.abs().T < 2.0 ** 127
    bound = bound + k * ref.TINY
    ref.within(torch.where(inside, y, torch.zeros_like(y)),
               torch.where(inside, want, torch.zeros_like(want)), bound)


@pytest.mark.parametrize("k", [32, 96, 288])
@pytest.mark.parametrize("m", [4, 20, 60, 70, 300])
def test_product_quantized_scales_over_the_whole_range(device, gen, m, k):
    """Every scale byte of the matrix against bytes of x from 0 to 254, in both kernels."""
    n = 255
    (blocks, _), (x_blocks, _) = ref.matrix(gen, n, k), ref.matrix(gen, m, k)
    byte = torch.arange(n, device=device).to(torch.uint8)[:, None].repeat(1, k // 32)
    x_byte = torch.randint(0, 253, (m, 1), generator=gen, device=device).to(torch.uint8)
    x_byte[:4, 0] = torch.tensor([0, 252, 253, 254]).to(torch.uint8)
    x_byte = x_byte.repeat(1, k // 32)
    packed = ops.mxfp4_pack(blocks, byte)
    y = ops.mxfp4_product_quantized(x_blocks, x_byte, packed, n)
    x, w = ref.decode(x_blocks, x_byte), ref.decode(blocks, byte)
    want, bound = ref.sum_bound(x, w)
    # (as for bf16 x: terms below fp32's normal numbers are off by at most 2^-126 each, and sums
    # may overflow on the way where the terms' magnitudes add up to 2^128)
    bound = bound + k * ref.TINY
    inside = x.abs() @ w.abs().T < 2.0 ** 127
    zero = torch.zeros_like(want)
    # bytes 253 and 254 take 4 and 6 past fp32: at their value, or infinite (NaN beside zeros)
    fits = (byte[:, 0] <= 252)[None] & (x_byte[:, 0] <= 252)[:, None]
    assert int((inside & fits).sum()) > m * n // 4 and bool((inside & ~fits).any())
    held = inside & (fits | torch.isfinite(y))
    ref.within(torch.where(held, y.double(), zero), torch.where(held, want, zero), bound)
    # 255 is NaN in its row of x
    x_byte[1] = 255
    y = ops.mxfp4_product_quantized(x_blocks, x_byte, packed, n)
    assert bool(torch.isnan(y[1]).all())


@pytest.mark.parametrize("m", [3, 40, 200])
def test_scales_past_252_are_infinite_weights_of_bf16_rows(device, gen, m):
    """4 and 6 are infinite from the byte on that takes them past fp32, the others their value."""
    n, k = 64, 32
    code = torch.arange(n, device=device) % 8  # a row's first code; the others are zero
    blocks = torch.zeros(n, k // 2, dtype=torch.uint8, device=device)
    blocks[:, 0] = code.to(torch.uint8)
    byte = (253 + torch.arange(n, device=device) // 32).to(torch.uint8)[:, None].contiguous()
    x = torch.zeros(m, k, dtype=BF16, device=device)
    x[:, 0] = 2.0 ** -126
    y = ops.mxfp4_product(x, ops.mxfp4_pack(blocks, byte), n).double()
    value = ref.decode(blocks, byte)[:, 0]  # past fp32 from 2^128 on
    want = torch.where(value >= 2.0 ** 128, float("inf"), value * 2.0 ** -126)
    assert torch.equal(y, want.expand(m, n))


@pytest.mark.parametrize("m", [4, 40, 200])
@pytest.mark.parametrize("quantized", [False, True])
def test_scale_255_is_nan_in_its_rows_only(device, gen, m, quantized):
    n, k = 70, 288
    blocks, scales = ref.matrix(gen, n, k)
    clean = ops.mxfp4_pack(blocks, scales)
    scales[37, 8] = 255
    bad = ops.mxfp4_pack(blocks, scales)
    if quantized:
        x = ref.matrix(gen, m, k)
        run = lambda p: ops.mxfp4_product_quantized(*x, p, n)
    else:
        x = normal(gen, m, k).bfloat16()
        run = lambda p: ops.mxfp4_product(x, p, n)
    a, b = run(clean), run(bad)
    assert bool(torch.isnan(b[:, 37]).all())
    keep = torch.arange(n, device=device) != 37
    assert torch.equal(a[:, keep], b[:, keep])


@pytest.mark.parametrize("k", [96, 128, 1056])
@pytest.mark.parametrize("m", [3, 40, 100, 300])
def test_values_that_are_not_finite_stay_in_their_row(device, gen, m, k):
    n = 130
    w = ref.matrix(gen, n, k)
    packed = ops.mxfp4_pack(*w)
    x = normal(gen, m, k).bfloat16()
    clean = ops.mxfp4_product(x, packed, n)
    x[1, k - 1] = float("inf")
    x[2, 0] = float("nan")
    y = ops.mxfp4_product(x, packed, n)
    other = (torch.arange(m, device=device) != 1) & (torch.arange(m, device=device) != 2)
    assert torch.equal(y[other], clean[other])
    assert bool(torch.isnan(y[2]).all())
    last = ref.decode(*w)[:, k - 1]
    want = torch.where(last == 0, float("nan"), last.sign() * float("inf"))
    assert torch.equal(torch.nan_to_num(y[1].double(), nan=7.0), torch.nan_to_num(want, nan=7.0))


def without_zeros(blocks):
    """The codes with 0 made 0.5, so that an infinity's products are infinite."""
    return blocks | ((blocks & 0x07) == 0).to(torch.uint8) | \
        (((blocks & 0x70) == 0).to(torch.uint8) << 4)


@pytest.mark.parametrize("k", [512, 640, 1440, 4352, 9600])
@pytest.mark.parametrize("m", [4, 12, 20, 32, 70])
def test_an_infinity_anywhere_in_a_row_is_the_rows_result(device, gen, m, k):
    """Wherever the wavefronts' shares of a row end, and a batch past such an end."""
    n = 48
    blocks, scales = ref.matrix(gen, n, k)
    blocks = without_zeros(blocks)
    packed, w = ops.mxfp4_pack(blocks, scales), ref.decode(blocks, scales)
    for first in range(0, k, 32 * m):
        at = (torch.arange(m, device=device) * 32 + first) % k
        x = normal(gen, m, k).bfloat16()
        x[torch.arange(m, device=device), at] = float("inf")
        want = w[:, at].t().sign() * float("inf")
        assert torch.equal(ops.mxfp4_product(x, packed, n).double(), want)


@pytest.mark.parametrize("n", [512, 640, 1440, 4352])
@pytest.mark.parametrize("m", [4, 12, 20, 32, 70])
def test_an_infinite_gradient_anywhere_in_a_row_is_the_rows_result(device, gen, m, n):
    k = 96
    blocks, scales = ref.matrix(gen, n, k)
    blocks = without_zeros(blocks)
    packed, w = ops.mxfp4_pack(blocks, scales, transposed=True), ref.decode(blocks, scales)
    kept = torch.ones(m, 2 * n, dtype=BF16, device=device)
    for first in range(0, n, 32 * m):
        at = (torch.arange(m, device=device) * 32 + first) % n
        dh = normal(gen, m, n).bfloat16()
        dh[torch.arange(m, device=device), at] = float("inf")
        dx, _ = ops.mxfp4_gated_backward(dh, kept, packed, packed, k)
        assert torch.equal(dx.double(), w[at].sign() * float("inf"))


@pytest.mark.parametrize("m,n,k", [(1, 40, 96), (20, 70, 64), (50, 100, 160), (140, 300, 96)])
def test_strided_rows_and_untouched_neighbours(device, gen, m, n, k):
    w = ref.matrix(gen, n, k)
    packed = ops.mxfp4_pack(*w)
    wide = normal(gen, m, k + 40).bfloat16()
    x = wide[:, 16:16 + k]
    plain = ops.mxfp4_product(x.contiguous(), packed, n)
    for dtype in (F32, BF16):
        frame = torch.full((m + 2, n + 5), 3.5, dtype=dtype, device=device)
        y = frame[1:m + 1, 2:n + 2]
        assert ops.mxfp4_product(x, packed, n, dtype, out=y) is y
        assert torch.equal(y, plain.to(dtype))
        frame[1:m + 1, 2:n + 2] = 3.5
        assert bool((frame == 3.5).all())


@pytest.mark.parametrize("m,k", [(5, 96), (50, 288), (300, 1056), (2100, 288)])
def test_a_block_that_is_not_finite_stays_in_its_row_of_x(device, gen, m, k):
    n = 1100
    packed = ops.mxfp4_pack(*ref.matrix(gen, n, k))
    x = normal(gen, m, k)
    clean = ops.mxfp4_product_quantized(*ops.mxfp4_quantize(x), packed, n)
    x[m - 2, k - 1] = float("inf")
    blocks, scales = ops.mxfp4_quantize(x)
    assert int(scales[m - 2, -1]) == 255
    y = ops.mxfp4_product_quantized(blocks, scales, packed, n)
    assert bool(torch.isnan(y[m - 2]).all())
    rest = torch.arange(m, device=device) != m - 2
    assert torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("k", [32, 96, 288, 2080])
@pytest.mark.parametrize("m", [3, 70, 260])
def test_scales_of_x_that_start_anywhere_in_a_dword(device, gen, m, k):
    """Rows of 1, 3, 9 and 65 scale bytes; the tensor's end followed by other data."""
    n = 96
    w, (blocks, scales) = ref.matrix(gen, n, k), ref.matrix(gen, m, k)
    held = torch.full((scales.numel() + 64,), 255, dtype=torch.uint8, device=device)
    held[:scales.numel()] = scales.reshape(-1)
    view = held[:scales.numel()].view(m, k // 32)
    y = ops.mxfp4_product_quantized(blocks, view, ops.mxfp4_pack(*w), n)
    want, bound = ref.sum_bound(ref.decode(blocks, scales), ref.decode(*w))
    ref.within(y, want, bound)


@pytest.mark.parametrize("m", [2, 40, 300])
def test_gated_strided_rows_and_untouched_neighbours(device, gen, m):
    n, k = 96, 160
    wg, wu = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    packed = [ops.mxfp4_pack(*w) for w in (wg, wu)]
    x = normal(gen, m, k + 8).bfloat16()[:, 8:]
    plain = ops.mxfp4_gated(x.contiguous(), *packed, n)
    frame = torch.full((m + 2, n + 3), 3.5, dtype=BF16, device=device)
    assert torch.equal(ops.mxfp4_gated(x, *packed, n, out=frame[1:m + 1, 1:n + 1]), plain)
    tg, tu = (ops.mxfp4_pack(*w, transposed=True) for w in (wg, wu))
    dh = normal(gen, m, n + 16).bfloat16()[:, 8:8 + n]
    kept = normal(gen, m, 2 * n).bfloat16()
    dx, dgu = ops.mxfp4_gated_backward(dh.contiguous(), kept, tg, tu, k)
    wide = torch.full((m + 2, k + 5), 3.5, dtype=BF16, device=device)
    got, again = ops.mxfp4_gated_backward(dh, kept, tg, tu, k, out=wide[1:m + 1, 2:k + 2])
    assert torch.equal(got, dx) and torch.equal(again, dgu)
    for f, inner in ((frame, (slice(1, m + 1), slice(1, n + 1))),
                     (wide, (slice(1, m + 1), slice(2, k + 2)))):
        f[inner] = 3.5
        assert bool((f == 3.5).all())


def test_the_same_matrix_twice_and_the_same_rows_twice(device, gen):
    """Gate and up of one tensor; rows that are each other's copies."""
    n, k = 64, 96
    w = ref.matrix(gen, n, k)
    p, t = ops.mxfp4_pack(*w), ops.mxfp4_pack(*w, transposed=True)
    for m in (4, 70):
        row = (normal(gen, 1, k) * 0.5).bfloat16()
        x = row.repeat(m, 1)
        h, saved = ops.mxfp4_gated(x, p, p, n, save="bf16")
        assert torch.equal(h, h[:1].expand_as(h)) and torch.equal(saved[:, :n], saved[:, n:])
        *_, (want, bound) = ref.gated(x.double(), ref.decode(*w), ref.decode(*w))
        ref.within(h, want, bound)
        dx, dgu = ops.mxfp4_gated_backward(h, saved, t, t, k)
        assert torch.equal(dx, dx[:1].expand_as(dx))


def test_rows_do_not_depend_on_their_number_within_a_kernel(device, gen):
    """The same rows in calls of the same kernel give the same bits, whatever lies behind."""
    n, k = 96, 512
    packed = ops.mxfp4_pack(*ref.matrix(gen, n, k))
    x = normal(gen, 128, k).bfloat16()
    whole = ops.mxfp4_product(x, packed, n)
    assert torch.equal(ops.mxfp4_product(x[:101], packed, n), whole[:101])
    assert torch.equal(ops.mxfp4_product(x, packed, n), whole)


def test_offsets_past_32_bits(device, gen):
    """Outputs and inputs of more than 4 GiB."""
    m, n, k = 36000, 65536, 32
    w = ref.matrix(gen, n, k)
    packed = ops.mxfp4_pack(*w)
    x = normal(gen, m, k).bfloat16()
    y = ops.mxfp4_product(x, packed, n, BF16)
    at = torch.tensor([0, 1, 17000, m - 2, m - 1], device=device)
    want, bound = ref.sum_bound(x[at].double(), ref.decode(*w))
    ref.within(y[at], want, rounded(want, bound, BF16))
    del y
    m, n, k = 530000, 16, 4096
    w = ref.matrix(gen, n, k)
    x = torch.empty(m, k, dtype=BF16, device=device).fill_(0.25)
    at = torch.tensor([0, 262143, 262145, 524288, m - 1], device=device)
    x[at] = normal(gen, 5, k).bfloat16()
    y = ops.mxfp4_product(x, ops.mxfp4_pack(*w), n)
    want, bound = ref.sum_bound(x[at].double(), ref.decode(*w))
    ref.within(y[at], want, bound)


# ---------------------------------------------------------------- the gated projection

GATED = [(1, 32, 32), (3, 64, 96), (16, 96, 2048), (17, 2880, 320), (32, 32, 4096), (33, 32, 64),
         (64, 160, 1056), (100, 96, 2880), (129, 2048, 96), (260, 1056, 512), (600, 288, 160)]


# sizes that reach every tile, with and without K slices: with nothing kept, and kept
GATED_TILES = [(67, 11456, 608), (133, 13344, 544), (2211, 1312, 1632), (3005, 32, 12512),
               (65, 11072, 7968), (397, 2496, 9120)]
GATED_TILES_KEPT = [(77, 10976, 544), (3291, 544, 544), (325, 9024, 1632), (2735, 32, 12448),
                    (73, 5440, 12640), (101, 9344, 8864)]
BACKWARD_TILES = [(129, 32, 13152), (289, 32, 13408), (385, 32, 13152), (35, 6208, 11744),
                  (65, 4864, 11360), (109, 4896, 8288)]


GATED_WIDE = [(1, 8224, 32), (7, 8192, 1056), (11, 8672, 768), (16, 8224, 4128), (17, 8256, 32),
              (32, 8192, 672)]


@pytest.mark.parametrize("m,n,k", GATED_WIDE)
def test_gated_few_rows_of_wide_matrices(device, gen, m, n, k):
    wg, wu = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    x = (normal(gen, m, k) * (8 / k ** 0.5)).bfloat16()
    h = ops.mxfp4_gated(x, ops.mxfp4_pack(*wg), ops.mxfp4_pack(*wu), n)
    *_, (want, bound) = ref.gated(x.double(), ref.decode(*wg), ref.decode(*wu))
    ref.within(h, want, bound, "h")


def check_q8(saved, exact, error):
    """Codes and scales against the pre-activations they stand for: a value is off by half a
    code of its block's scale, which is off by the largest error of the block."""
    q, d = saved
    v = exact.reshape(exact.shape[0], -1, 32)
    e = error.reshape(v.shape).amax(-1, keepdim=True)
    top = v.abs().amax(-1, keepdim=True)
    scale = (top + e) / 127
    ref.within(d.double().unsqueeze(-1), top / 127, e / 127 + top / 127 * 2.0 ** -22 + ref.TINY)
    got = q.double().reshape(v.shape) * d.double().unsqueeze(-1)
    ref.within(got, v, scale * (0.5 + 2.0 ** -15) + e + ref.TINY)
    assert int(q.to(torch.int32).abs().max()) <= 127


@pytest.mark.parametrize("m,n,k,save", [
    (*size, save) for save in (None, "bf16", "q8")
    for size in GATED + (GATED_TILES_KEPT if save else GATED_TILES)])
def test_gated(device, gen, m, n, k, save):
    wg, wu = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    x = (normal(gen, m, k) * (8 / k ** 0.5)).bfloat16()
    got = ops.mxfp4_gated(x, ops.mxfp4_pack(*wg), ops.mxfp4_pack(*wu), n, save=save)
    h, saved = got if save else (got, None)
    (g, dg), (u, du), (want, bound) = ref.gated(x.double(), ref.decode(*wg), ref.decode(*wu))
    ref.within(h, want, bound, "h")
    exact, error = torch.cat([g, u], 1), torch.cat([dg, du], 1)
    if save == "bf16":
        ref.within(saved, exact, rounded(exact, error, BF16), "kept")
    elif save == "q8":
        check_q8(saved, exact, error)


def test_gated_far_gates(device, gen):
    """Gates whose exponential overflows, underflows, or is not finite."""
    n, k = 32, 32
    one = (torch.full((n, k // 2), 0, dtype=torch.uint8, device=device),
           torch.full((n, 1), 127, dtype=torch.uint8, device=device))
    one[0][:, 0] = 0x02  # the first value 1, the others 0: g = u = x[0]
    packed = ops.mxfp4_pack(*one)
    first = [-1e38, -500.0, -100.0, -89.0, -87.0, -30.0, 0.0, -0.0, 30.0, 89.0, 500.0, 1e19,
             float("inf"), float("nan")]
    for m in (len(first), 40):
        x = torch.zeros(m, k, dtype=BF16, device=device)
        x[:len(first), 0] = torch.tensor(first).to(BF16).to(device)
        h = ops.mxfp4_gated(x, packed, packed, n)[:len(first), 0].double().cpu()
        v = x[:len(first), 0].double().cpu()
        for i, t in enumerate(v.tolist()):
            if i == 12:    # inf * sigmoid(inf) * inf
                assert h[i] == float("inf")
            elif i == 13:
                assert np.isnan(float(h[i]))
            elif i == 0:   # -1e38 * 0 * -1e38
                assert h[i] == 0
            else:
                want = t * t / (1 + np.exp(-t))
                assert abs(float(h[i]) - want) <= abs(want) * (ref.HALF_BF16 + 2.0 ** -15) + 1e-30


def test_gated_q8_blocks_that_cannot_be_kept(device, gen):
    """A zero block, one too small for its scale, and one that is not finite."""
    n, k, m = 96, 32, 40
    blocks = torch.zeros(n, k // 2, dtype=torch.uint8, device=device)
    blocks[:, 0] = 0x02
    scales = torch.full((n, 1), 127, dtype=torch.uint8, device=device)
    packed = ops.mxfp4_pack(blocks, scales)
    x = torch.zeros(m, k, dtype=BF16, device=device)
    x[1, 0], x[2, 0], x[3, 0] = 2.0 ** -122, float("inf"), 2.0 ** -119
    _, (q, d) = ops.mxfp4_gated(x, packed, packed, n, save="q8")
    assert not bool(d[:2].any()) and not bool(q[:3].any())
    assert bool(torch.isnan(d[2]).all())
    assert bool((q[3] == 127).all()) and bool((d[3] > 0).all())
    kept = (q, d)
    pt = ops.mxfp4_pack(blocks, scales, transposed=True)
    dx, dgu = ops.mxfp4_gated_backward(torch.ones(m, n, dtype=BF16, device=device), kept, pt, pt,
                                       k)
    assert bool(torch.isnan(dgu[2]).all()) and bool(torch.isnan(dx[2]).all())
    rest = torch.arange(m, device=device) != 2
    assert bool(torch.isfinite(dx[rest]).all())


# ---------------------------------------------------------------- its backward pass

@pytest.mark.parametrize("save", ["bf16", "q8"])
@pytest.mark.parametrize("m,n,k", GATED + BACKWARD_TILES + [(40, 2048, 2080), (7, 4128, 96),
                                                          (200, 320, 4992)])
def test_gated_backward(device, gen, m, n, k, save):
    wg, wu = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    tg, tu = (ops.mxfp4_pack(*w, transposed=True) for w in (wg, wu))
    dh = normal(gen, m, n).bfloat16()
    if save == "bf16":
        saved = (3 * normal(gen, m, 2 * n)).bfloat16()
        kept = saved.double()
    else:
        q = torch.randint(-127, 128, (m, 2 * n), generator=gen, device=device).to(torch.int8)
        d = torch.rand(m, n // 16, generator=gen, device=device) * 0.1
        saved = (q, d)
        kept = q.double() * d.double().repeat_interleave(32, 1)
        kept = kept.float().double()  # code times scale is rounded to fp32
    dx, dgu = ops.mxfp4_gated_backward(dh, saved, tg, tu, k)
    want, bound = ref.gate_gradients(dh.double(), kept[:, :n], kept[:, n:])
    ref.within(dgu, want, bound, "dgu")
    both = torch.cat([ref.decode(*wg), ref.decode(*wu)]).T.contiguous()
    y, e = ref.sum_bound(dgu.double(), both)  # of the gradients as they were rounded
    ref.within(dx, y, rounded(y, e, BF16), "dx of dgu")
    full = want @ both.T
    ref.within(dx, full, bound @ both.abs().T + rounded(y, e, BF16) + 1e-30, "dx")


@pytest.mark.parametrize("m,n,k", BACKWARD_TILES + [(64, 768, 2048)])
def test_gated_backward_reads_nothing_of_the_kernel_before(device, gen, m, n, k):
    """Calls right behind a product whose rows are NaN, which leaves NaN in every compute unit's
    LDS, and behind nothing, with dgu out of the caches: the same bits."""
    t, t2 = (ops.mxfp4_pack(*ref.matrix(gen, n, k), transposed=True) for _ in range(2))
    dh, kept = normal(gen, m, n).bfloat16(), normal(gen, m, 2 * n).bfloat16()
    want = ops.mxfp4_gated_backward(dh, kept, t, t2, k)
    packed = ops.mxfp4_pack(*ref.matrix(gen, 8192, 1024))
    bad = torch.full((1024, 1024), float("nan"), dtype=BF16, device=device)
    other = torch.empty(1 << 29, dtype=torch.uint8, device=device)
    for i in range(12):
        if i % 2:
            other.fill_(i)
        ops.mxfp4_product(bad, packed, 8192, BF16)
        got = ops.mxfp4_gated_backward(dh, kept, t, t2, k)
        assert bool(torch.isfinite(got[0]).all())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gated_backward_against_differences(device, gen):
    """The loss sum(dh * h(x)) in 64 bits along random directions, by central differences."""
    m, n, k = 12, 64, 96
    wg, wu = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    dg, du = ref.decode(*wg), ref.decode(*wu)
    x = (normal(gen, m, k) * (8 / k ** 0.5)).bfloat16()
    dh = normal(gen, m, n).bfloat16()
    _, saved = ops.mxfp4_gated(x, ops.mxfp4_pack(*wg), ops.mxfp4_pack(*wu), n, save="bf16")
    dx, _ = ops.mxfp4_gated_backward(dh, saved, ops.mxfp4_pack(*wg, transposed=True),
                                     ops.mxfp4_pack(*wu, transposed=True), k)

    def loss(at):
        g, u = at @ dg.T, at @ du.T
        return (dh.double() * (g * torch.sigmoid(g) * u)).sum(1)

    # how far dx may be: dgu's bound at the kept values, what keeping them in bf16 moves dgu
    # (its derivatives in g and u are at most |dh| (|u| / 2 + 1.1) and |dh| 1.1 per unit), the
    # sums and the last rounding
    g, u = x.double() @ dg.T, x.double() @ du.T
    _, bound = ref.gate_gradients(dh.double(), g, u)
    eg, eu = (v.abs() * ref.HALF_BF16 + 1e-4 for v in (g, u))
    size = dh.double().abs()
    move = torch.cat([size * (0.5 * u.abs() * eg + 1.1 * eu), size * 1.1 * eg], 1)
    both = torch.cat([dg, du])
    slack = 1.05 * ((bound + move) @ both.abs()) + dx.double().abs() * ref.HALF_BF16 + 1e-3
    step = 1e-5
    for _ in range(5):
        v = normal(gen, m, k).double()
        numeric = (loss(x.double() + step * v) - loss(x.double() - step * v)) / (2 * step)
        assert bool(((dx.double() * v).sum(1) - numeric).abs().le((slack * v.abs()).sum(1)).all())


# ---------------------------------------------------------------- together

def test_a_layer_quantised_served_and_trained(device, gen):
    """A float checkpoint's block quantised, a decode token and a prompt through gate/up and
    down (bf16 and MXFP4 activations), and an adapter's gradient through the frozen base."""
    hidden, inter, rank = 288, 352, 4
    gate, up = (ops.mxfp4_quantize(normal(gen, inter, hidden) / hidden ** 0.5) for _ in range(2))
    down = ops.mxfp4_quantize(normal(gen, hidden, inter) / inter ** 0.5)
    pg, pu, pd = (ops.mxfp4_pack(*w) for w in (gate, up, down))
    tg, tu = (ops.mxfp4_pack(*w, transposed=True) for w in (gate, up))
    wg, wu, wd = (ref.decode(*w) for w in (gate, up, down))
    for m in (1, 150):
        x = normal(gen, m, hidden).bfloat16()
        h, saved = ops.mxfp4_gated(x, pg, pu, inter, save="q8")
        assert torch.equal(h, ops.mxfp4_gated(x, pg, pu, inter, save="bf16")[0])
        *_, (want, bound) = ref.gated(x.double(), wg, wu)
        ref.within(h, want, bound, "h")
        y = ops.mxfp4_product(h, pd, hidden)
        exact, e = ref.sum_bound(h.double(), wd)
        ref.within(y, exact, e, "down")
        hq = ops.mxfp4_quantize(h)
        yq = ops.mxfp4_product_quantized(*hq, pd, hidden)
        exact, e = ref.sum_bound(ref.decode(*hq), wd)
        ref.within(yq, exact, e, "down of quantised rows")
        # an adapter on the gate: g = x Wg^T + (x A) B; its gradients from dgu and x
        dh = ops.mxfp4_product(y.bfloat16(), ops.mxfp4_pack(*ops.mxfp4_quantize(wd.T.float()
                                                            .contiguous())), inter, BF16)
        dx, dgu = ops.mxfp4_gated_backward(dh, saved, tg, tu, hidden)
        q, d = saved
        kept = (q.float() * d.repeat_interleave(32, 1)).double()
        wantg, boundg = ref.gate_gradients(dh.double(), kept[:, :inter], kept[:, inter:])
        ref.within(dgu, wantg, boundg, "dgu")
        a = normal(gen, hidden, rank).bfloat16()
        db = (x @ a).float().T @ dgu[:, :inter].float()
        assert db.shape == (rank, inter) and bool(torch.isfinite(db).all())
        exact, e = ref.sum_bound(dgu.double(), torch.cat([wg, wu]).T.contiguous())
        ref.within(dx, exact, rounded(exact, e, BF16), "dx")


def passes(gen, m, n, k):
    """Every operator at one size, as callables over tensors made once."""
    w, w2 = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    x, dh = normal(gen, m, k).bfloat16(), normal(gen, m, n).bfloat16()
    xq = ops.mxfp4_quantize(x)
    p, p2 = ops.mxfp4_pack(*w), ops.mxfp4_pack(*w2)
    t, t2 = (ops.mxfp4_pack(*v, transposed=True) for v in (w, w2))
    kept = normal(gen, m, 2 * n).bfloat16()
    return x, [lambda: ops.mxfp4_quantize(x),
               lambda: (ops.mxfp4_product(x, p, n),),
               lambda: (ops.mxfp4_product_quantized(*xq, p, n),),
               lambda: (ops.mxfp4_gated(x, p, p2, n),),
               lambda: (lambda h, s: (h, *s))(*ops.mxfp4_gated(x, p, p2, n, save="q8")),
               lambda: ops.mxfp4_gated_backward(dh, kept, t, t2, k)]


@pytest.mark.parametrize("m,n,k", [(2, 64, 256), (70, 64, 2048), (300, 2880, 288)])
def test_captured_and_replayed(device, gen, m, n, k):
    """Each operator captured once and replayed with new inputs, eager calls (one of a larger
    size, so of a larger workspace) between the replays; two graphs alive together."""
    x, fs = passes(gen, m, n, k)
    _, larger = passes(gen, 300, 96, 2112)
    torch.cuda.synchronize()
    graphs = []
    for f in fs:  # (captured before any eager call)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    for _ in range(4):
        x.copy_(normal(gen, m, k).bfloat16())
        for graph, _ in graphs:
            graph.replay()
        for f in larger:
            f()
        torch.cuda.synchronize()
        for f, (_, out) in zip(fs, graphs):
            for got, want in zip(out, f()):
                assert torch.equal(got, want)


def test_calls_on_two_streams(device, gen):
    """Calls that overlap on two streams share nothing."""
    _, fs = passes(gen, 70, 64, 4096)
    _, others = passes(gen, 65, 96, 2048)
    want = [f() for f in fs + others]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, calls in zip(streams, (fs, others)):
            with torch.cuda.stream(s):
                got += [f() for f in calls]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for p, q in zip(a, b):
                assert torch.equal(p, q)


def test_refusals_on_the_device(device, gen):
    w = ref.matrix(gen, 64, 128)
    p = ops.mxfp4_pack(*w)
    t = ops.mxfp4_pack(*w, transposed=True)
    x = normal(gen, 40, 128).bfloat16()
    kept = torch.zeros(40, 128, dtype=BF16, device=device)
    with pytest.raises(kadan_amd.KdqError, match="kdq_alias"):
        ops.mxfp4_product(x, p, 64, BF16, out=x[:, :64])
    with pytest.raises(ValueError):
        ops.mxfp4_product(x, p, 32)              # another matrix's size
    with pytest.raises(ValueError):
        ops.mxfp4_product(x, p, 0)
    with pytest.raises(ValueError):
        ops.mxfp4_product(x[:, :64], p, 64)
    with pytest.raises(ValueError):
        ops.mxfp4_product(x.t(), p, 64)          # columns side by side
    with pytest.raises(ValueError):
        ops.mxfp4_product(x.float(), p, 64)
    with pytest.raises(ValueError):
        ops.mxfp4_product(x, p, 64, torch.int8)
    with pytest.raises(kadan_amd.KdqUnsupported):
        ops.mxfp4_product(x, p, 64, torch.float16)
    with pytest.raises(kadan_amd.KdqError, match="kdq_argument"):
        ops.mxfp4_product(x[:0], p, 64)
    with pytest.raises(kadan_amd.KdqError, match="kdq_alignment"):
        ops.mxfp4_product(torch.empty(40 * 128 + 8, dtype=BF16, device=device)[1:40 * 128 + 1]
                          .view(40, 128), p, 64)
    with pytest.raises(ValueError):
        ops.mxfp4_product(normal(gen, 5, 132).bfloat16()[:, :128], p, 64)  # rows 132 apart
    with pytest.raises(ValueError):
        ops.mxfp4_product(x[:1].expand(40, 128), p, 64)
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(normal(gen, 4, 40))
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(torch.zeros(4, 32, dtype=torch.int32, device=device))
    with pytest.raises(ValueError):
        ops.mxfp4_gated(x, p, p, 64, save="q4")
    with pytest.raises(ValueError):
        ops.mxfp4_gated(x, p, t[:-128], 64)
    with pytest.raises(ValueError):
        ops.mxfp4_gated_backward(x[:, :64], kept[:39], t, t, 128)
    with pytest.raises(ValueError):
        ops.mxfp4_gated_backward(x[:, :64], (kept.to(torch.int8), kept[:, :4]), t, t, 128)
    with pytest.raises(ValueError):
        ops.mxfp4_product_quantized(w[0], w[1][:, :3].contiguous(), p, 64)
    torch.cuda.synchronize()


def test_the_other_packed_form_is_refused(device, gen):
    n, k = 64, 256  # 8704 bytes in both
    w = ref.matrix(gen, n, k)
    p, t = ops.mxfp4_pack(*w), ops.mxfp4_pack(*w, transposed=True)
    assert p.numel() == t.numel() and t.shape == (4, 2176)
    x, dh = normal(gen, 3, k).bfloat16(), normal(gen, 3, n).bfloat16()
    kept = normal(gen, 3, 2 * n).bfloat16()
    for call in (lambda: ops.mxfp4_product(x, t, n),
                 lambda: ops.mxfp4_product_quantized(*ops.mxfp4_quantize(x), t, n),
                 lambda: ops.mxfp4_gated(x, t, p, n), lambda: ops.mxfp4_gated(x, p, t, n),
                 lambda: ops.mxfp4_gated_backward(dh, kept, p, t, k),
                 lambda: ops.mxfp4_gated_backward(dh, kept, t, p, k),
                 lambda: ops.mxfp4_gated_backward(dh, kept, t, t.view(-1), k)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


class Gated(torch.autograd.Function):
    """The gated projection over frozen weights as a user's program records it."""

    @staticmethod
    def forward(ctx, x, gate, up, gate_t, up_t, n):
        h, saved = ops.mxfp4_gated(x, gate, up, n, save="bf16")
        ctx.save_for_backward(saved, gate_t, up_t)
        ctx.k = x.shape[1]
        return h

    @staticmethod
    def backward(ctx, dh):
        dx, _ = ops.mxfp4_gated_backward(dh.contiguous(), *ctx.saved_tensors, ctx.k)
        return dx, None, None, None, None, None


def test_recorded_by_a_function_and_refused_without_one(device, gen):
    m, n, k = 40, 96, 128
    wg, wu = ref.matrix(gen, n, k), ref.matrix(gen, n, k)
    packed = [ops.mxfp4_pack(*w) for w in (wg, wu)]
    transposed = [ops.mxfp4_pack(*w, transposed=True) for w in (wg, wu)]
    x = normal(gen, m, k).bfloat16().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        ops.mxfp4_gated(x, *packed, n)
    with torch.no_grad():
        plain, saved = ops.mxfp4_gated(x, *packed, n, save="bf16")
    h = Gated.apply(x, *packed, *transposed, n)
    assert torch.equal(h, plain)
    dh = normal(gen, m, n).bfloat16()
    h.backward(dh)
    assert torch.equal(x.grad, ops.mxfp4_gated_backward(dh, saved, *transposed, k)[0])
    x.grad = None
    Gated.apply(x, *packed, *transposed, n).sum().backward()  # (a gradient of rows that overlap)
    ones = torch.ones(m, n, dtype=BF16, device=device)
    assert torch.equal(x.grad, ops.mxfp4_gated_backward(ones, saved, *transposed, k)[0])
