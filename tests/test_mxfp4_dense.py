"""CPU checks of the MXFP4 dense operators: sizes, workspaces and refusals of the C ABI
before any launch, and the reference that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import kadan_amd
from kadan_amd import ops

import mxfp4_reference as ref

W, X, Y, Z, V = (0x10000000 * i for i in range(1, 6))  # never dereferenced
K256 = dict(argument=1, shape=2, unsupported=3, alias=4, scratch=6, alignment=7)


def test_packed_sizes():
    lib = kadan_amd.lib()
    size, transposed = lib.kdq_mxfp4_packed_bytes, lib.kdq_mxfp4_packed_transposed_bytes
    assert size(32, 64) == 1024 + 256 == lib.kdq_moe_mxfp4_packed_bytes(1, 32, 64)
    assert size(2880, 2880) == lib.kdq_moe_mxfp4_packed_bytes(1, 2880, 2880)
    assert size(1, 32) == 1024 + 256
    assert size(33, 288) == 2 * 5 * 1024 + 2 * 2 * 256
    assert transposed(64, 64) == 2048 + 128
    assert transposed(65, 96) == 2 * 2 * (2048 + 128)
    for f in (size, transposed):
        assert f(0, 64) == f(64, 0) == f(64, 48) == f(64, (1 << 20) + 32) == 0


def test_pack_refusals():
    lib = kadan_amd.lib()
    for f in (lib.kdq_mxfp4_pack, lib.kdq_mxfp4_pack_transposed):
        assert f(None, X, 32, 64, Y, None) == 1
        assert f(W, X, 0, 64, Y, None) == 1
        assert f(W, X, 32, 48, Y, None) == 2
        assert f(W + 8, X, 32, 64, Y, None) == 7
        assert f(W, X, 32, 64, Y + 8, None) == 7
        assert f(W, X, 32, 64, W + 512, None) == 4
        assert f(W, Y + 512, 32, 64, Y, None) == 4


def test_quantize_refusals():
    f = kadan_amd.lib().kdq_mxfp4_quantize
    assert f(0, None, 64, 2, 64, Y, Z, None, None) == 1
    assert f(0, X, 64, 0, 64, Y, Z, None, None) == 1
    assert f(8, X, 64, 2, 64, Y, Z, None, None) == 3
    assert f(0, X, 64, 2, 48, Y, Z, None, None) == 2
    assert f(0, X, 63, 2, 64, Y, Z, None, None) == 2
    assert f(0, X, 68, 2, 64, Y, Z, None, None) == 2
    assert f(0, X, 1 << 62, 1 << 10, 64, Y, Z, None, None) == 2
    assert f(0, X + 8, 64, 2, 64, Y, Z, None, None) == 7
    assert f(0, X, 64, 2, 64, Y + 2, Z, None, None) == 7
    assert f(0, X, 64, 2, 64, X + 256, Z, None, None) == 4
    assert f(0, X, 64, 2, 64, Y, X + 64, None, None) == 4
    assert f(0, X, 64, 2, 64, Y, Y + 16, None, None) == 4


def test_product_refusals():
    lib = kadan_amd.lib()
    f = lib.kdq_mxfp4_product
    good = dict(x=X, xs=64, m=2, w=W, n=40, k=64, t=0, y=Y, ys=40, ws=None, wb=0)

    def call(**change):
        a = {**good, **change}
        return f(a["x"], a["xs"], a["m"], a["w"], a["n"], a["k"], a["t"], a["y"], a["ys"],
                 a["ws"], a["wb"], None)

    for name in ("x", "w", "y"):
        assert call(**{name: None}) == 1
    for name in ("m", "n", "k"):
        assert call(**{name: 0}) == 1
    assert call(k=48, xs=48) == 2 and call(xs=63) == 2 and call(xs=68) == 2
    assert call(xs=(1 << 21) + 8) == 2 and call(m=(1 << 20) + 1) == 2
    assert call(n=(1 << 24) + 1, ys=1 << 25) == 2 and call(ys=39) == 2
    assert call(t=1) == 3 and call(t=8) == 3
    assert call(x=X + 8) == 7 and call(w=W + 8) == 7 and call(y=Y + 2) == 7
    assert call(t=30, y=Y + 1) == 7
    assert call(y=X + 128) == 4 and call(y=W + 64) == 4
    # K slices need their workspace, aligned and apart from the output
    need = lib.kdq_mxfp4_product_workspace(77, 4096, 14336, 0)
    assert need > 0
    big = dict(m=77, n=4096, k=14336, xs=14336, ys=4096, y=Y * 4, x=X * 4, w=W * 8)
    assert call(**big) == 6 and call(**big, ws=Z * 8, wb=need - 1) == 6
    assert call(**big, ws=Z * 8 + 8, wb=need) == 7
    assert call(**big, ws=Y * 4 + 256, wb=need) == 4


def test_product_quantized_refusals():
    f = kadan_amd.lib().kdq_mxfp4_product_quantized
    ok = [X, Z, 2, W, 40, 64, 0, Y, 40, None, 0, None]

    def call(at, value):
        return f(*[value if i == at else v for i, v in enumerate(ok)])

    for at in (0, 1, 3, 7):
        assert call(at, None) == 1
    for at in (2, 4, 5):
        assert call(at, 0) == 1
    assert call(5, 48) == 2 and call(8, 39) == 2 and call(6, 1) == 3
    assert call(0, X + 4) == 7 and call(3, W + 4) == 7 and call(7, Y + 2) == 7
    assert call(7, X) == 4 and call(7, Z) == 4 and call(7, W) == 4


def test_gated_refusals():
    f = kadan_amd.lib().kdq_mxfp4_gated
    ok = [X, 64, 2, W, W + 65536, 32, 64, Y, 32, None, None, None, None, 0, None]

    def call(**change):
        return f(*[change.get(f"a{i}", v) for i, v in enumerate(ok)])

    for at in (0, 3, 4, 7):
        assert call(**{f"a{at}": None}) == 1
    for at in (2, 5, 6):
        assert call(**{f"a{at}": 0}) == 1
    assert call(a10=Z) == 1 and call(a11=Z) == 1 and call(a9=Z, a10=V, a11=V + 4096) == 1
    assert call(a5=40, a8=40) == 2 and call(a6=48) == 2 and call(a1=60) == 2 and call(a8=31) == 2
    assert call(a0=X + 8) == 7 and call(a4=W + 65544) == 7 and call(a9=Z + 8) == 7
    assert call(a10=Z + 4, a11=V) == 7
    assert call(a7=X + 32) == 4 and call(a7=W + 64) == 4 and call(a9=Y + 16) == 4
    assert call(a10=Z, a11=Z + 64) == 4 and call(a10=W, a11=V) == 4


def test_gated_backward_refusals():
    f = kadan_amd.lib().kdq_mxfp4_gated_backward
    ok = [X, 32, 2, Z, None, None, W, W + 65536, 32, 64, Y, Y + 65536, 64, None, 0, None]

    def call(**change):
        return f(*[change.get(f"a{i}", v) for i, v in enumerate(ok)])

    for at in (0, 3, 6, 7, 10, 11):
        assert call(**{f"a{at}": None}) == 1
    for at in (2, 8, 9):
        assert call(**{f"a{at}": 0}) == 1
    assert call(a4=V) == 1 and call(a3=None, a4=V) == 1 and call(a5=V) == 1
    assert call(a8=40, a1=40) == 2 and call(a9=48) == 2 and call(a1=36) == 2 and call(a12=63) == 2
    assert call(a0=X + 2) == 7 and call(a3=Z + 8) == 7 and call(a10=Y + 8) == 7
    assert call(a11=Y + 65537) == 7
    assert call(a10=X) == 4 and call(a10=Z) == 4 and call(a11=Y) == 4 and call(a11=W) == 4


def test_sizes_without_a_workspace_and_with_one():
    lib = kadan_amd.lib()
    assert lib.kdq_mxfp4_product_workspace(1, 14336, 4096, 0) == 0
    assert lib.kdq_mxfp4_product_workspace(0, 14336, 4096, 0) == 0
    assert lib.kdq_mxfp4_product_workspace(8, 64, 48, 0) == 0
    assert lib.kdq_mxfp4_gated_workspace(1, 14336, 4096, 0) == 0
    # a slice's results are 8 KB per pair of 32 x 32 tiles
    for got in (lib.kdq_mxfp4_product_workspace(77, 4096, 14336, 0),
                lib.kdq_mxfp4_gated_workspace(1, 64, 4096, 1),
                lib.kdq_mxfp4_gated_backward_workspace(40, 4096, 64)):
        assert got % 8192 == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_wrappers_refuse_host_tensors(dtype):
    x = torch.zeros(2, 64, dtype=dtype)
    u8 = torch.zeros(1280, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ops.mxfp4_quantize(x)
    with pytest.raises(ValueError):
        ops.mxfp4_product(x, u8, 32)
    with pytest.raises(ValueError):
        ops.mxfp4_gated(x, u8, u8, 32)
    with pytest.raises(ValueError):
        ops.mxfp4_gated_backward(x, x, u8, u8, 64)
    with pytest.raises(ValueError):
        ops.mxfp4_pack(u8.view(1, -1), u8[:80].view(1, -1))


@pytest.mark.parametrize("status", [torch.zeros(1, dtype=torch.int32), torch.zeros(1),
                                    torch.zeros(0, dtype=torch.int32)])
def test_quantize_refuses_a_status_that_the_device_cannot_write(status):
    with pytest.raises(ValueError, match="status"):
        ops.mxfp4_quantize(torch.zeros(2, 64), status)


def test_workspaces_are_asked_for_on_each_device(monkeypatch):
    """Their sizes follow from the current device's compute units."""
    current = 0

    class Library:
        kdq_mxfp4_packed_bytes = staticmethod(lambda rows, cols: rows * cols)
        kdq_mxfp4_product_workspace = staticmethod(lambda *sizes: 8192 * (1 + current))

    monkeypatch.setattr(ops, "lib", lambda: Library)
    monkeypatch.setattr(ops, "_current_device", lambda: current, raising=False)
    sizes = ("kdq_mxfp4_packed_bytes", 7, 32, "kdq_mxfp4_product_workspace", 5, 7, 32, 0)
    try:
        for current in (0, 1, 0):
            assert ops._mxfp4_sizes(*sizes) == (7 * 32, 8192 * (1 + current))
    finally:  # (sizes of the stand-in stay in no cache)
        for name in ("_mxfp4_size", "_mxfp4_sizes", "_mxfp4_sizes_on"):
            getattr(getattr(ops, name, None), "cache_clear", lambda: None)()


@pytest.mark.parametrize("quantized", [0, 1])
def test_a_workspace_over_an_input_is_refused(quantized):
    """K slices' partial results would replace x or the matrix while others still read them."""
    lib = kadan_amd.lib()
    m, n, k = (77, 4096, 14336) if not quantized else (200, 4096, 14336)
    need = lib.kdq_mxfp4_product_workspace(m, n, k, quantized)
    assert need > 0
    x, scales, w, y, ws = (i << 40 for i in range(1, 6))
    x_bytes, w_bytes = m * k * 2 // (1 if not quantized else 4), lib.kdq_mxfp4_packed_bytes(n, k)

    def call(workspace, size=need):
        if quantized:
            return lib.kdq_mxfp4_product_quantized(x, scales, m, w, n, k, 0, y, n, workspace, size,
                                                   None)
        return lib.kdq_mxfp4_product(x, k, m, w, n, k, 0, y, n, workspace, size, None)

    for base, size in ((x, x_bytes), (w, w_bytes), (y, m * n * 4)) + (
            ((scales, m * k // 32),) if quantized else ()):
        assert call(base) == 4 and call(base + size - 16) == 4 and call(base - need + 16) == 4
    assert call(ws, need - 1) == 6  # (apart from all of them: the next check)
    # a workspace that the call does not need is the caller's word for what it may write, too
    assert lib.kdq_mxfp4_product_workspace(1, 64, 64, quantized) == 0
    if quantized:
        assert lib.kdq_mxfp4_product_quantized(x, scales, 1, w, 64, 64, 0, y, 64, x, 16, None) == 4
    else:
        assert lib.kdq_mxfp4_product(x, 64, 1, w, 64, 64, 0, y, 64, w, 16, None) == 4


def test_a_gradient_that_would_be_lost_is_refused():
    """Before anything else about the call; not where no graph is recorded."""
    x, u8 = torch.zeros(2, 64, dtype=torch.bfloat16, requires_grad=True), torch.zeros(
        1280, dtype=torch.uint8)
    calls = (lambda: ops.mxfp4_product(x, u8, 32), lambda: ops.mxfp4_gated(x, u8, u8, 32),
             lambda: ops.mxfp4_gated_backward(x, x, u8, u8, 64))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="device tensor"):
            call()


class Packed:
    """What the wrappers look at of a packed device tensor."""
    dtype, is_cuda = torch.uint8, True

    def __init__(self, *shape):
        self.shape = torch.Size(shape)
        self.dim, self.numel = lambda: len(shape), self.shape.numel
        self.is_contiguous, self.data_ptr = lambda: True, lambda: W


@pytest.mark.parametrize("rows,cols", [(64, 256), (14336, 4096), (4096, 8192), (64, 64)])
def test_the_two_packed_forms_are_told_apart(rows, cols):
    """Also where they take the same number of bytes, or the same but for a few."""
    lib = kadan_amd.lib()
    size = lib.kdq_mxfp4_packed_bytes(rows, cols)
    transposed = lib.kdq_mxfp4_packed_transposed_bytes(rows, cols)
    assert (size == transposed) == (cols != 64)
    groups = cols // 64
    t = Packed(groups, transposed // groups)
    assert ops._matrix(Packed(size), size, "packed") == W
    assert ops._transposed_matrix(t, transposed, cols, "gate") == W
    with pytest.raises(ValueError, match="gate"):
        ops._transposed_matrix(Packed(size), transposed, cols, "gate")
    with pytest.raises(ValueError, match="packed"):
        ops._matrix(t, size, "packed")
    if groups > 1:  # another matrix of as many bytes
        with pytest.raises(ValueError, match="gate"):
            ops._transposed_matrix(Packed(groups // 2, 2 * transposed // groups), transposed, cols,
                                   "gate")


def test_matrices_past_a_launch_of_32_bits_are_refused():
    """A packing launch counts its threads in 32 bits: up to 2^36 values, 32 GB of codes."""
    lib = kadan_amd.lib()
    far = 1 << 45
    assert lib.kdq_mxfp4_packed_bytes(1 << 23, 1 << 13) == (1 << 35) + (1 << 31)
    assert lib.kdq_mxfp4_packed_bytes((1 << 23) + 1, 1 << 13) == 0
    assert lib.kdq_mxfp4_pack(W, far, 1 << 24, 1 << 13, 2 * far, None) == 2
    assert lib.kdq_mxfp4_packed_transposed_bytes(1 << 18, 1 << 18) == (1 << 35) + (1 << 31)
    assert lib.kdq_mxfp4_packed_transposed_bytes(1 << 18, (1 << 18) + 32) == 0
    assert lib.kdq_mxfp4_pack_transposed(W, far, 1 << 20, 1 << 18, 2 * far, None) == 2
    n, k = 1 << 24, 1 << 13
    assert lib.kdq_mxfp4_product_workspace(1, n, k, 0) == 0
    assert lib.kdq_mxfp4_product(X, k, 1, far, n, k, 0, 2 * far, n, None, 0, None) == 2
    assert lib.kdq_mxfp4_product_quantized(X, Z, 1, far, n, k, 0, 2 * far, n, None, 0, None) == 2
    assert lib.kdq_mxfp4_gated(X, k, 1, far, 2 * far, n, k, 4 * far, n, None, None, None, None, 0,
                               None) == 2
    n = k = 1 << 19
    assert lib.kdq_mxfp4_gated_backward(X, n, 1, Y, None, None, far, 2 * far, n, k, Z, W, k, None,
                                        0, None) == 2


def test_reference_quantiser_is_nearest_and_ties_to_even():
    """The oracle of the GPU tests, by hand: the format's own values, ties, and saturation."""
    row = np.zeros((1, 32))
    row[0, :12] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.5, -6.9, 0.26, 7.0]
    blocks, scales = ref.quantize(row)
    assert scales.tolist() == [[127]]
    codes = [int(b) >> s & 15 for b in blocks[0] for s in (0, 4)]
    assert codes[:12] == [7, 0, 2, 2, 4, 4, 6, 6, 9, 15, 1, 7]
    for e in (-127, -3, 90):
        got = ref.quantize(row * 2.0 ** e)
        assert got[1].tolist() == [[127 + e]] and np.array_equal(got[0], blocks)
    values = ref.decode(torch.from_numpy(blocks), torch.from_numpy(scales))[0, :12].tolist()
    assert values == [6, 0, 1, 1, 2, 2, 4, 4, -0.5, -6, 0.5, 6]


def test_gradient_formula_against_differences():
    g, u, dh = (torch.randn(3, 32, dtype=torch.float64) * 3 for _ in range(3))
    want, _ = ref.gate_gradients(dh, g, u)
    f = lambda a, b: dh * a * torch.sigmoid(a) * b
    e = 1e-6
    numeric = torch.cat([(f(g + e, u) - f(g - e, u)) / (2 * e),
                         (f(g, u + e) - f(g, u - e)) / (2 * e)], 1)
    # Central differences of f in x are off by e^2 / 6 times the third derivative, which is below
    # |dh u| in g (silu's is below 1) and 0 in u; by the rounding of f's two values, 8 * 2^-53 of
    # them (three products and a sigmoid of at most five roundings), over e; and by that of
    # x + e and x - e, 2^-53 of them each, times the slope, over e.  Slopes are at most
    # 1.1 |dh u| in g and |dh g| in u.  The formula itself is off by a few of its terms' roundings.
    half = 2.0 ** -53

    def bound(x, slope, third):
        value = f(g, u).abs() + slope * e
        return third * e * e / 6 + (8 * half * value + half * (x.abs() + e) * slope) / e

    terms = (dh * u).abs() * (2 + 2 * g.abs()) + (dh * g).abs()
    limit = torch.cat([bound(g, 1.1 * (dh * u).abs(), (dh * u).abs()),
                       bound(u, (dh * g).abs(), torch.zeros_like(g))], 1)
    limit = limit + 16 * half * torch.cat([terms, terms], 1)
    assert bool(((want - numeric).abs() <= limit).all())
