"""CPU checks of the MXFP4 products with an epilogue and of the experts' forms: sizes, workspaces
and refusals of the C ABI before any launch (the pointers are never dereferenced), and the
reference that the GPU tests compare with."""
import pytest
import torch

import kadan_amd

import mxfp4_epilogue_reference as epi

W, V, X, Y, Z, B, O, R, K, Q, S = (0x10000000 * i for i in range(1, 12))


def caller(name, order, good):
    f = getattr(kadan_amd.lib(), name)

    def call(**change):
        a = {**good, **change}
        return f(*(a[key] for key in order.split()), None)

    return call


def test_packed_sizes():
    lib = kadan_amd.lib()
    size = lib.kdq_mxfp4_experts_packed_bytes
    turned = lib.kdq_mxfp4_experts_packed_transposed_bytes
    assert size(32, 2880, 2880) == lib.kdq_moe_mxfp4_packed_bytes(32, 2880, 2880)
    assert size(3, 33, 288) == 3 * lib.kdq_mxfp4_packed_bytes(33, 288)
    assert turned(3, 65, 96) == 3 * lib.kdq_mxfp4_packed_transposed_bytes(65, 96)
    assert size(256, 1, 32) and turned(256, 1, 32)
    for f in (size, turned):
        assert f(0, 64, 64) == f(257, 64, 64) == f(4, 0, 64) == f(4, 64, 48) == 0
    assert lib.kdq_mxfp4_linear_workspace(64, 0, 4096, 14336) == \
        lib.kdq_mxfp4_product_workspace(64, 4096, 14336, 0)
    work = lib.kdq_mxfp4_linear_backward_workspace
    assert work(64, 0, 14336, 4096) and work(0, 0, 64, 64) == work(64, 0, 64, 48) == 0
    # of experts: partial sums where the tiles are few, and none where they are many
    fits = [(lib.kdq_mxfp4_linear_workspace, ()), (work, ()),
            (lib.kdq_mxfp4_experts_gated_workspace, (1,)),
            (lib.kdq_mxfp4_experts_gated_backward_workspace, ())]
    for f, last in fits:
        assert f(64, 1, 4096, 14336, *last) and f(32768, 32, 2880, 2880, *last) == 0
        assert f(0, 2, 64, 64, *last) == f(64, 257, 2880, 2880, *last) == 0
        assert f(64, 2, 2880, 2872, *last) == 0
    assert lib.kdq_mxfp4_experts_gated_workspace(4, 32, 2880, 2880, 0) == 0  # (one kernel)
    assert lib.kdq_mxfp4_experts_gated_workspace(64, 2, 0, 64, 0) == 0


def test_pack_refusals():
    lib = kadan_amd.lib()
    for f in (lib.kdq_mxfp4_experts_pack, lib.kdq_mxfp4_experts_pack_transposed):
        assert f(None, X, 2, 32, 64, Y, None) == 1 and f(W, X, 0, 32, 64, Y, None) == 1
        assert f(W, X, 257, 32, 64, Y, None) == 2 and f(W, X, 2, 32, 48, Y, None) == 2
        assert f(W + 8, X, 2, 32, 64, Y, None) == 7 and f(W, X, 2, 32, 64, Y + 8, None) == 7
        assert f(W, X, 2, 32, 64, W + 1024, None) == 4  # (the second matrix)
        assert f(W, Y + 2048, 2, 32, 64, Y, None) == 4


LINEAR = "x xs m o e w n k b act r rs t y ys kept ws wb"


def linear(**more):
    return caller("kdq_mxfp4_linear", LINEAR,
                  dict(x=X, xs=64, m=2, o=None, e=1, w=W, n=40, k=64, b=B, act=2, r=R, rs=40, t=0,
                       y=Y, ys=40, kept=K, ws=None, wb=0, **more))


@pytest.mark.parametrize("experts", [0, 4])
def test_linear_refusals(experts):
    call = linear()
    if experts:
        dense = call
        call = lambda **c: dense(**{"o": O, "e": experts, **c})  # noqa: E731
    for name in ("x", "w", "y"):
        assert call(**{name: None}) == 1
    for name in ("m", "n", "k", "e"):
        assert call(**{name: 0}) == 1
    assert call(k=48, xs=48) == 2 and call(xs=63) == 2 and call(xs=68) == 2
    assert call(xs=(1 << 21) + 8) == 2 and call(m=(1 << 20) + 1) == 2
    assert call(ys=39) == 2 and call(rs=39) == 2
    assert call(act=3) == 3 and call(act=-1) == 3 and call(t=1) == 3
    assert call(x=X + 8) == 7 and call(w=W + 8) == 7 and call(y=Y + 2) == 7
    assert call(b=B + 2) == 7 and call(r=R + 2) == 7 and call(kept=K + 1) == 7
    assert call(y=X + 128) == 4 and call(y=W + 64) == 4 and call(y=B) == 4 and call(kept=Y) == 4
    assert call(y=R + 16) == 4 and call(y=R, rs=41) == 4 and call(kept=X) == 4
    if experts:
        assert call(y=O) == 4 and call(o=O + 2) == 7 and call(e=257) == 2
        assert call(y=B + 3 * 40 * 4) == 4  # (the last expert's bias)
        many = dict(m=64, e=1, n=4096, k=14336, xs=14336, ys=4096, rs=4096)
        need = kadan_amd.lib().kdq_mxfp4_linear_workspace(64, 1, 4096, 14336)
        assert call(**many) == 6 and call(**many, ws=Z, wb=need - 16) == 6
        assert call(**many, ws=Z + 8, wb=need) == 7 and call(**many, ws=O, wb=need) == 4
    else:
        assert call(e=2) == 1
        # K slices need their workspace, aligned and apart from everything else
        many = dict(m=64, n=4096, k=14336, xs=14336, ys=4096, rs=4096)
        need = kadan_amd.lib().kdq_mxfp4_linear_workspace(64, 0, 4096, 14336)
        assert call(**many) == 6 and call(**many, ws=Z, wb=need - 16) == 6
        assert call(**many, ws=Z + 8, wb=need) == 7 and call(**many, ws=X, wb=need) == 4
        assert call(**many, ws=K, wb=need) == 4 and call(**many, ws=R, wb=need) == 4


BACK = "d ds m o e kept act w n k dp dx dxs ws wb"


@pytest.mark.parametrize("experts", [0, 4])
def test_linear_backward_refusals(experts):
    call = caller("kdq_mxfp4_linear_backward", BACK,
                  dict(d=Y, ds=40, m=2, o=O if experts else None, e=experts or 1, kept=K, act=1,
                       w=W, n=40, k=64, dp=Q, dx=X, dxs=64, ws=None, wb=0))
    for name in ("d", "w", "dx", "kept", "dp"):
        assert call(**{name: None}) == 1
    for name in ("m", "n", "k", "e"):
        assert call(**{name: 0}) == 1
    assert call(act=0) == 1 and call(act=0, kept=None) == 1  # (nothing to keep, no dpre)
    assert call(n=36, ds=40) == 2 and call(k=48, dxs=48) == 2 and call(ds=39) == 2
    assert call(ds=44) == 2 and call(dxs=63) == 2 and call(m=(1 << 20) + 1) == 2
    assert call(act=3) == 3
    assert call(d=Y + 8) == 7 and call(w=W + 8) == 7 and call(dp=Q + 8) == 7
    assert call(dx=X + 1) == 7 and call(kept=K + 1) == 7
    assert call(dx=Y) == 4 and call(dp=Y) == 4 and call(dx=Q) == 4 and call(dp=K) == 4
    assert call(dx=W + 16) == 4
    if experts:
        assert call(dx=O) == 4 and call(o=O + 1) == 7 and call(e=257) == 2
        many = dict(m=64, e=1, n=14336, k=4096, ds=14336, dxs=4096)
        need = kadan_amd.lib().kdq_mxfp4_linear_backward_workspace(64, 1, 14336, 4096)
        assert call(**many) == 6 and call(**many, ws=Z + 8, wb=need) == 7
        assert call(**many, ws=O, wb=need) == 4 and call(**many, ws=Q, wb=need) == 4
    else:
        many = dict(m=64, n=14336, k=4096, ds=14336, dxs=4096)
        need = kadan_amd.lib().kdq_mxfp4_linear_backward_workspace(64, 0, 14336, 4096)
        assert call(**many) == 6 and call(**many, ws=Z + 8, wb=need) == 7
        assert call(**many, ws=Q, wb=need) == 4


def test_experts_gated_refusals():
    call = caller("kdq_mxfp4_experts_gated", "x xs m o e g u n k bg bu act h hs kb kq ks ws wb",
                  dict(x=X, xs=64, m=2, o=O, e=4, g=W, u=V, n=32, k=64, bg=B, bu=R, act=1, h=Y,
                       hs=32, kb=None, kq=Q, ks=S, ws=None, wb=0))
    for name in ("x", "o", "g", "u", "h", "bg", "bu", "kq", "ks"):
        assert call(**{name: None}) == 1
    for name in ("m", "n", "k", "e"):
        assert call(**{name: 0}) == 1
    assert call(kb=K) == 1
    assert call(n=40, hs=40) == 2 and call(xs=60) == 2 and call(hs=31) == 2 and call(e=257) == 2
    assert call(act=0) == 3 and call(act=2) == 3 and call(act=4) == 3
    for name, at in (("x", X), ("g", W), ("u", V), ("kq", Q)):
        assert call(**{name: at + 8}) == 7
    assert call(o=O + 2) == 7 and call(bg=B + 2) == 7 and call(ks=S + 2) == 7
    assert call(h=X) == 4 and call(h=B) == 4 and call(kq=R) == 4 and call(ks=Y) == 4
    assert call(h=O) == 4 and call(kb=V, kq=None, ks=None) == 4
    many = dict(m=64, e=1, n=4096, k=14336, xs=14336, hs=4096)
    need = kadan_amd.lib().kdq_mxfp4_experts_gated_workspace(64, 1, 4096, 14336, 1)
    assert call(**many) == 6 and call(**many, ws=Z + 8, wb=need) == 7
    assert call(**many, ws=O, wb=need) == 4 and call(**many, ws=S, wb=need) == 4


def test_experts_gated_backward_refusals():
    call = caller("kdq_mxfp4_experts_gated_backward", "d ds m o e kb kq ks act g u n k dgu dx dxs ws "
                  "wb",
                  dict(d=Y, ds=32, m=2, o=O, e=4, kb=K, kq=None, ks=None, act=3, g=W, u=V, n=32,
                       k=64, dgu=Q, dx=X, dxs=64, ws=None, wb=0))
    for name in ("d", "o", "kb", "g", "u", "dgu", "dx"):
        assert call(**{name: None}) == 1
    for name in ("m", "n", "k", "e"):
        assert call(**{name: 0}) == 1
    assert call(kq=S, ks=B) == 1 and call(kb=None, kq=S) == 1
    assert call(n=40, ds=40) == 2 and call(k=48, dxs=48) == 2 and call(ds=28) == 2
    assert call(act=0) == 3 and call(act=2) == 3
    assert call(d=Y + 8) == 7 and call(g=W + 8) == 7 and call(dgu=Q + 8) == 7 and call(o=O + 2) == 7
    assert call(dx=Y) == 4 and call(dgu=K) == 4 and call(dx=Q) == 4 and call(dgu=V) == 4
    assert call(dx=O) == 4
    many = dict(m=64, e=1, n=14336, k=4096, ds=14336, dxs=4096)
    need = kadan_amd.lib().kdq_mxfp4_experts_gated_backward_workspace(64, 1, 14336, 4096)
    assert call(**many) == 6 and call(**many, ws=Z + 8, wb=need) == 7
    assert call(**many, ws=O, wb=need) == 4 and call(**many, ws=V, wb=need) == 4


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_reference_activations(act):
    """The reference's slope against differences, and its gelu against torch's."""
    v = torch.linspace(-12, 12, 2001, dtype=torch.float64)
    y, _ = epi.activated(v, torch.zeros_like(v), act)
    if act == "gelu":
        assert torch.allclose(y, torch.nn.functional.gelu(v, approximate="tanh"), rtol=1e-9,
                              atol=1e-13)
    step = 2.0 ** -14
    up, _ = epi.activated(v + step, torch.zeros_like(v), act)
    down, _ = epi.activated(v - step, torch.zeros_like(v), act)
    d, _ = epi.slope(v, act)
    # (a central difference is off by step^2 / 6 of the third derivative, which is below 6)
    assert torch.allclose((up - down) / (2 * step), d, rtol=0, atol=step * step + 1e-10)


def test_reference_clamped_gate():
    g = torch.tensor([0.5, 6.9, 7.0, 7.1, -9.0, 2.0], dtype=torch.float64, requires_grad=True)
    u = torch.tensor([0.3, 7.0, -7.0, 7.2, -7.5, -1.0], dtype=torch.float64, requires_grad=True)
    c, v = torch.clamp(g, max=7.0), torch.clamp(u, -7.0, 7.0)
    (c * torch.sigmoid(1.702 * c) * (v + 1)).sum().backward()
    h, by_g, by_u = epi.clamped(g.detach(), u.detach())
    assert torch.allclose(by_g, g.grad, rtol=1e-12) and torch.allclose(by_u, u.grad, rtol=1e-12)
    assert float(h[5]) == 0.0
