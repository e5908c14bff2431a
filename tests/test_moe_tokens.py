"""CPU checks of the mixture's pieces: refusals of the C ABI before any launch (the pointers are
never dereferenced)."""
import kadan_amd

X, P, R, Q, Y, V = (0x10000000 * i for i in range(1, 7))
F32, F16, BF16 = 0, 1, 30


def caller(name, order, good):
    f = getattr(kadan_amd.lib(), name)

    def call(**change):
        a = {**good, **change}
        return f(*(a[key] for key in order), None)

    return call


def test_sort_refusals():
    call = caller("kdq_moe_sort", "type x xs t c k perm rows rs place".split(),
                  dict(type=BF16, x=X, xs=64, t=4, c=64, k=2, perm=P, rows=R, rs=64, place=Q))
    for name in ("x", "perm", "rows", "place"):
        assert call(**{name: None}) == 1
    for name in ("t", "c", "k"):
        assert call(**{name: 0}) == 1
    assert call(k=9) == 2 and call(t=(1 << 20) + 1) == 2 and call(c=(1 << 20) + 1) == 2
    assert call(xs=63) == 2 and call(rs=63) == 2 and call(xs=1 << 62) == 2
    assert call(type=8) == 3
    assert call(x=X + 1) == 7 and call(rows=R + 1) == 7 and call(perm=P + 2) == 7
    assert call(place=Q + 2) == 7 and call(type=F32, x=X + 2) == 7
    assert call(rows=X + 510) == 4 and call(place=X + 4) == 4 and call(place=P + 28) == 4
    assert call(place=R + 8 * 128 - 4) == 4


def test_sort_backward_refusals():
    call = caller("kdq_moe_sort_backward", "type d ds place t c k dx dxs".split(),
                  dict(type=F16, d=R, ds=64, place=Q, t=4, c=64, k=2, dx=X, dxs=64))
    for name in ("d", "place", "dx"):
        assert call(**{name: None}) == 1
    for name in ("t", "c", "k"):
        assert call(**{name: 0}) == 1
    assert call(k=9) == 2 and call(ds=63) == 2 and call(dxs=63) == 2
    assert call(type=12) == 3
    assert call(d=R + 1) == 7 and call(dx=X + 1) == 7 and call(place=Q + 1) == 7
    assert call(dx=R + 8 * 128 - 2) == 4 and call(dx=Q) == 4


def test_combine_refusals():
    call = caller("kdq_moe_combine", "type r rs place w t c k ytype add adds y ys".split(),
                  dict(type=BF16, r=R, rs=64, place=Q, w=V, t=4, c=64, k=2, ytype=F32, add=P,
                       adds=64, y=Y, ys=64))
    for name in ("r", "place", "w", "y"):
        assert call(**{name: None}) == 1
    for name in ("t", "c", "k"):
        assert call(**{name: 0}) == 1
    assert call(k=9) == 2 and call(rs=63) == 2 and call(adds=63) == 2 and call(ys=63) == 2
    assert call(type=2) == 3 and call(ytype=F16) == 3 and call(ytype=8) == 3
    assert call(r=R + 1) == 7 and call(y=Y + 2) == 7 and call(add=P + 2) == 7
    assert call(w=V + 2) == 7 and call(place=Q + 2) == 7
    assert call(y=R) == 4 and call(y=Q) == 4 and call(y=V) == 4
    # the residual in part, or with another stride
    assert call(y=P + 64) == 4 and call(y=P, ys=65) == 4


def test_combine_backward_refusals():
    call = caller("kdq_moe_combine_backward", "type r rs place w t c k dtype d ds o os dw".split(),
                  dict(type=BF16, r=R, rs=64, place=Q, w=V, t=4, c=64, k=2, dtype=BF16, d=X, ds=64,
                       o=Y, os=64, dw=P))
    for name in ("r", "place", "w", "d", "o", "dw"):
        assert call(**{name: None}) == 1
    for name in ("t", "c", "k"):
        assert call(**{name: 0}) == 1
    assert call(k=9) == 2 and call(rs=63) == 2 and call(ds=63) == 2 and call(os=63) == 2
    assert call(type=2) == 3 and call(dtype=F16) == 3
    assert call(r=R + 1) == 7 and call(d=X + 1) == 7 and call(o=Y + 1) == 7 and call(dw=P + 2) == 7
    assert call(o=R) == 4 and call(o=X) == 4 and call(dw=V) == 4 and call(dw=Y) == 4
    assert call(o=Q) == 4 and call(dw=Q) == 4


def test_route_backward_refusals():
    call = caller("kdq_moe_route_backward", "idx w dw t e k out".split(),
                  dict(idx=X, w=P, dw=R, t=4, e=8, k=2, out=Y))
    for name in ("idx", "w", "dw", "out"):
        assert call(**{name: None}) == 1
    for name in ("t", "e", "k"):
        assert call(**{name: 0}) == 1
    assert call(e=257) == 2 and call(k=9, e=16) == 2 and call(k=3, e=2) == 2
    assert call(idx=X + 2) == 7 and call(out=Y + 1) == 7
    assert call(out=X) == 4 and call(out=P) == 4 and call(out=R) == 4
