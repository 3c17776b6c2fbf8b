"""vb_qk_norm_rope and its backward against their definition in 64 bits: head sizes on both kernels, views, positions, refusals."""
import ctypes as C

import numpy as np
import pytest

from tests.decoder_ops_util import Dev, U, norm_rope, norm_rope_grad, outputs, rnd

pytestmark = pytest.mark.gpu
THETA = 10000.0


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def case(seed, T, hq, hk, dk, scale=1.0):
    return (rnd(seed, T, hq, dk, scale=scale), rnd(seed + 1, T, hk, dk, scale=scale), 1 + rnd(seed + 2, dk, scale=0.2), 1 + rnd(seed + 3, dk, scale=0.2))


def forward_bound(y, dk, w):
    """Per element: the sum of squares carries at most (dk / 8 + 4) roundings on the vector path and dk / 32 + 6 on the scalar one
    (under (dk / 8 + 8) U, halved by the root), the quotient, its root, two products and the two terms of the turn one each; the cosine and
    sine are good to 2 U plus the angle's U.  A turned component is at most the length of its pair, at most max |w| sqrt(dk)
    (a head of unit mean square); measured against its own pair it is under |y_a| + |y_b|, bounded here by the head's largest."""
    return (dk / 16 + 16) * U * np.abs(y).max(-1, keepdims=True) * 1.5


SHAPES = [  # tokens, q heads, k heads, head size, rotated width, interleaved
    (1, 1, 1, 8, 8, False), (1, 12, 4, 64, 64, False), (7, 3, 1, 64, 64, True), (33, 12, 4, 64, 32, False), (129, 5, 5, 128, 128, False),
    (50, 16, 2, 128, 64, True), (19, 2, 1, 80, 80, False), (19, 2, 1, 80, 40, True), (9, 2, 2, 256, 256, False), (6, 2, 1, 200, 0, False),
    (5, 3, 2, 6, 4, False), (5, 3, 2, 1, 0, False), (11, 2, 1, 20, 20, False), (11, 2, 1, 20, 12, True), (4, 1, 1, 512, 512, False), (3, 1, 2, 300, 26, True),
    (2000, 12, 4, 64, 64, False),
]


@pytest.mark.parametrize("T,hq,hk,dk,rot,inter", SHAPES)
def test_forward(vb, T, hq, hk, dk, rot, inter):
    q, k, wq, wk = case(1, T, hq, hk, dk)
    pos = (np.arange(T) * 37 % 8192).astype(np.float32)
    d = [Dev(vb, a) for a in (q, k, wq, wk, pos)]
    oq, ok = outputs(vb, vb.lib().vb_qk_norm_rope, *d, THETA, rot, int(inter), 1e-6, n=2)
    for o, x, w in ((oq, q, wq), (ok, k, wk)):
        y = norm_rope(x, w, pos, THETA, rot, inter, 1e-6)
        assert (np.abs(o - y) <= forward_bound(y, dk, w)).all()


def grad_bounds(x, w, g, eps, T, H):
    """gx: the terms g' w inv and x-hat c inv each carry the roundings of forward_bound and those of the mean c, all relative to
    inv * max |w| * |g|_head.  gw: a sum of T H products, each with some twenty roundings, added in at most T H + 64 steps (few in practice)."""
    dk = x.shape[-1]
    x64 = x.astype(np.float64)
    inv = 1.0 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + eps)
    size = inv * np.abs(w).max() * np.sqrt((g.astype(np.float64) ** 2).sum(-1, keepdims=True))
    gx = (dk / 8 + 40) * U * size
    steps = 40 + T * H / 64 + 700
    gw = steps * U * (np.sqrt((g.astype(np.float64) ** 2).sum(-1, keepdims=True)) * np.abs(x64 * inv).max(-1, keepdims=True)).sum()
    return gx, gw


@pytest.mark.parametrize("T,hq,hk,dk,rot,inter", SHAPES)
def test_backward(vb, T, hq, hk, dk, rot, inter):
    q, k, wq, wk = case(11, T, hq, hk, dk, scale=2.0)
    gq, gk = rnd(21, T, hq, dk), rnd(22, T, hk, dk)
    pos = (np.arange(T) * 91 % 5000).astype(np.float32)
    d = [Dev(vb, a) for a in (q, k, wq, wk, pos)]
    got = outputs(vb, vb.lib().vb_qk_norm_rope_backward, *d, THETA, rot, int(inter), 1e-6, Dev(vb, gq), Dev(vb, gk), n=4)
    for gx, gw, x, w, g in ((got[0], got[2], q, wq, gq), (got[1], got[3], k, wk, gk)):
        ex, ew = norm_rope_grad(x, w, pos, THETA, rot, inter, 1e-6, g)
        bx, bw = grad_bounds(x, w, g, 1e-6, T, x.shape[1])
        assert (np.abs(gx - ex) <= bx).all()
        assert (np.abs(gw - ew) <= bw).all()


def test_gradient_against_differences(vb):
    """d(sum of y g) along a direction, by central differences of the 64-bit definition."""
    T, h, dk = 5, 3, 64
    q, _, wq, _ = case(31, T, h, h, dk)
    g, dx, dw, pos = rnd(35, T, h, dk), rnd(36, T, h, dk), rnd(37, dk), np.arange(T, dtype=np.float32) + 100
    args = (Dev(vb, q), None, Dev(vb, wq), None, Dev(vb, pos), THETA, dk, 0, 1e-6, Dev(vb, g), None)
    outs = [vb.VbTensor() for _ in range(2)]
    vb.vb_check(vb.lib().vb_qk_norm_rope_backward(*[a.ref if isinstance(a, Dev) else a for a in args], C.byref(outs[0]), None, C.byref(outs[1]), None))
    gx, gw = np.empty((T, h, dk), np.float32), np.empty(dk, np.float32)
    for o, a in zip(outs, (gx, gw)):
        vb.vb_check(vb.lib().vb_read(o.slot, 0, a.ctypes.data_as(vb.c_f32p), a.size))
        vb.lib().vb_release(o.slot, None)

    def f(step):
        x64, w64 = q.astype(np.float64) + step * dx, wq.astype(np.float64) + step * dw
        y = x64 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + 1e-6) * w64
        from tests.decoder_ops_util import rope
        return (rope(y, pos, THETA, dk, False) * g).sum()
    h_ = 1e-4
    want = (f(h_) - f(-h_)) / (2 * h_)
    # second-order error of the difference about h^2 times third derivatives of order one a component, and f32 sums of 960 terms of order one
    assert abs((gx.astype(np.float64) * dx).sum() + (gw.astype(np.float64) * dw).sum() - want) <= 1e-8 * 1000 + 960 * 64 * U


@pytest.mark.parametrize("view", ["strided", "odd", "turned"])
@pytest.mark.parametrize("dk,rot", [(64, 64), (20, 12)])
def test_views_give_the_same_values(vb, view, dk, rot):
    q, k, wq, wk = case(41, 13, 4, 2, dk)
    g, gk_ = rnd(45, 13, 4, dk), rnd(46, 13, 2, dk)
    pos = np.arange(13, dtype=np.float32)
    ws = [Dev(vb, a) for a in (wq, wk, pos)]
    L = vb.lib()
    for fn, extra, n in ((L.vb_qk_norm_rope, False, 2), (L.vb_qk_norm_rope_backward, True, 4)):
        tail = lambda v: [Dev(vb, g, v), Dev(vb, gk_, v)] if extra else []  # noqa: E731
        a = outputs(vb, fn, Dev(vb, q), Dev(vb, k), *ws, THETA, rot, 0, 1e-6, *tail("whole"), n=n)
        b = outputs(vb, fn, Dev(vb, q, view), Dev(vb, k, view), *ws, THETA, rot, 0, 1e-6, *tail(view), n=n)
        for x, y in zip(a, b):      # other kernels may take other orders: the bounds of the tests above, twice
            assert np.abs(x - y).max() <= 2 * (dk / 8 + 60) * U * max(1.0, np.abs(x).max()) * 8


def test_far_negative_and_fractional_positions(vb):
    T, dk = 6, 64
    q, _, wq, _ = case(51, T, 2, 1, dk)
    pos = np.array([0.0, 16777215.0, -16777215.0, 1.5, -0.25, 4194303.5], np.float32)
    outs = vb.VbTensor()
    dq, dw, dp = Dev(vb, q), Dev(vb, wq), Dev(vb, pos)
    vb.vb_check(vb.lib().vb_qk_norm_rope(dq.ref, None, dw.ref, None, dp.ref, THETA, dk, 0, 1e-6, C.byref(outs), None))
    a = np.empty((T, 2, dk), np.float32)
    vb.vb_check(vb.lib().vb_read(outs.slot, 0, a.ctypes.data_as(vb.c_f32p), a.size))
    vb.lib().vb_release(outs.slot, None)
    y = norm_rope(q, wq, pos, THETA, dk, False, 1e-6)
    assert (np.abs(a - y) <= forward_bound(y, dk, wq)).all()


def test_zero_rows_infinities_and_no_tokens(vb):
    q = rnd(61, 4, 2, 64)
    q[1] = 0.0
    q[2, 1, 5] = np.inf
    wq, pos = Dev(vb, np.ones(64, np.float32)), Dev(vb, np.arange(4, dtype=np.float32))
    oq, ok = outputs(vb, vb.lib().vb_qk_norm_rope, Dev(vb, q), Dev(vb, q), wq, wq, pos, THETA, 64, 0, 1e-6, n=2)
    assert (oq[1] == 0).all() and np.isfinite(oq[[0, 1, 3]]).all() and np.isfinite(oq[2, 0]).all() and not np.isfinite(oq[2, 1]).all()
    empty = np.zeros((0, 2, 64), np.float32)
    p0 = Dev(vb, np.zeros(0, np.float32))
    oq, ok = outputs(vb, vb.lib().vb_qk_norm_rope, Dev(vb, empty), Dev(vb, empty), wq, wq, p0, THETA, 64, 0, 1e-6, n=2)
    assert oq.shape == (0, 2, 64)
    got = outputs(vb, vb.lib().vb_qk_norm_rope_backward, Dev(vb, empty), Dev(vb, empty), wq, wq, p0, THETA, 64, 0, 1e-6, Dev(vb, empty), Dev(vb, empty), n=4)
    assert (got[2] == 0).all() and (got[3] == 0).all()


def test_refusals_leave_no_slot_behind(vb):
    q, k, w, pos = Dev(vb, rnd(71, 5, 2, 64)), Dev(vb, rnd(72, 5, 1, 64)), Dev(vb, rnd(73, 64)), Dev(vb, np.arange(5, dtype=np.float32))
    short, flat, wide = Dev(vb, rnd(74, 4, 1, 64)), Dev(vb, rnd(75, 5, 64)), Dev(vb, rnd(76, 5, 1, 514))
    w514 = Dev(vb, rnd(77, 514))
    L = vb.lib()
    o = [vb.VbTensor(), vb.VbTensor()]
    r = lambda x: None if x is None else x.ref  # noqa: E731
    before = vb.memory_stats()["live_slots"]
    for args in ((q, k, w, None, pos, THETA, 64, 0, 1e-6), (q, None, w, w, pos, THETA, 64, 0, 1e-6), (flat, None, w, None, pos, THETA, 64, 0, 1e-6),
                 (q, short, w, w, pos, THETA, 64, 0, 1e-6), (q, k, w514, w, pos, THETA, 64, 0, 1e-6), (q, k, w, w, w, THETA, 64, 0, 1e-6),
                 (q, k, w, w, pos, THETA, 63, 0, 1e-6), (q, k, w, w, pos, THETA, 66, 0, 1e-6), (q, k, w, w, pos, THETA, -2, 0, 1e-6),
                 (q, k, w, w, pos, 0.0, 64, 0, 1e-6), (q, k, w, w, pos, float("nan"), 64, 0, 1e-6), (q, k, w, w, pos, THETA, 64, 0, -1.0),
                 (None, None, w, None, pos, THETA, 64, 0, 1e-6), (wide, None, w514, None, pos, THETA, 64, 0, 1e-6)):
        rc = L.vb_qk_norm_rope(*[r(a) for a in args[:5]], *args[5:], C.byref(o[0]), C.byref(o[1]))
        assert rc in (1, 8), (rc, args)
        assert L.vb_last_error()
    assert L.vb_qk_norm_rope(q.ref, k.ref, w.ref, w.ref, pos.ref, THETA, 64, 0, 1e-6, C.byref(o[0]), None) == 1
    assert L.vb_qk_norm_rope_backward(q.ref, k.ref, w.ref, w.ref, pos.ref, THETA, 64, 0, 1e-6, q.ref, None, C.byref(o[0]), C.byref(o[1]), C.byref(o[0]), C.byref(o[1])) == 1
    assert vb.memory_stats()["live_slots"] == before


def test_the_same_bits_twice(vb):
    q, k, wq, wk = case(81, 777, 6, 2, 64)
    pos = np.arange(777, dtype=np.float32)
    d = [Dev(vb, a) for a in (q, k, wq, wk, pos, rnd(85, 777, 6, 64), rnd(86, 777, 2, 64))]
    run = lambda: outputs(vb, vb.lib().vb_qk_norm_rope_backward, *d[:5], THETA, 64, 0, 1e-6, *d[5:], n=4)  # noqa: E731
    for a, b in zip(run(), run()):
        assert (a == b).all()
