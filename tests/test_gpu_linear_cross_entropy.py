"""vb_linear_cross_entropy and its backward against their definition in 64 bits: ragged sizes, left-out rows, magnitudes, refusals."""
import ctypes as C

import numpy as np
import pytest

from tests.decoder_ops_util import Dev, U, outputs, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def product_error(k, size):
    """Bound of one element of a product of half-precision pairs over k, size = sum |a b|: splitting 2^-22 twice and the dropped term 2^-24 (9 U);
    at most 24 truncating additions within a run of 128 (each 2 U of what has been added, 48 U); k / 128 rounded additions."""
    return (57 + k / 128 + 2) * U * size


def truth(x, w, target, ignore, g=1.0):
    x, w = x.reshape(-1, x.shape[-1]).astype(np.float64), w.astype(np.float64)
    live = target != ignore
    z = x @ w.T
    top = z.max(1, keepdims=True)
    lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0]
    n = max(1, live.sum())
    t = np.where(live, target, 0).astype(np.int64)
    loss = np.where(live, lse - z[np.arange(len(t)), t], 0).sum() / n
    p = np.exp(z - lse[:, None])
    d = p.copy()
    d[np.arange(len(t)), t] -= 1
    d *= live[:, None] * (g / n)
    # bounds: a logit, then what follows from it
    ez = product_error(x.shape[1], np.abs(x) @ np.abs(w).T)
    span = np.abs(z - lse[:, None])
    # the exponential's argument is rounded twice (2 U of |z| + |lse| + 20), the exponential is good to 4 U; sums of <= V terms in <= V / 128 + 136 steps
    rel = ez + ez.max(1, keepdims=True) + (4 + 2 * (np.abs(z) + np.abs(lse)[:, None] + 20) + w.shape[0] / 128 + 136) * U
    e_lse = (p * rel).sum(1) + (8 + 2 * np.abs(lse)) * U
    e_loss = (live * (e_lse + ez[np.arange(len(t)), t])).sum() / n + 140 * U * (live * (np.abs(lse) + np.abs(z[np.arange(len(t)), t]))).sum() / n
    ed = live[:, None] * abs(g) / n * (p * (rel + e_lse[:, None]) + 2.0 ** -38 + 8 * U * np.abs(d) * n / abs(g if g else 1.0))
    pieces = 1 + x.shape[0] * w.shape[0] * 4 / 2 ** 29
    egx = ed @ np.abs(w) + product_error(w.shape[0] + 128 * 4 * pieces, np.abs(d) @ np.abs(w)) + 4 * U * np.abs(d @ w)
    egw = ed.T @ np.abs(x) + product_error(x.shape[0] + 512, np.abs(d).T @ np.abs(x)) + 4 * U * np.abs(d.T @ x)
    return (lse, loss, d @ w, d.T @ x), (e_lse, e_loss, egx, egw)


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (33, 128, 512), (128, 64, 256), (129, 72, 257), (5, 768, 1000), (200, 100, 130), (64, 131, 1023), (300, 256, 2049), (1000, 48, 300)]


@pytest.mark.parametrize("n,d,v", SHAPES)
@pytest.mark.parametrize("ignored", [0.0, 0.3])
def test_loss_and_gradients(vb, n, d, v, ignored):
    x, w = rnd(1, n, d), rnd(2, v, d, scale=3.0 / np.sqrt(d))
    r = np.random.default_rng(3)
    t = np.where(r.random(n) < ignored, -100, r.integers(0, v, n)).astype(np.float32)
    (lse, loss, gx, gw), (e_lse, e_loss, egx, egw) = truth(x, w, t, -100, 0.7)
    D = [Dev(vb, a) for a in (x, w, t)]
    got_loss, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    assert (np.abs(got_lse - lse) <= e_lse).all()
    assert abs(got_loss[0] - loss) <= e_loss
    got_gx, got_gw = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, got_lse), Dev(vb, np.array([0.7], np.float32)), n=2)
    vb.check_errors()
    assert got_gx.shape == x.shape and got_gw.shape == w.shape
    assert (np.abs(got_gx - gx) <= egx).all()
    assert (np.abs(got_gw - gw) <= egw).all()


def test_all_rows_left_out(vb):
    x, w, t = rnd(4, 10, 32), rnd(5, 50, 32), np.full(10, -1, np.float32)
    D = [Dev(vb, a) for a in (x, w, t)]
    loss, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -1, n=2)
    gx, gw = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -1, Dev(vb, lse), Dev(vb, np.ones(1, np.float32)), n=2)
    vb.check_errors()
    assert loss[0] == 0 and (gx == 0).all() and (gw == 0).all() and np.isfinite(lse).all()


def test_bad_targets_are_reported_and_left_out(vb):
    x, w = rnd(6, 6, 32), rnd(7, 40, 32)
    t = np.array([3, 40, 39, -2, 0, np.nan], np.float32)
    kept = np.where(np.isin(np.arange(6), [0, 2, 4]), np.nan_to_num(t), -100)
    (_, loss, gx, gw), (_, e_loss, egx, egw) = truth(x, w, kept, -100)
    D = [Dev(vb, a) for a in (x, w, t)]
    got, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    with pytest.raises(vb.VearoError, match="negative.*out of bounds"):
        vb.check_errors()
    assert abs(got[0] - loss) <= e_loss
    a, b = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, lse), Dev(vb, np.ones(1, np.float32)), n=2)
    with pytest.raises(vb.VearoError):
        vb.check_errors()
    assert (np.abs(a - gx) <= egx).all() and (np.abs(b - gw) <= egw).all()


@pytest.mark.parametrize("scale_x,scale_w", [(1e-20, 1e20), (1e15, 1e-15), (300.0, 0.02)])
def test_magnitudes(vb, scale_x, scale_w):
    x, w, t = rnd(8, 70, 96, scale=scale_x), rnd(9, 333, 96, scale=scale_w * 0.3), np.arange(70, dtype=np.float32)
    (lse, loss, gx, gw), (e_lse, e_loss, egx, egw) = truth(x, w, t, -100)
    D = [Dev(vb, a) for a in (x, w, t)]
    got, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    assert (np.abs(got_lse - lse) <= e_lse).all() and abs(got[0] - loss) <= e_loss
    a, b = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, got_lse), Dev(vb, np.ones(1, np.float32)), n=2)
    assert (np.abs(a - gx) <= egx).all() and (np.abs(b - gw) <= egw).all()


def test_large_logits_and_a_certain_row(vb):
    """Logits of some hundreds: one class holds all the mass, the others underflow to 0."""
    x, w = np.eye(8, 16, dtype=np.float32) * 200, np.eye(24, 16, dtype=np.float32)
    t = np.array([0, 1, 2, 3, 4, 5, 6, 23], np.float32)
    (lse, loss, gx, gw), (e_lse, e_loss, egx, egw) = truth(x, w, t, -100)
    D = [Dev(vb, a) for a in (x, w, t)]
    got, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    assert (np.abs(got_lse - lse) <= e_lse).all() and abs(got[0] - loss) <= e_loss
    a, b = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, got_lse), Dev(vb, np.ones(1, np.float32)), n=2)
    assert (np.abs(a - gx) <= egx).all() and (np.abs(b - gw) <= egw).all()


def test_nan_and_infinity_stay_in_their_rows(vb):
    x, w, t = rnd(10, 140, 64), rnd(11, 300, 64), np.zeros(140, np.float32)
    x[3, 7] = np.nan
    x[131, 0] = np.inf
    D = [Dev(vb, a) for a in (x, w, t)]
    loss, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    assert not np.isfinite(lse[[3, 131]]).any() and np.isfinite(np.delete(lse, [3, 131])).all() and not np.isfinite(loss[0])
    gx, _ = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, lse), Dev(vb, np.ones(1, np.float32)), n=2)
    assert not np.isfinite(gx[[3, 131]]).all() and np.isfinite(np.delete(gx, [3, 131], 0)).all()


def test_rows_of_unequal_size(vb):
    """Neighbouring rows of x that differ by 2^60: each has an exponent of its own in the logits and in its gradient."""
    x, w, t = rnd(43, 130, 96), rnd(44, 150, 96, scale=0.2), np.arange(130, dtype=np.float32)
    x[::3] *= 2.0 ** -60
    (lse, loss, gx, _), (e_lse, e_loss, egx, _) = truth(x, w, t, -100)
    D = [Dev(vb, a) for a in (x, w, t)]
    got, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    a, _ = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, got_lse), Dev(vb, np.ones(1, np.float32)), n=2)
    assert (np.abs(got_lse - lse) <= e_lse).all() and abs(got[0] - loss) <= e_loss and (np.abs(a - gx) <= egx).all()


def test_rows_left_out_may_hold_anything(vb):
    x, w = rnd(40, 150, 64), rnd(41, 200, 64)
    t = np.random.default_rng(42).integers(0, 200, 150).astype(np.float32)
    t[[5, 60, 149]] = -100
    (_, loss, gx, gw), (_, e_loss, egx, egw) = truth(x, w, t, -100)
    x[5], x[60], x[149] = np.nan, np.inf, 1e30
    D = [Dev(vb, a) for a in (x, w, t)]
    got, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    a, b = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, lse), Dev(vb, np.ones(1, np.float32)), n=2)
    assert abs(got[0] - loss) <= e_loss and (np.abs(b - gw) <= egw).all()
    assert (a[[5, 60, 149]] == 0).all() and (np.abs(a - gx) <= egx).all()


def test_views_leading_dims_and_one_gradient(vb):
    x, w = rnd(12, 2, 15, 40), rnd(13, 90, 40)
    t = np.random.default_rng(14).integers(0, 90, (2, 15)).astype(np.float32)
    one = Dev(vb, np.ones(1, np.float32))
    L = vb.lib()
    whole = [Dev(vb, a) for a in (x, w, t)]
    _, lse = outputs(vb, L.vb_linear_cross_entropy, *whole, -100, n=2)
    want = outputs(vb, L.vb_linear_cross_entropy_backward, *whole, -100, Dev(vb, lse), one, n=2)
    assert want[0].shape == (2, 15, 40)
    for view in ("strided", "odd", "turned"):
        D = [Dev(vb, x, view), Dev(vb, w, view), Dev(vb, t, view)]
        _, l2 = outputs(vb, L.vb_linear_cross_entropy, *D, -100, n=2)
        got = outputs(vb, L.vb_linear_cross_entropy_backward, *D, -100, Dev(vb, l2), one, n=2)
        assert (l2 == lse).all() and (got[0] == want[0]).all() and (got[1] == want[1]).all()
    o, kept = vb.VbTensor(), Dev(vb, lse)
    D = whole
    for args, ref in (((C.byref(o), None), want[0]), ((None, C.byref(o)), want[1])):
        vb.vb_check(L.vb_linear_cross_entropy_backward(*[d.ref for d in D], -100, kept.ref, one.ref, *args))
        a = np.empty(ref.shape, np.float32)
        vb.vb_check(L.vb_read(o.slot, 0, a.ctypes.data_as(vb.c_f32p), a.size))
        L.vb_release(o.slot, None)
        assert (a == ref).all()


def test_several_pieces_of_the_vocabulary(vb):
    """Enough rows that a piece is 1024 classes wide: three pieces, the last one ragged; against the logits in memory."""
    n, d, v = 131072, 16, 2500
    x, w = rnd(15, n, d), rnd(16, v, d, scale=0.5)
    t = np.random.default_rng(17).integers(0, v, n).astype(np.float32)
    D = [Dev(vb, a) for a in (x, w, t)]
    loss, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    gx, gw = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, lse), Dev(vb, np.full(1, n, np.float32)), n=2)
    pick = np.random.default_rng(18).choice(n, 300, replace=False)
    (l2, _, gx2, _), (e_lse, _, egx, _) = truth(x[pick], w, t[pick], -100, 300.0)
    assert (np.abs(lse[pick] - l2) <= e_lse).all()
    assert (np.abs(gx[pick] - gx2) <= egx).all()
    z = x.astype(np.float64) @ w.astype(np.float64).T
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = float(np.mean(np.log(1 / p[np.arange(n), t.astype(int)])))
    p[np.arange(n), t.astype(int)] -= 1
    gw2 = p.T @ x.astype(np.float64)
    size = np.abs(p).T @ np.abs(x)
    # the bound of truth() with its largest relative error of a probability: logits under 6, 16 components
    worst = (57 + 3) * U * (np.abs(x).max() * np.abs(w).sum(1).max()) * 2 + (40 + 136 + 20) * U
    assert abs(loss[0] - want) <= 2 * worst + 140 * U * 10
    assert (np.abs(gw - gw2) <= (worst * 2 + (59 + n / 128) * U) * size + n * 2.0 ** -38 * np.abs(x).max()).all()


def test_refusals_leave_no_slot_behind(vb):
    x, w, t = Dev(vb, rnd(20, 4, 8)), Dev(vb, rnd(21, 9, 8)), Dev(vb, np.zeros(4, np.float32))
    flat, w7, t5, none = Dev(vb, rnd(22, 8)), Dev(vb, rnd(23, 9, 7)), Dev(vb, np.zeros(5, np.float32)), Dev(vb, np.zeros((0, 8), np.float32))
    lse, g, g2 = Dev(vb, np.zeros(4, np.float32)), Dev(vb, np.ones(1, np.float32)), Dev(vb, np.ones(2, np.float32))
    L = vb.lib()
    o = [vb.VbTensor(), vb.VbTensor()]
    r = lambda a: None if a is None else a.ref  # noqa: E731
    before = vb.memory_stats()["live_slots"]
    for a in ((None, w, t), (x, None, t), (x, w, None), (flat, w, t), (x, w7, t), (x, w, t5), (none, w, t)):
        assert L.vb_linear_cross_entropy(*[r(i) for i in a], -100, C.byref(o[0]), C.byref(o[1])) == 1, a
        assert L.vb_last_error()
    assert L.vb_linear_cross_entropy(x.ref, w.ref, t.ref, -100, None, C.byref(o[1])) == 1
    for tail in ((t5, g), (None, g), (lse, g2), (lse, None)):
        assert L.vb_linear_cross_entropy_backward(x.ref, w.ref, t.ref, -100, *[r(i) for i in tail], C.byref(o[0]), C.byref(o[1])) == 1
    assert vb.memory_stats()["live_slots"] == before


def test_the_same_bits_twice(vb):
    D = [Dev(vb, a) for a in (rnd(30, 515, 136), rnd(31, 1111, 136, scale=0.3), np.arange(515, dtype=np.float32))]
    one = Dev(vb, np.ones(1, np.float32))

    def run():
        loss, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
        return [loss, lse] + outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, lse), one, n=2)
    for a, b in zip(run(), run()):
        assert (a == b).all()


@pytest.mark.parametrize("n,d,v", [(2, 40, 20000), (1, 129, 9001), (70, 260, 5000), (5000, 64, 10), (3000, 33, 70)])
def test_long_sums_of_few_tiles(vb, n, d, v):
    """dx sums over the vocabulary and dW over the rows: with few rows, or few classes, they are formed in parts."""
    x, w = rnd(40, n, d), rnd(41, v, d, scale=2.0 / np.sqrt(d))
    t = np.random.default_rng(42).integers(0, v, n).astype(np.float32)
    (lse, loss, gx, gw), (e_lse, e_loss, egx, egw) = truth(x, w, t, -100, 1.5)
    D = [Dev(vb, a) for a in (x, w, t)]
    got_loss, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    assert (np.abs(got_lse - lse) <= e_lse).all() and abs(got_loss[0] - loss) <= e_loss
    rest = (*D, -100, Dev(vb, got_lse), Dev(vb, np.array([1.5], np.float32)))
    got = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *rest, n=2)
    vb.check_errors()
    assert (np.abs(got[0] - gx) <= egx).all() and (np.abs(got[1] - gw) <= egw).all()
    for a, b in zip(got, outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *rest, n=2)):
        assert (a == b).all()


@pytest.mark.parametrize("n,d,v", [(1, 4, 1), (2, 2048, 70), (4, 128, 64), (5, 132, 65), (8, 1024, 3000), (9, 260, 129), (16, 2048, 500), (16, 64, 20011), (17, 64, 700), (12, 2052, 100),
                                   (40, 512, 900), (150, 96, 64), (3, 516, 40000)])
def test_few_rows(vb, n, d, v):
    """Up to 16 rows, or few blocks of logits: W is read in 32 bits, once a pass.  A row that is left out may hold anything."""
    x, w = rnd(50, n, d), rnd(51, v, d, scale=2.0 / np.sqrt(d))
    t = np.random.default_rng(52).integers(0, v, n).astype(np.float32)
    if n > 2:
        t[1] = -7
    (lse, loss, gx, gw), (e_lse, e_loss, egx, egw) = truth(x, w, t, -7, -0.3)
    x0 = x.copy()
    if n > 2:
        x[1] = np.nan
    D = [Dev(vb, a) for a in (x, w, t)]
    live = t != -7
    got_loss, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -7, n=2)
    assert (np.abs(got_lse - lse) <= e_lse)[live].all() and abs(got_loss[0] - loss) <= e_loss
    rest = (*D, -7, Dev(vb, got_lse), Dev(vb, np.array([-0.3], np.float32)))
    got = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *rest, n=2)
    vb.check_errors()
    assert (np.abs(got[0] - gx) <= egx).all() and (np.abs(got[1] - gw) <= egw).all()
    assert (got[0][~live] == 0).all() and np.isfinite(x0).all()
    L = vb.lib()
    for i, want in ((0, got[0]), (1, got[1])):      # one gradient alone, the same bits
        o = vb.VbTensor()
        args = [a.ref if isinstance(a, Dev) else a for a in rest]
        vb.vb_check(L.vb_linear_cross_entropy_backward(*args, C.byref(o) if i == 0 else None, C.byref(o) if i == 1 else None))
        a = np.empty(o.shape, np.float32)
        vb.vb_check(L.vb_read(o.slot, 0, a.ctypes.data_as(vb.c_f32p), a.size))
        L.vb_release(o.slot, None)
        assert (a == want).all()


@pytest.mark.parametrize("n,d,v", [(17, 64, 700), (33, 128, 512), (100, 1024, 300), (500, 260, 200), (600, 36, 60), (18, 2048, 1), (150, 68, 64)])
def test_gradients_of_few_blocks(vb, n, d, v):
    """Several groups of rows and so few columns that one wave of blocks has them all; rows left out hold NaN."""
    x, w = rnd(60, n, d), rnd(61, v, d, scale=2.0 / np.sqrt(d))
    t = np.random.default_rng(62).integers(0, v, n).astype(np.float32)
    t[1::5] = -1
    (lse, loss, gx, gw), (e_lse, e_loss, egx, egw) = truth(x, w, t, -1, 2.0)
    x[1::5] = np.nan
    D = [Dev(vb, a) for a in (x, w, t)]
    got_loss, got_lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -1, n=2)
    assert (np.abs(got_lse - lse) <= e_lse)[t != -1].all() and abs(got_loss[0] - loss) <= e_loss
    rest = (*D, -1, Dev(vb, got_lse), Dev(vb, np.array([2.0], np.float32)))
    got = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *rest, n=2)
    vb.check_errors()
    assert (np.abs(got[0] - gx) <= egx).all() and (np.abs(got[1] - gw) <= egw).all()
    for a, b in zip(got, outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *rest, n=2)):
        assert (a == b).all()
