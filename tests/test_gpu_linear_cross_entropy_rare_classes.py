"""Gradients of the vocabulary projection for classes that no row holds probable: every row of dW is good relative to itself."""
import numpy as np
import pytest

from tests.decoder_ops_util import Dev, U, outputs, rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def run(vb, x, w, t, g=1.0):
    D = [Dev(vb, a) for a in (x, w, t)]
    _, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    return outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, Dev(vb, lse), Dev(vb, np.array([g], np.float32)), n=2)


def truth(x, w, t, g=1.0):
    """dx and dW in 64 bits and bounds of every element.  A class's dz is held relative to the largest of the class in 128 rows."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    n, d, v = len(x), x.shape[1], len(w)
    live = t != -100
    at = np.arange(n), np.where(live, t, 0).astype(np.int64)
    z = x @ w.T
    top = z.max(1, keepdims=True)
    lse = top + np.log(np.exp(z - top).sum(1, keepdims=True))
    p = np.exp(z - lse)
    dz = p.copy()
    dz[at] -= 1
    scale = live[:, None] * g / max(1, live.sum())
    # a logit: 57 U of its products' absolute sum for pairs of halves and truncation within a run of 128, an addition a run; its row's lse the
    # average of such errors; the exponent's argument rounded twice, the exponential good to 4 U; dz in two halves 2^-22, 1 - p one rounding of 1
    ez = (59 + d / 128) * U * (np.abs(x) @ np.abs(w).T)
    rel = ez + ez.max(1, keepdims=True) + (4 + 2 * (np.abs(z) + np.abs(lse) + 20) + v / 128 + 136 + 8 + 2 * np.abs(lse)) * U + 2.0 ** -22
    e = p * rel
    e[at] += 2 * U
    dz, e = dz * scale, e * np.abs(scale)
    # a plane's least step: 2^-40 of the largest of 128 rows of a class (dW), 2^-38 of a probability of 1 (dx); of x, 2^-40 of the largest of a 128 x 128 block
    step = np.concatenate([np.broadcast_to(2.0 ** -39 * np.abs(dz[i:i + 128]).max(0), dz[i:i + 128].shape) for i in range(0, n, 128)])
    product = lambda k, size: (57 + k / 128 + 6) * U * size  # noqa: E731
    egw = (e + step).T @ np.abs(x) + product(n, np.abs(dz).T @ np.abs(x)) + 2.0 ** -39 * np.abs(x).max() * np.abs(dz).sum(0)[:, None]
    egx = (e + 2.0 ** -38 * np.abs(scale)) @ np.abs(w) + product(v, np.abs(dz) @ np.abs(w))
    return dz @ w, dz.T @ x, egx, egw


def improbable(seed, n, d, v, depths):
    """x with a first component of 4; classes v // 2 .. take turns at being e^-depth as probable as the others, in every row."""
    x, w = rnd(seed, n, d), rnd(seed + 1, v, d, scale=0.5 * d ** -0.5)
    x[:, 0] = 4
    w[:, 0] = 0
    for i, c in enumerate(range(v // 2, v)):
        w[c, 0] = -depths[i % len(depths)] / 4
    t = np.random.default_rng(seed + 2).integers(0, v // 2, n).astype(np.float32)
    return x, w, t


@pytest.mark.parametrize("n,d,v", [(17, 64, 12000), (300, 64, 700), (512, 96, 1500), (1000, 48, 333)])
@pytest.mark.parametrize("ignored", [0.0, 0.3])
def test_rows_of_improbable_classes(vb, n, d, v, ignored):
    depths = [10, 20, 25, 30, 45, 60]
    x, w, t = improbable(1, n, d, v, depths)
    t[np.random.default_rng(4).random(n) < ignored] = -100
    gx, gw, egx, egw = truth(x, w, t)
    a, b = run(vb, x, w, t)
    vb.check_errors()
    assert (np.abs(b - gw) <= egw).all(), (np.abs(b - gw) / egw).max()
    assert (np.abs(a - gx) <= egx).all()
    # and what that comes to: the bound's largest part is the error of a logit of -60, its own and once more in the row's lse, 2 x 57 U x 62
    own = np.linalg.norm(b - gw, axis=1) / np.linalg.norm(gw, axis=1)
    assert own.max() <= 4e-4, own.max()


def test_a_class_that_is_one_rows_target(vb):
    """Improbable everywhere, the target of a few rows: those 128 rows hold the class at 1, the others at its own size."""
    x, w, t = improbable(10, 700, 64, 900, [40])
    t[[5, 640]] = 500, 899
    gx, gw, egx, egw = truth(x, w, t)
    a, b = run(vb, x, w, t)
    assert (np.abs(b - gw) <= egw).all() and (np.abs(a - gx) <= egx).all()


@pytest.mark.parametrize("n", [130, 1000])
def test_probabilities_far_below_the_least_normal_number(vb, n):
    """e^-200 as probable: nothing, or next to it, and never NaN."""
    x, w, t = improbable(20, n, 64, 700, [80, 100, 200, 1000])
    a, b = run(vb, x, w, t)
    assert np.isfinite(a).all() and np.isfinite(b).all() and (np.abs(b[-4:]) <= 1e-30).all()


def test_one_gradient_alone_is_the_same(vb):
    import ctypes as C
    x, w, t = improbable(30, 400, 64, 1000, [0, 25])
    D = [Dev(vb, a) for a in (x, w, t)]
    _, lse = outputs(vb, vb.lib().vb_linear_cross_entropy, *D, -100, n=2)
    one, lse = Dev(vb, np.ones(1, np.float32)), Dev(vb, lse)
    both = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, lse, one, n=2)
    (only_w,) = outputs(vb, vb.lib().vb_linear_cross_entropy_backward, *D, -100, lse, one, None, n=1)
    assert (only_w == both[1]).all()
    o = vb.VbTensor()
    vb.vb_check(vb.lib().vb_linear_cross_entropy_backward(*[a.ref for a in D], -100, lse.ref, one.ref, C.byref(o), None))
    only_x = np.empty(x.shape, np.float32)
    vb.vb_check(vb.lib().vb_read(o.slot, 0, only_x.ctypes.data_as(vb.c_f32p), only_x.size))
    vb.lib().vb_release(o.slot, None)
    assert (only_x == both[0]).all()
