"""The decoder operators on tensors of more than 2^31 elements, looked at in their last rows: what lies before them is zero."""
import ctypes as C

import numpy as np
import pytest

from tests.decoder_ops_util import Dev, U, rnd, segment_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


class Far:
    """A tensor of zeros with `tail` in its last rows."""

    def __init__(self, vb, shape, tail):
        self.vb, n = vb, int(np.prod(shape, dtype=np.int64))
        slot = C.c_uint32()
        vb.vb_check(vb.lib().vb_alloc(n, 1, C.byref(slot)))
        vb.vb_check(vb.lib().vb_write(slot.value, n - tail.size, np.ascontiguousarray(tail).ctypes.data_as(vb.c_f32p), tail.size))
        vb.sync()
        self.desc = vb.VbTensor.contiguous(slot.value, shape)

    def __del__(self):
        self.vb.lib().vb_release(self.desc.slot, None)

    @property
    def ref(self):
        return C.byref(self.desc)


def last(vb, t, rows):
    """The last rows of an output, which is released."""
    shape = (rows,) + tuple(t.shape[1:])
    a = np.empty(shape, np.float32)
    vb.vb_check(vb.lib().vb_read(t.slot, int(np.prod(t.shape, dtype=np.int64)) - a.size, a.ctypes.data_as(vb.c_f32p), a.size))
    vb.lib().vb_release(t.slot, None)
    return a


def test_segment_attention(vb):
    T, hq, dk, n = 140000, 128, 128, 150
    q, k, v, g = rnd(1, n, hq, dk), rnd(2, n, 1, dk), rnd(3, n, 1, dk), rnd(4, n, hq, dk, scale=0.01)
    starts = np.concatenate([np.arange(0, T - n, 100), [T - n, T - 60, T]]).astype(np.float32)
    D = [Far(vb, (T, h, dk), a) for h, a in ((hq, q), (1, k), (1, v))] + [Dev(vb, starts)]
    o = [vb.VbTensor() for _ in range(5)]
    at = [C.byref(x) for x in o]
    vb.vb_check(vb.lib().vb_segment_attention(*[d.ref for d in D], 0.1, at[0], at[1]))
    G = Far(vb, (T, hq, dk), g)
    vb.vb_check(vb.lib().vb_segment_attention_backward(*[d.ref for d in D], 0.1, at[0], at[1], G.ref, *at[2:]))
    vb.check_errors()
    vals, errs = segment_attention(q, k, v, [0, n - 60, n], 0.1, g, err=True)
    vb.lib().vb_release(o[1].slot, None)
    for x, want, e in ((o[0], vals[0], errs[0]), (o[2], vals[2], errs[2]), (o[3], vals[3], errs[3]), (o[4], vals[4], errs[4])):
        assert (np.abs(last(vb, x, n) - want) <= e).all()


def test_qk_norm_rope(vb):
    T, h, dk, n = 140000, 128, 128, 3
    x, g, w = rnd(5, n, h, dk), rnd(6, n, h, dk), 1 + rnd(7, dk, scale=0.1)
    pos = np.zeros(T, np.float32)      # (not turned: cosine 1, sine 0)
    X, G, W, P = Far(vb, (T, h, dk), x), Far(vb, (T, h, dk), g), Dev(vb, w), Dev(vb, pos)
    o = [vb.VbTensor() for _ in range(3)]
    at = [C.byref(i) for i in o]
    L, f = vb.lib(), C.c_float
    vb.vb_check(L.vb_qk_norm_rope(X.ref, None, W.ref, None, P.ref, f(1e4), dk, 0, f(1e-6), at[0], None))
    vb.vb_check(L.vb_qk_norm_rope_backward(X.ref, None, W.ref, None, P.ref, f(1e4), dk, 0, f(1e-6), G.ref, None, at[1], None, at[2], None))
    x, g, w = x.astype(np.float64), g.astype(np.float64), w.astype(np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
    xh, gw = x * r, g * w
    # a sum of 128 squares in 32 bits, a root, a quotient and three products: some 30 U; the gradient's inner sum over 128 terms adds as many of its absolute sum
    assert (np.abs(last(vb, o[0], n) - xh * w) <= 40 * U * np.abs(xh * w) + 1e-30).all()
    want = r * (gw - xh * (gw * xh).mean(-1, keepdims=True))
    assert (np.abs(last(vb, o[1], n) - want) <= 80 * U * r * (np.abs(gw) + np.abs(xh) * np.abs(gw * xh).mean(-1, keepdims=True))).all()
    sums = (g * xh).sum((0, 1))
    assert (np.abs(last(vb, o[2], dk) - sums) <= (40 + 384) * U * np.abs(g * xh).sum((0, 1))).all()


@pytest.mark.parametrize("n", [2, 20])
def test_linear_cross_entropy(vb, n):
    d, v, m = 2048, 1100000, 40
    x, w = rnd(8, n, d), rnd(9, m, d, scale=d ** -0.5)
    t = np.full(n, v - 3, np.float32)
    t[0] = 5
    D = [Dev(vb, x), Far(vb, (v, d), w), Dev(vb, t)]
    o = [vb.VbTensor() for _ in range(4)]
    at = [C.byref(i) for i in o]
    L = vb.lib()
    vb.vb_check(L.vb_linear_cross_entropy(*[a.ref for a in D], -100, at[0], at[1]))
    one = Dev(vb, np.ones(1, np.float32))
    vb.vb_check(L.vb_linear_cross_entropy_backward(*[a.ref for a in D], -100, at[1], one.ref, at[2], at[3]))
    vb.check_errors()
    x, w = x.astype(np.float64), w.astype(np.float64)
    z = x @ w.T
    lse = np.log((v - m) + np.exp(z).sum(1))
    # a logit: 73 U of sum |x w|; the sum of exponentials and its logarithm: v / 128 / 148 additions of nearly equal numbers a step, 600 U are plenty
    ez = 73 * U * (np.abs(x) @ np.abs(w).T)
    assert (np.abs(last(vb, o[1], n) - lse) <= ez.max() + 600 * U).all()
    dz = np.exp(z - lse[:, None]) / n
    dz[1:, m - 3] -= 1 / n
    e = (dz + (np.arange(m) == m - 3) / n) * (2 * ez.max() + 1300 * U) + 4 * U * np.abs(dz) + 2.0 ** -38 / n
    assert (np.abs(last(vb, o[3], m) - dz.T @ x) <= e.T @ np.abs(x) + 80 * U * (np.abs(dz).T @ np.abs(x))).all()
    assert (np.abs(last(vb, o[2], n) - dz @ w) <= e @ np.abs(w) + (80 + v / 128 / 8) * U * (np.abs(dz) @ np.abs(w))).all()
    vb.lib().vb_release(o[0].slot, None)
