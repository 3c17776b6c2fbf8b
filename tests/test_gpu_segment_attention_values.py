"""Attention over packed segments where values of one row or text could reach others, and offsets at the ends of their range."""
import ctypes as C

import numpy as np
import pytest

from tests.decoder_ops_util import Dev, outputs, rnd, segment_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def forward(vb, q, k, v, starts, scale):
    return outputs(vb, vb.lib().vb_segment_attention, Dev(vb, q), Dev(vb, k), Dev(vb, v), Dev(vb, starts), scale, n=2)


def gradients(vb, q, k, v, starts, scale, out, lse, g):
    return outputs(vb, vb.lib().vb_segment_attention_backward, Dev(vb, q), Dev(vb, k), Dev(vb, v), Dev(vb, starts), scale, Dev(vb, out), Dev(vb, lse), Dev(vb, g), n=3)


@pytest.mark.parametrize("dk", [64, 80])
@pytest.mark.parametrize("row", [0, 150, 200, 201, 299])      # first of a text, inside one, a text of one token, first of the next, last
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_gradient_that_is_not_finite_is_not_lost(vb, dk, row, value):
    T, hq, hk, starts, c, head = 300, 4, 2, np.array([0, 200, 201, 300], np.float32), 5, 3
    q, k, v, g = rnd(1, T, hq, dk), rnd(2, T, hk, dk), rnd(3, T, hk, dk), rnd(4, T, hq, dk)
    out, lse = forward(vb, q, k, v, starts, 0.2)
    assert out[row, head, c] != 0
    g[row, head, c] = 0
    clean = gradients(vb, q, k, v, starts, 0.2, out, lse, g)
    g[row, head, c] = value
    dq, dk_, dv = gradients(vb, q, k, v, starts, 0.2, out, lse, g)
    vb.check_errors()
    begin = int(starts[np.searchsorted(starts, row, side="right") - 1])
    seen = np.zeros((T, hk), bool)
    seen[begin:row + 1, head // 2] = True
    mine = np.zeros((T, hq), bool)
    mine[row, head] = True
    assert np.isnan(dq[mine]).all() and np.isnan(dk_[seen]).all() and np.isnan(dv[seen]).all()
    # what the row does not enter is what it was
    for got, want, entered in ((dq, clean[0], mine), (dk_, clean[1], seen), (dv, clean[2], seen)):
        assert (got[~entered] == want[~entered]).all()


def bounded_by_text(q, k, v, starts, scale, g):
    """Gradients in 64 bits and bounds, every text by itself: what one text holds has no place in another's bound, but for the exponent that the
    planes of a tile of 128 rows share: a value of a tile is good to 2^-40 of the tile's largest."""
    T = len(q)
    vals, errs = [np.zeros(a.shape) for a in (q, k, v)], [np.zeros(a.shape) for a in (q, k, v)]
    a = np.abs
    group = q.shape[1] // k.shape[1]
    for b, e in zip(starts[:-1].astype(int), starts[1:].astype(int)):
        (_, _, *got), (_, _, *err) = segment_attention(q[b:e], k[b:e], v[b:e], [0, e - b], scale, g[b:e], err=True)
        tiles = slice(b // 128 * 128, min(T, -(-e // 128) * 128))
        shared = {name: 2.0 ** -40 * a(x[tiles]).max() for name, x in (("q", q), ("k", k), ("v", v), ("g", g))}
        n, dk = e - b, q.shape[2]
        # dS = p (do . v - do . o): v and, through o, its average each off by the shared step, do too; p is off by the scores' error
        g1, v1 = a(g[b:e]).sum(-1).max(), a(v[b:e]).sum(-1).max()
        off = scale * (a(q[b:e]).sum(-1).max() * shared["k"] + a(k[b:e]).sum(-1).max() * shared["q"])
        ds = scale * (2 * g1 * shared["v"] + 2 * v1 * shared["g"] + 4 * off * g1 * a(v[b:e]).max())      # over p, which sums to 1 over keys, to n at most over queries
        ds_size = scale * 2 * g1 * a(v[b:e]).max()
        errs[0][b:e] = err[0] + ds * a(k[b:e]).max() + ds_size * shared["k"]
        errs[1][b:e] = err[1] + group * n * (ds * a(q[b:e]).max() + ds_size * shared["q"])
        errs[2][b:e] = err[2] + group * n * (2 * off * a(g[b:e]).max() + shared["g"])
        for to, x in zip(vals, got):
            to[b:e] = x
    return vals, errs


@pytest.mark.parametrize("starts,power", [([0, 256, 600], 30), ([0, 384, 512, 900], 30), ([0, 300, 600], 20), ([0, 40, 90, 400], 20)])
@pytest.mark.parametrize("hq,hk,dk", [(4, 2, 64), (2, 1, 96)])
@pytest.mark.parametrize("large", [0, 1])
def test_values_of_one_text_do_not_take_bits_from_another(vb, starts, power, hq, hk, dk, large):
    """The values of one text 2^power times as large as the others' (by more than 2^20 where no tile of 128 rows holds rows of both)."""
    starts = np.array(starts, np.float32)
    T = int(starts[-1])
    q, k, v = rnd(11, T, hq, dk), rnd(12, T, hk, dk), rnd(13, T, hk, dk)
    g = rnd(14, T, hq, dk)
    g = (g / np.sqrt((g * g).sum(-1, keepdims=True))).astype(np.float32)
    b, e = int(starts[large]), int(starts[large + 1])
    v[b:e] *= np.float32(2.0 ** power)
    out, lse = forward(vb, q, k, v, starts, dk ** -0.5)
    got = gradients(vb, q, k, v, starts, dk ** -0.5, out, lse, g)
    vb.check_errors()
    vals, errs = bounded_by_text(q, k, v, starts, dk ** -0.5, g)
    for x, want, err, name in zip(got, vals, errs, ("dq", "dk", "dv")):
        assert (np.abs(x - want) <= err).all(), (name, (np.abs(x - want) / np.maximum(err, 1e-300)).max())


@pytest.mark.parametrize("T", [2 ** 23 + 2, 2 ** 24])
def test_the_last_offset_of_a_long_pack(vb, T):
    """Offsets of which neighbours are one step of f32 apart: T is a whole number of them, T + 1 rounds to one as well."""
    a = rnd(21, 300)
    slots = []

    def far(tail):      # [T, 1, 1], zeros with `tail` in its last rows
        slot = C.c_uint32()
        vb.vb_check(vb.lib().vb_alloc(T, 1, C.byref(slot)))
        vb.vb_check(vb.lib().vb_write(slot.value, T - tail.size, tail.ctypes.data_as(vb.c_f32p), tail.size))
        vb.sync()
        slots.append(slot.value)
        return vb.VbTensor.contiguous(slot.value, (T, 1, 1))
    x = far(a)
    out = vb.VbTensor()
    starts = Dev(vb, np.array([T - 300, T - 100, T], np.float32))
    vb.vb_check(vb.lib().vb_segment_attention(C.byref(x), C.byref(x), C.byref(x), starts.ref, 1.0, C.byref(out), None))
    vb.check_errors()
    got = np.empty(300, np.float32)
    vb.vb_check(vb.lib().vb_read(out.slot, T - 300, got.ctypes.data_as(vb.c_f32p), 300))
    vb.lib().vb_release(out.slot, None)
    want = np.concatenate([segment_attention(a[s, None, None], a[s, None, None], a[s, None, None], [0, n], 1.0, err=False)[0][:, 0, 0]
                           for s, n in ((slice(0, 200), 200), (slice(200, 300), 100))])
    assert np.abs(got - want).max() <= 200 * 2.0 ** -24 * np.abs(a).max() * (1 + np.abs(a).max() ** 2)      # (57 U of a score of at most max^2, 80 U of the sum)
    bad = Dev(vb, np.array([T - 300, T - 100, T + 2], np.float32))
    vb.vb_check(vb.lib().vb_segment_attention(C.byref(x), C.byref(x), C.byref(x), bad.ref, 1.0, C.byref(out), None))
    vb.lib().vb_release(out.slot, None)
    with pytest.raises(vb.VearoError):
        vb.check_errors()
    for s in slots:
        vb.lib().vb_release(s, None)


@pytest.mark.parametrize("starts,fine", [([0], True), ([0, 0, 0], True), ([0, 5], False), ([-3, 0], False), ([0, np.nan], False)])
def test_offsets_of_no_rows(vb, starts, fine):
    x = np.zeros((0, 2, 16), np.float32)
    out, lse = forward(vb, x, x, x, np.array(starts, np.float32), 0.5)
    assert out.shape == (0, 2, 16) and lse.shape == (2, 0)
    if fine:
        vb.check_errors()
    else:
        with pytest.raises(vb.VearoError):
            vb.check_errors()
    grads = gradients(vb, x, x, x, np.array(starts, np.float32), 0.5, out, lse, x)
    assert all(g.shape == x.shape for g in grads)
    if fine:
        vb.check_errors()
    else:
        with pytest.raises(vb.VearoError):
            vb.check_errors()
