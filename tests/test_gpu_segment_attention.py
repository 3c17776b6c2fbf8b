"""vb_segment_attention and its backward against their definition in 64 bits: segment layouts, groups, head sizes, views, refusals."""
import ctypes as C

import numpy as np
import pytest

from tests.decoder_ops_util import Dev, U, outputs, rnd, segment_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def run(vb, q, k, v, starts, scale, g=None, view="whole"):
    D = [Dev(vb, a, view) for a in (q, k, v)] + [Dev(vb, np.asarray(starts, np.float32))]
    o, lse = outputs(vb, vb.lib().vb_segment_attention, *D, scale, n=2)
    if g is None:
        return o, lse
    return [o, lse] + outputs(vb, vb.lib().vb_segment_attention_backward, *D, scale, Dev(vb, o, view), Dev(vb, lse), Dev(vb, g, view), n=3)


def check(got, vals, errs):
    for name, a, b, e in zip(("out", "lse", "dq", "dk", "dv"), got, vals, errs):
        dead = np.isneginf(b)
        assert (np.isneginf(a) == dead).all(), name
        over = np.where(dead, 0, np.abs(np.where(dead, 0, a) - np.where(dead, 0, b)) - e)
        assert (over <= 0).all(), "%s: %.3g over its bound at %s" % (name, over.max(), np.unravel_index(over.argmax(), over.shape))


CASES = [  # starts (the last one may lie before T), T, query heads, key heads, head size
    ([0, 1], 1, 1, 1, 64), ([0, 1], 1, 2, 1, 1), ([0, 2], 2, 2, 2, 7), ([0, 128], 128, 1, 1, 64), ([0, 129], 129, 2, 1, 64), ([0, 300], 300, 4, 2, 64),
    ([0, 5, 5, 9, 130, 131, 260], 260, 2, 1, 64), ([0, 100, 200], 237, 3, 3, 64), ([7, 60, 190], 200, 2, 2, 64), ([0], 70, 1, 1, 64),
    ([0, 257], 257, 2, 2, 128), ([0, 63, 64, 200, 390], 391, 4, 1, 128), ([0, 150], 150, 2, 1, 80), ([0, 150], 150, 2, 1, 96), ([0, 90, 333], 333, 3, 1, 40),
    ([0, 70], 70, 6, 2, 3), ([0, 140, 400], 400, 8, 2, 48), ([0] + list(range(1, 151)), 150, 2, 1, 64), ([0, 640], 640, 2, 1, 64), ([0, 512], 600, 2, 1, 128),
    ([0, 70, 700], 700, 2, 2, 33),
]


@pytest.mark.parametrize("starts,T,hq,hk,dk", CASES)
def test_against_the_definition(vb, starts, T, hq, hk, dk):
    q, k, v, g = rnd(1, T, hq, dk, scale=1.3), rnd(2, T, hk, dk, scale=1.3), rnd(3, T, hk, dk), rnd(4, T, hq, dk, scale=0.01)
    scale = 1.0 / np.sqrt(dk)
    got = run(vb, q, k, v, starts, scale, g)
    vb.check_errors()
    check(got, *segment_attention(q, k, v, starts, scale, g, err=True))


def test_large_scores_and_tiny_values(vb):
    """Scores of some hundreds (one key takes a row's whole weight), values and gradients near 1e-18."""
    T = 200
    q, k, v, g = rnd(5, T, 2, 64, scale=20), rnd(6, T, 1, 64, scale=20), rnd(7, T, 1, 64, scale=1e-18), rnd(8, T, 2, 64, scale=1e-12)
    check(run(vb, q, k, v, [0, 150, 200], 0.1, g), *segment_attention(q, k, v, [0, 150, 200], 0.1, g, err=True))


def test_blocks_of_unequal_size(vb):
    """Keys and values that differ by 2^20 from one 128-row block to the next: each block has an exponent of its own."""
    T = 400
    grow = (2.0 ** (10 * (np.arange(T) // 128)))[:, None, None].astype(np.float32)
    q, k, v, g = rnd(9, T, 1, 64), rnd(10, T, 1, 64) / grow, rnd(11, T, 1, 64) * grow, rnd(12, T, 1, 64)
    check(run(vb, q, k, v, [0, T], 0.125, g), *segment_attention(q, k, v, [0, T], 0.125, g, err=True))


def test_zero_inputs(vb):
    T = 130
    z, v, g = np.zeros((T, 2, 64), np.float32), rnd(13, T, 2, 64), rnd(14, T, 2, 64)
    check(run(vb, z, z, v, [0, T], 0.125, g), *segment_attention(z, z, v, [0, T], 0.125, g, err=True))
    got = run(vb, z, z, z, [0, T], 0.125, z)
    assert all((np.isfinite(a)).all() for a in got) and (got[0] == 0).all() and all((a == 0).all() for a in got[2:])


def test_other_segments_never_matter(vb):
    """Infinities and NaN in a segment stay there, and so do those behind the last segment; those ahead of a row do not reach it."""
    T = 300
    q, k, v, g = rnd(15, T, 2, 64), rnd(16, T, 1, 64), rnd(17, T, 1, 64), rnd(18, T, 2, 64)
    starts = [0, 100, 190, 290]
    want = run(vb, q, k, v, starts, 0.125, g)
    for x in (q, k, v, g):
        x[100:190] = np.nan
        x[290:] = np.inf
    got = run(vb, q, k, v, starts, 0.125, g)
    rows = np.r_[0:100, 190:290]
    for i, (a, b) in enumerate(zip(got, want)):
        a, b = (a[:, rows], b[:, rows]) if i == 1 else (a[rows], b[rows])
        assert np.isfinite(a).all() and np.abs(a - b).max() <= 1e-4 * np.abs(b).max()
    assert (got[0][290:] == 0).all() and all((x[290:] == 0).all() for x in got[2:])
    q, k, v = rnd(15, T, 2, 64), rnd(16, T, 1, 64), rnd(17, T, 1, 64)
    k[250], v[251] = np.inf, np.nan
    o, lse = run(vb, q, k, v, [0, T], 0.125)
    assert np.isfinite(o[:250]).all() and np.isfinite(lse[:, :250]).all()


def test_offsets_out_of_order_or_range_are_reported(vb):
    q, k, v, g = rnd(20, 50, 2, 64), rnd(21, 50, 1, 64), rnd(22, 50, 1, 64), rnd(23, 50, 2, 64)
    for starts in ([0, 30, 20, 50], [0, 51], [-3, 50], [0, np.nan, 50], [0, 1e30], [-1e30, 50], [50, 0], [0, np.inf, 50, -np.inf]):
        run(vb, q, k, v, starts, 0.125, g)
        with pytest.raises(vb.VearoError):
            vb.check_errors()
    run(vb, q, k, v, [0, 50], 0.125)
    vb.check_errors()


@pytest.mark.parametrize("view", ["strided", "odd", "turned"])
@pytest.mark.parametrize("dk", [64, 48, 128, 10])
def test_views_give_the_same_bits(vb, view, dk):
    T = 140
    q, k, v, g = rnd(24, T, 4, dk), rnd(25, T, 2, dk), rnd(26, T, 2, dk), rnd(27, T, 4, dk)
    for a, b in zip(run(vb, q, k, v, [0, 60, 135], 0.2, g), run(vb, q, k, v, [0, 60, 135], 0.2, g, view)):
        assert (a == b).all()


def test_gradient_against_differences(vb):
    T, dk = 12, 16
    q, k, v, g = rnd(28, T, 2, dk), rnd(29, T, 1, dk), rnd(30, T, 1, dk), rnd(31, T, 2, dk)
    d = [rnd(32 + i, *x.shape) for i, x in enumerate((q, k, v))]
    got = run(vb, q, k, v, [0, 5, 12], 0.25, g)

    def f(step):
        o, _ = segment_attention(*[x.astype(np.float64) + step * y for x, y in zip((q, k, v), d)], [0, 5, 12], 0.25)
        return (o * g).sum()
    h = 1e-4
    want = (f(h) - f(-h)) / (2 * h)
    have = sum((a.astype(np.float64) * y).sum() for a, y in zip(got[2:], d))
    # the difference's own error is h^2 times third derivatives, of order one for each of 384 terms; the gradients' is some hundred U a term
    assert abs(have - want) <= 1e-8 * 384 * 10 + 768 * 200 * U


def test_the_same_bits_twice_and_no_tokens(vb):
    q, k, v, g = rnd(40, 500, 4, 64), rnd(41, 500, 2, 64), rnd(42, 500, 2, 64), rnd(43, 500, 4, 64)
    for a, b in zip(run(vb, q, k, v, [0, 123, 500], 0.125, g), run(vb, q, k, v, [0, 123, 500], 0.125, g)):
        assert (a == b).all()
    e = np.zeros((0, 2, 64), np.float32)
    got = run(vb, e, e, e, [0], 0.125, e)
    assert got[0].shape == (0, 2, 64) and got[1].shape == (2, 0)


def test_refusals_leave_no_slot_behind(vb):
    q, k, v, s = (Dev(vb, rnd(50, 6, 4, 64)), Dev(vb, rnd(51, 6, 2, 64)), Dev(vb, rnd(52, 6, 2, 64)), Dev(vb, np.array([0, 6], np.float32)))
    k3, k5, k32, flat = Dev(vb, rnd(53, 6, 3, 64)), Dev(vb, rnd(54, 5, 2, 64)), Dev(vb, rnd(55, 6, 2, 32)), Dev(vb, rnd(56, 6, 64))
    wide, s2, s0 = Dev(vb, rnd(57, 6, 2, 129)), Dev(vb, np.zeros((1, 2), np.float32)), Dev(vb, np.zeros(0, np.float32))
    lse, bad_lse = Dev(vb, np.zeros((4, 6), np.float32)), Dev(vb, np.zeros((6, 4), np.float32))
    L = vb.lib()
    o = [vb.VbTensor() for _ in range(3)]
    r = lambda a: None if a is None else a.ref  # noqa: E731
    before = vb.memory_stats()["live_slots"]
    for a in ((None, k, v, s, 1.0), (q, None, v, s, 1.0), (q, k, None, s, 1.0), (q, k, v, None, 1.0), (q, k3, k3, s, 1.0), (q, k5, k5, s, 1.0), (q, k32, k32, s, 1.0),
              (q, k, k3, s, 1.0), (flat, k, v, s, 1.0), (wide, wide, wide, s, 1.0), (q, k, v, s2, 1.0), (q, k, v, s0, 1.0), (q, k, v, s, 0.0), (q, k, v, s, float("nan"))):
        assert L.vb_segment_attention(*[r(i) for i in a[:4]], a[4], C.byref(o[0]), C.byref(o[1])) in (1, 8), a
        assert L.vb_last_error()
    assert L.vb_segment_attention(q.ref, k.ref, v.ref, s.ref, 1.0, None, None) == 1
    for a in ((k, lse, q), (q, bad_lse, q), (q, lse, k), (None, lse, q), (q, None, q), (q, lse, None)):
        assert L.vb_segment_attention_backward(q.ref, k.ref, v.ref, s.ref, 1.0, *[r(i) for i in a], *[C.byref(x) for x in o]) == 1
    assert L.vb_segment_attention_backward(q.ref, k.ref, v.ref, s.ref, 1.0, q.ref, lse.ref, q.ref, C.byref(o[0]), None, C.byref(o[2])) == 1
    assert vb.memory_stats()["live_slots"] == before


@pytest.mark.parametrize("fill", [1e30, -3e-30, np.nan])
def test_rows_of_no_segment_may_hold_anything(vb, fill):
    """Rows before the first segment and behind the last share tiles, and so exponents, with rows that have one."""
    T, starts = 300, [9, 140, 270]
    q, k, v, g = rnd(50, T, 2, 64), rnd(51, T, 1, 64), rnd(52, T, 1, 64), rnd(53, T, 2, 64)
    for x in (q, k, v, g):
        x[:9], x[270:] = 0, 0
    want = run(vb, q, k, v, starts, 0.125, g)
    for x in (q, k, v, g):
        x[:9], x[270:] = fill, fill
    for a, b in zip(run(vb, q, k, v, starts, 0.125, g), want):
        assert (a == b).all()


def test_gradients_may_go_to_the_descriptors_of_the_inputs(vb):
    """Outputs are written to the descriptors after the last look at the inputs, whichever descriptors they are."""
    T = 60
    q, k, v, g = rnd(54, T, 4, 16), rnd(55, T, 1, 16), rnd(56, T, 1, 16), rnd(57, T, 4, 16)
    want = run(vb, q, k, v, [0, 25, T], 0.25, g)
    D = [Dev(vb, a) for a in (q, k, v, [0, 25, T], want[0], want[1], g)]
    d = [vb.VbTensor.from_buffer_copy(x.desc) for x in D[:4]]
    at = [C.byref(x) for x in d]
    vb.vb_check(vb.lib().vb_segment_attention_backward(*at, 0.25, D[4].ref, D[5].ref, D[6].ref, at[1], at[3], at[0]))
    for x, b in zip((d[1], d[3], d[0]), want[2:]):
        assert x.shape == b.shape
        a = np.empty(b.shape, np.float32)
        vb.vb_check(vb.lib().vb_read(x.slot, 0, a.ctypes.data_as(vb.c_f32p), a.size))
        vb.lib().vb_release(x.slot, None)
        assert (a == b).all()


@pytest.mark.parametrize("hq,hk,dk", [(4, 2, 64), (6, 1, 64), (6, 1, 96), (4, 4, 40)])
def test_several_heads_of_a_group_in_one_block(vb, hq, hk, dk):
    """Enough tiles that a key head's gradient is not dealt out to a block for each query head, or to fewer than all."""
    T, starts = 3300, [0, 3, 350, 351, 900, 1200, 1200, 1800, 2303, 2305, 3000, 3290]
    q, k, v, g = rnd(60, T, hq, dk, scale=1.3), rnd(61, T, hk, dk, scale=1.3), rnd(62, T, hk, dk), rnd(63, T, hq, dk, scale=0.01)
    scale = 1.0 / np.sqrt(dk)
    got = run(vb, q, k, v, starts, scale, g)
    vb.check_errors()
    check(got, *segment_attention(q, k, v, starts, scale, g, err=True))


def test_the_first_row_of_a_segment_has_no_gradient_of_its_score(vb):
    """It sees itself alone: its weight is 1, and queries and keys of texts of one token have gradients of 0, not of rounding."""
    T, starts = 7, [0, 1, 2, 5, 6]
    q, k, v, g = rnd(70, T, 8, 96, scale=3.0), rnd(71, T, 4, 96, scale=3.0), rnd(72, T, 4, 96, scale=30.0), rnd(73, T, 8, 96)
    got = run(vb, q, k, v, starts, 0.1, g)
    check(got, *segment_attention(q, k, v, starts, 0.1, g, err=True))
    assert (got[2][[0, 1, 2, 5, 6]] == 0).all() and (got[3][[0, 1, 5, 6]] == 0).all()
    assert (got[2][[3, 4]] != 0).any() and (got[4][:6] != 0).any()
    k[5, 1, 3] = np.nan                                        # (a text of one token that is not finite: NaN, as in longer ones)
    got = run(vb, q, k, v, starts, 0.1, g)
    assert np.isnan(got[0][5, 2:4]).all() and np.isnan(got[2][5, 2:4]).any(-1).all() and np.isnan(got[3][5, 1]).any() and np.isnan(got[4][5, 1]).any()
    assert all(np.isfinite(x[r]).all() for x in (got[0], *got[2:]) for r in (0, 1, 2, 3, 4))


def test_keys_broadcast_over_heads_and_rows_in_reverse(vb):
    """A view with a stride of 0 or a negative one is read in place: the same bits as its copy."""
    T, dk, starts = 200, 64, [0, 90, 200]
    q, k, g = rnd(80, T, 4, dk), rnd(81, T, 1, dk), rnd(82, T, 4, dk)
    many = np.repeat(k, 2, 1)
    want = run(vb, q, many, many, starts, 0.125, g)
    Q, K, G = Dev(vb, q[::-1]), Dev(vb, k), Dev(vb, g)
    K.desc.dims[1], K.desc.strides[1] = 2, 0
    Q.desc.offset, Q.desc.strides[0] = (T - 1) * 4 * dk, -4 * dk
    S, O, LSE = Dev(vb, np.asarray(starts, np.float32)), Dev(vb, want[0]), Dev(vb, want[1])
    got = outputs(vb, vb.lib().vb_segment_attention, Q, K, K, S, 0.125, n=2)
    got += outputs(vb, vb.lib().vb_segment_attention_backward, Q, K, K, S, 0.125, O, LSE, G, n=3)
    for a, b in zip(got, want):
        assert (a == b).all()
