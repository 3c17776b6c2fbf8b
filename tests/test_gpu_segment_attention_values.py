"""Attention over packed segments where values of one row or text could reach others, and offsets at the ends of their range."""
import ctypes as C

import numpy as np
import pytest

from tests.decoder_ops_util import Dev, outputs, rnd

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
