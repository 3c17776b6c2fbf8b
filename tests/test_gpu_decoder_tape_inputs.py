"""Tape nodes of the decoder operators whose only input that wants a gradient is one that has none (targets, offsets, positions)."""
import numpy as np
import pytest

from tests.decoder_ops_util import rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def calls(vb, wanted):
    """name -> a call whose second kind of input (the one without a gradient) wants one, its other inputs where `wanted`"""
    def t(a, grad=False):
        return vb.Tensor.from_numpy(np.asarray(a, np.float32), grad)
    x, w, targets = t(rnd(1, 20, 16), wanted), t(rnd(2, 30, 16), wanted), t(np.arange(20), True)
    q, k, v, starts = t(rnd(3, 40, 4, 16), wanted), t(rnd(4, 40, 2, 16), wanted), t(rnd(5, 40, 2, 16), wanted), t([0, 13, 40], True)
    n, positions = t(np.ones(16), wanted), t(np.arange(40), True)
    return {"loss": (lambda: x.linear_cross_entropy(w, targets), (x, w), targets),
            "attention": (lambda: q.segment_attention(k, v, starts).reshape([1, 40 * 4 * 16]).sum(1), (q, k, v), starts),
            "norm_rope": (lambda: q.norm_rope(n, positions).reshape([1, 40 * 4 * 16]).sum(1), (q, n), positions)}


@pytest.mark.parametrize("name", ["loss", "attention", "norm_rope"])
@pytest.mark.parametrize("wanted", [False, True])
def test_an_input_without_a_gradient_may_ask_for_one(vb, name, wanted):
    vb.zero_gradients(); vb.reset_active_tape()
    call, inputs, asks = calls(vb, wanted)[name]
    call().backward()
    vb.check_errors()
    assert asks.grad() is None
    for x in inputs:
        assert (x.grad() is not None) == wanted
        if wanted:
            assert np.isfinite(x.grad().contiguous().numpy()).all()
