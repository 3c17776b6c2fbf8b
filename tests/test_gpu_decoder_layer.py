"""The decoder-training operators together, as a layer uses them: projections, norm and rotation of queries and keys, attention over packed
segments, output projection and residual, vocabulary loss; forward and backward through the tape, against the same layer in 64 bits."""
import numpy as np
import pytest
import torch

from tests.decoder_ops_util import rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vb():
    import vearo_b200 as v
    v.init()
    return v


def layer_64(p, x, pos, starts, targets, hq, hk, dk, theta=10000.0, eps=1e-6):
    """Loss and gradients by torch on the CPU in 64 bits, attention through an explicit mask."""
    P = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in p.items()}
    X = torch.tensor(x, dtype=torch.float64, requires_grad=True)
    T = len(x)
    seg = np.searchsorted(np.asarray(starts), np.arange(T), side="right") - 1
    live = torch.tensor((seg >= 0) & (seg < len(starts) - 1))
    mask = torch.tensor((seg[:, None] == seg[None]) & (np.arange(T)[:, None] >= np.arange(T)[None])) & live[:, None] & live[None]
    ang = torch.tensor(pos, dtype=torch.float64)[:, None, None] * theta ** (-2.0 * torch.arange(dk // 2, dtype=torch.float64) / dk)

    def heads(w, h):
        return (X @ P[w].T).reshape(T, h, dk)

    def turn(y, w):
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * P[w]
        a, b = y[..., : dk // 2], y[..., dk // 2 :]
        return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
    q, k, v = turn(heads("wq", hq), "nq"), turn(heads("wk", hk), "nk"), heads("wv", hk)
    k, v = k.repeat_interleave(hq // hk, 1), v.repeat_interleave(hq // hk, 1)
    s = torch.einsum("thd,shd->hts", q, k) * dk ** -0.5
    s = s.masked_fill(~mask, -1e300)
    a = torch.softmax(s, -1) * live[None, :, None]
    o = torch.einsum("hts,shd->thd", a, v).reshape(T, hq * dk)
    h = X + o @ P["wo"].T
    z = h @ P["head"].T
    t = torch.tensor(targets)
    keep = t != -100
    loss = (torch.logsumexp(z, -1) - z.gather(1, t.clamp_min(0)[:, None])[:, 0])[keep].mean()
    loss.backward()
    return loss.item(), {**{k: v.grad.numpy() for k, v in P.items()}, "x": X.grad.numpy()}


def layer_vb(vb, p, x, pos, starts, targets, hq, hk, dk, one_launch=True, checkpointed=False):
    vb.zero_gradients(); vb.reset_active_tape()
    T, d = x.shape
    P = {k: vb.Tensor.from_numpy(v, True) for k, v in p.items()}
    X = vb.Tensor.from_numpy(x, True)
    POS, ST, TG = (vb.Tensor.from_numpy(np.asarray(a, np.float32)) for a in (pos, starts, targets))

    def block(X):
        q, k, v = (X.linear(P[w]).reshape([T, h, dk]) for w, h in (("wq", hq), ("wk", hk), ("wv", hk)))
        if one_launch:
            q, k = q.qk_norm_rope(k, P["nq"], P["nk"], POS)
        else:
            q, k = q.norm_rope(P["nq"], POS), k.norm_rope(P["nk"], POS)
        return X.add(q.segment_attention(k, v, ST).reshape([T, hq * dk]).linear(P["wo"]))
    h = vb.checkpoint(X, block) if checkpointed else block(X)
    loss = h.linear_cross_entropy(P["head"], TG)
    value = loss.numpy()[0]
    loss.backward()
    vb.check_errors()
    return value, {**{k: v.grad().contiguous().numpy() for k, v in P.items()}, "x": X.grad().contiguous().numpy()}


def case(seed, T, d, hq, hk, dk, vocab):
    p = dict(wq=rnd(seed, hq * dk, d, scale=d ** -0.5), wk=rnd(seed + 1, hk * dk, d, scale=d ** -0.5), wv=rnd(seed + 2, hk * dk, d, scale=d ** -0.5),
             wo=rnd(seed + 3, d, hq * dk, scale=(hq * dk) ** -0.5), nq=1 + rnd(seed + 4, dk, scale=0.1), nk=1 + rnd(seed + 5, dk, scale=0.1),
             head=rnd(seed + 6, vocab, d, scale=2 * d ** -0.5))
    t = np.random.default_rng(seed + 7).integers(0, vocab, T)
    t[:: 7] = -100
    return p, rnd(seed + 8, T, d), t


@pytest.mark.parametrize("T,starts,d,hq,hk,dk,vocab", [(150, [0, 40, 40, 149], 64, 4, 2, 16, 100), (300, [0, 130, 260], 128, 4, 1, 64, 333), (64, [0, 64], 96, 2, 2, 128, 50)])
def test_layer_against_64_bits(vb, T, starts, d, hq, hk, dk, vocab):
    p, x, t = case(100, T, d, hq, hk, dk, vocab)
    pos = np.arange(T) % 50
    want, grads = layer_64(p, x, pos, starts, t, hq, hk, dk)
    got, mine = layer_vb(vb, p, x, pos, starts, t, hq, hk, dk)
    # A chain of eight operators; each is within some 1e-6 of its terms' size (its own tests), the existing products within 2e-6 of theirs, and no
    # step of this layer enlarges a relative error more than tenfold: 8 x 1e-6 x 10, against the whole tensor's length
    assert abs(got - want) <= 8e-5 * abs(want)
    for k, g in grads.items():
        assert np.linalg.norm(mine[k] - g) <= 8e-5 * np.linalg.norm(g), k


def test_two_launches_and_a_checkpoint_give_the_same_gradients(vb):
    p, x, t = case(200, 140, 64, 4, 2, 32, 90)
    args = (p, x, np.arange(140), [0, 60, 140], t, 4, 2, 32)
    a, ga = layer_vb(vb, *args)
    for kw in (dict(one_launch=False), dict(checkpointed=True)):
        b, gb = layer_vb(vb, *args, **kw)
        assert a == b
        for k in ga:
            assert (ga[k] == gb[k]).all(), (kw, k)


def test_no_gradient_is_made_where_none_is_wanted(vb):
    p, x, t = case(300, 70, 64, 2, 1, 32, 40)
    vb.zero_gradients(); vb.reset_active_tape()
    X = vb.Tensor.from_numpy(x)
    head = vb.Tensor.from_numpy(p["head"], True)
    loss = X.linear_cross_entropy(head, vb.Tensor.from_numpy(t.astype(np.float32)))
    loss.backward()
    assert X.grad() is None and head.grad().shape == p["head"].shape
    q = vb.Tensor.from_numpy(rnd(310, 70, 2, 32))
    starts = vb.Tensor.from_numpy(np.array([0, 70], np.float32))
    before = vb.memory_stats()["live_slots"]
    o = q.segment_attention(q, q, starts)
    assert vb.memory_stats()["live_slots"] == before + 1       # no lse is kept
    del o


def test_an_error_names_the_call(vb):
    q, k = vb.Tensor.from_numpy(rnd(320, 8, 3, 16)), vb.Tensor.from_numpy(rnd(321, 8, 2, 16))
    with pytest.raises(vb.VearoError, match="multiple of the number of key heads"):
        q.segment_attention(k, k, vb.Tensor.from_numpy(np.array([0, 8], np.float32)))
    with pytest.raises(vb.VearoError, match="even"):
        q.norm_rope(vb.Tensor.from_numpy(np.ones(16, np.float32)), vb.Tensor.from_numpy(np.zeros(8, np.float32)), rot_dim=3)


def test_calls_are_refused_while_the_stream_is_captured(vb):
    import ctypes as C
    L = vb.lib()
    stream = C.c_void_p()
    vb.vb_check(L.vb_stream(C.byref(stream)))
    q = vb.Tensor.from_numpy(rnd(330, 8, 2, 16))
    w, pos, starts = vb.Tensor.from_numpy(np.ones(16, np.float32)), vb.Tensor.from_numpy(np.zeros(8, np.float32)), vb.Tensor.from_numpy(np.array([0, 8], np.float32))
    x, head, t = vb.Tensor.from_numpy(rnd(331, 8, 16)), vb.Tensor.from_numpy(rnd(332, 30, 16)), vb.Tensor.from_numpy(np.zeros(8, np.float32))
    vb.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(torch.cuda.ExternalStream(stream.value)):
        with torch.cuda.graph(graph, stream=torch.cuda.current_stream(), capture_error_mode="thread_local"):
            for call in (lambda: q.norm_rope(w, pos), lambda: q.segment_attention(q, q, starts), lambda: x.linear_cross_entropy(head, t)):
                with pytest.raises(vb.VearoError, match="captured"):
                    call()
    assert np.isfinite(x.linear_cross_entropy(head, t).numpy()).all()


def test_another_current_device_does_not_matter(vb):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    torch.cuda.set_device(1)
    try:
        q = vb.Tensor.from_numpy(rnd(340, 8, 2, 16))
        assert np.isfinite(q.segment_attention(q, q, vb.Tensor.from_numpy(np.array([0, 8], np.float32))).numpy()).all()
    finally:
        torch.cuda.set_device(0)


def test_one_tensor_in_every_place(vb):
    """Queries, keys and values the same tensor, one weight for both norms: its gradients add up."""
    T, h, dk, starts = 90, 2, 32, [0, 33, 90]
    x, w, r = rnd(400, T, h, dk), 1 + rnd(401, dk, scale=0.1), rnd(402, T, h, dk)
    vb.zero_gradients(); vb.reset_active_tape()
    X, W, POS = vb.Tensor.from_numpy(x, True), vb.Tensor.from_numpy(w, True), vb.Tensor.from_numpy(np.arange(T, dtype=np.float32))
    ST, R = vb.Tensor.from_numpy(np.asarray(starts, np.float32)), vb.Tensor.from_numpy(r)
    q, k = X.qk_norm_rope(X, W, W, POS)
    q.segment_attention(k, X, ST).mul(R).reshape([1, T * h * dk]).sum(1).backward()
    a = q.segment_attention(q, q, ST)      # (and in one call)
    assert np.isfinite(a.numpy()).all()
    X64, W64 = (torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in (x, w))
    y = X64 * torch.rsqrt((X64 * X64).mean(-1, keepdim=True) + 1e-6) * W64
    ang = torch.arange(T, dtype=torch.float64)[:, None, None] * 10000.0 ** (-2.0 * torch.arange(dk // 2, dtype=torch.float64) / dk)
    y = torch.cat([y[..., : dk // 2] * ang.cos() - y[..., dk // 2 :] * ang.sin(), y[..., : dk // 2] * ang.sin() + y[..., dk // 2 :] * ang.cos()], -1)
    seg = np.searchsorted(starts, np.arange(T), side="right")
    mask = torch.tensor((seg[:, None] == seg[None]) & (np.arange(T)[:, None] >= np.arange(T)[None]))
    s = (torch.einsum("thd,shd->hts", y, y) * dk ** -0.5).masked_fill(~mask, -1e300)
    (torch.einsum("hts,shd->thd", torch.softmax(s, -1), X64) * torch.tensor(r, dtype=torch.float64)).sum().backward()
    for got, want in ((X.grad(), X64.grad), (W.grad(), W64.grad)):
        # some hundred roundings on the way from a sum of a few hundred terms of order one: 2^-24 * 1000 of the largest
        assert np.abs(got.contiguous().numpy() - want.numpy()).max() <= 1000 * 2.0 ** -24 * np.abs(want.numpy()).max()
