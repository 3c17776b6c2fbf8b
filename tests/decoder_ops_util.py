"""What the tests of the decoder-training operators share: tensors of the library made from numpy arrays (whole, strided or at an
odd offset), calls through the C ABI, and the operators' definitions in 64 bits."""
import ctypes as C

import numpy as np

U = 2.0 ** -24          # half a step of f32, relative


def rnd(seed, *shape, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(np.float32)


class Dev:
    """A tensor of the library; `view` lays the values out in a larger buffer: "whole", "strided" (a gap behind every row of the
    last two dimensions), "odd" (starting one element into the buffer) or "turned" (last dimension not contiguous)."""

    def __init__(self, vb, a, view="whole"):
        self.vb = vb
        a = np.ascontiguousarray(a, dtype=np.float32)
        shape = a.shape
        if view == "strided":
            buf = np.full(shape[:-2] + (shape[-2] + 1, shape[-1] + 4), np.nan, np.float32)
            buf[..., : shape[-2], : shape[-1]] = a
            base, strides = 0, [x // 4 for x in buf.strides]
        elif view == "odd":
            buf = np.full(a.size + 1, np.nan, np.float32)
            buf[1:] = a.reshape(-1)
            base, strides = 1, [x // 4 for x in a.strides]
        elif view == "turned":
            t = np.ascontiguousarray(np.swapaxes(a, -1, -2))
            buf, base, strides = t, 0, [x // 4 for x in t.strides]
            strides[-1], strides[-2] = strides[-2], strides[-1]
        else:
            buf, base, strides = a, 0, [x // 4 for x in a.strides]
        buf = np.ascontiguousarray(buf)
        slot = C.c_uint32()
        vb.vb_check(vb.lib().vb_alloc(max(1, buf.size), 0, C.byref(slot)))
        if buf.size:
            vb.vb_check(vb.lib().vb_write(slot.value, 0, buf.ctypes.data_as(vb.c_f32p), buf.size))
            vb.sync()
        self.desc = vb.VbTensor.contiguous(slot.value, shape, base)
        for i, s in enumerate(strides):
            self.desc.strides[i] = s

    def __del__(self):
        self.vb.lib().vb_release(self.desc.slot, None)

    @property
    def ref(self):
        return C.byref(self.desc)


def outputs(vb, fn, *args, n):
    """Calls fn(*args, out_1 .. out_n) and returns the outputs as arrays; raises VearoError on a refusal."""
    outs = [vb.VbTensor() for _ in range(n)]
    vb.vb_check(fn(*[a.ref if isinstance(a, Dev) else a for a in args], *[C.byref(o) for o in outs]), fn.__name__)
    got = []
    for o in outs:
        a = np.empty(o.shape, np.float32)
        vb.vb_check(vb.lib().vb_read(o.slot, o.offset, a.ctypes.data_as(vb.c_f32p), a.size))
        vb.lib().vb_release(o.slot, None)
        got.append(a)
    return got


# ---- definitions in 64 bits -----------------------------------------------------------------------------------------------------
def rope(x, pos, theta, rot, inter, sign=1.0):
    x = x.copy()
    if rot == 0:
        return x
    ang = sign * pos.astype(np.float64)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / rot)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = (x[..., 0:rot:2].copy(), x[..., 1:rot:2].copy()) if inter else (x[..., : rot // 2].copy(), x[..., rot // 2 : rot].copy())
    ya, yb = a * c - b * s, a * s + b * c
    if inter:
        x[..., 0:rot:2], x[..., 1:rot:2] = ya, yb
    else:
        x[..., : rot // 2], x[..., rot // 2 : rot] = ya, yb
    return x


def norm_rope(x, w, pos, theta, rot, inter, eps):
    x, w = x.astype(np.float64), w.astype(np.float64)
    return rope(x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w, pos, theta, rot, inter)


def norm_rope_grad(x, w, pos, theta, rot, inter, eps, g):
    x, w = x.astype(np.float64), w.astype(np.float64)
    g = rope(g.astype(np.float64), pos, theta, rot, inter, -1.0)
    inv = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * inv
    return inv * (g * w - xh * (g * w * xh).mean(-1, keepdims=True)), (g * xh).sum((0, 1))


def segment_attention(q, k, v, starts, scale, g=None, err=False):
    """(out, lse[, dq, dk, dv]) in 64 bits and, with err, a bound for every element of each.

    Bounds, in units of U: a score carries 57 of scale sum |q k| (split 2^-22 twice, the dropped term, 24 truncating additions a run);
    p = exp(s - lse) turns the score's error and two roundings of |s| + |lse| + 20 into a relative one, plus 4 for the exponential;
    a sum over keys adds 60 (splitting and truncation) and 3 for every 128 keys (rescaling, additions) of its terms' absolute sum, and
    what the halves' subnormals lose: 2^-38 of the largest weight for each key.  dS is held on a scale set by the row and value lengths
    of a block: 2^-36 of the largest |do| |v| product a key."""
    T, hq, dk = q.shape
    hk = k.shape[1]
    grp = hq // hk
    f = lambda x: x.astype(np.float64)  # noqa: E731
    q, k, v = f(q), f(k), f(v)
    o, lse = np.zeros((T, hq, dk)), np.full((hq, T), -np.inf)
    eo, el = np.zeros((T, hq, dk)), np.zeros((hq, T))
    dq, dk_, dv = np.zeros((T, hq, dk)), np.zeros((T, hk, dk)), np.zeros((T, hk, dk))
    edq, edk, edv = np.zeros((T, hq, dk)), np.zeros((T, hk, dk)), np.zeros((T, hk, dk))
    g = None if g is None else f(g)
    a = np.abs
    top = 0.0 if g is None else np.sqrt((g * g).sum(-1)).max() * np.sqrt((v * v).sum(-1)).max()
    for b, e in zip(starts[:-1], starts[1:]):
        b, e = int(b), int(e)
        n = e - b
        if n <= 0:
            continue
        mask = np.tril(np.ones((n, n), bool))
        for h in range(hq):
            Q, K, V = q[b:e, h], k[b:e, h // grp], v[b:e, h // grp]
            s = np.where(mask, Q @ K.T * scale, -np.inf)
            m = s.max(1, keepdims=True)
            L = m + np.log(np.exp(s - m).sum(1, keepdims=True))
            p = np.exp(s - L)
            o[b:e, h], lse[h, b:e] = p @ V, L[:, 0]
            es = 57 * U * scale * (a(Q) @ a(K).T)
            sa = np.where(mask, a(s), 0.0)
            r = es + (4 + 2 * (sa + a(L) + 20)) * U
            e_l = (p * r).sum(1, keepdims=True) + (20 + n / 40 + 2 * a(L)) * U
            r = r + e_l
            steps = (60 + 3 * n / 128 + 10) * U
            eo[b:e, h] = (p * (r + steps)) @ a(V) + 2.0 ** -38 * (mask @ a(V))
            el[h, b:e] = e_l[:, 0]
            if g is None:
                continue
            G = g[b:e, h]
            dp, delta = G @ V.T, (G * o[b:e, h]).sum(1, keepdims=True)
            ds = p * (dp - delta) * scale
            dq[b:e, h] = ds @ K
            dk_[b:e, h // grp] += ds.T @ Q
            dv[b:e, h // grp] += p.T @ G
            e_dp = 57 * U * (a(G) @ a(V).T)
            e_delta = (a(G) * (eo[b:e, h] + dk * U * a(o[b:e, h]))).sum(1, keepdims=True)
            e_ds = scale * mask * (p * (r * a(dp - delta) + e_dp + e_delta + 8 * U * (a(dp) + a(delta))) + 2.0 ** -36 * top)
            edq[b:e, h] = e_ds @ a(K) + steps * (a(ds) @ a(K))
            gsteps = steps * grp
            edk[b:e, h // grp] += e_ds.T @ a(Q) + gsteps * (a(ds).T @ a(Q))
            edv[b:e, h // grp] += (p * (r + gsteps)).T @ a(G) + 2.0 ** -38 * (mask.T @ a(G))
    vals = (o, lse) if g is None else (o, lse, dq, dk_, dv)
    errs = (eo, el) if g is None else (eo, el, edq, edk, edv)
    return (vals, errs) if err else vals
