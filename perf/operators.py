"""Cases of the decoder-training operators: the norm and rotation of queries and keys, causal attention with grouped heads over
packed segments, and the vocabulary projection with its cross entropy.

Each case is one pass through an operator, in its plain form (elementary torch operations) or, with `own`, through the calls
of this repository's C ABI.  Sizes are those of the workloads of bench.py (GPT-small: 12 heads of 64, width 768; GPT-medium:
16 heads of 64, width 1024; vocabulary 50304; 1024 tokens a sequence) and odd ones around them.
"""
import ctypes as C
import math
import random

import torch

own = False


def listed():
    return [
        # one token of a short prompt: what a call costs when there is nothing to do
        dict(name="norm_rope_1_token", op="norm_rope", tokens=1, hq=12, hk=4, dk=64, rot=64, interleaved=False),
        # GPT-small's micro-batch, 8 x 1024 tokens, with grouped keys
        dict(name="norm_rope_gpt_small", op="norm_rope", tokens=8192, hq=12, hk=4, dk=64, rot=64, interleaved=False),
        # its gradient
        dict(name="norm_rope_grad_gpt_small", op="norm_rope_grad", tokens=8192, hq=12, hk=4, dk=64, rot=64, interleaved=False),
        # wide heads of which half are rotated, neighbouring pairs, an odd number of tokens
        dict(name="norm_rope_grad_wide_odd", op="norm_rope_grad", tokens=4099, hq=16, hk=4, dk=128, rot=64, interleaved=True),
        # a few short texts in one pack, three rows behind the last of them
        dict(name="attention_short_pack", op="attention", tokens=203, segments=7, tail=3, hq=4, hk=2, dk=64),
        # GPT-small's micro-batch: every head has its own keys, all texts equally long
        dict(name="attention_gpt_small", op="attention", tokens=8192, segments=8, tail=0, hq=12, hk=12, dk=64),
        # one long text, wide grouped heads
        dict(name="attention_long", op="attention", tokens=16384, segments=1, tail=0, hq=8, hk=2, dk=128),
        # training on texts of many lengths packed into GPT-medium's micro-batch
        dict(name="attention_train_packed", op="attention_train", tokens=4096, segments=9, tail=17, hq=16, hk=4, dk=64),
        # an odd head size, odd lengths
        dict(name="attention_train_odd", op="attention_train", tokens=1531, segments=3, tail=0, hq=6, hk=2, dk=80),
        # evaluation of a handful of tokens with a small vocabulary
        dict(name="head_loss_small", op="head_loss", tokens=33, dim=128, vocab=512, ignored=0.1),
        # evaluation at GPT-small's size
        dict(name="head_loss_gpt_small", op="head_loss", tokens=8192, dim=768, vocab=50304, ignored=0.0),
        # training at GPT-medium's width, an odd number of tokens, some of them padding
        dict(name="head_loss_train_medium", op="head_loss_train", tokens=4097, dim=1024, vocab=50304, ignored=0.05),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope_grad", "attention", "attention_train", "head_loss", "head_loss_train"])
    hk = rng.choice([1, 2, 4, 6])
    hq = hk * rng.choice([1, 2, 3, 4])
    if op.startswith("norm_rope"):
        dk = rng.choice([32, 64, 80, 96, 128])
        return dict(op=op, tokens=_log_uniform(rng, 1, 9000), hq=hq, hk=hk, dk=dk, rot=dk if rng.random() < 0.6 else dk // 2,
                    interleaved=rng.random() < 0.5)
    if op.startswith("attention"):
        tokens = _log_uniform(rng, 2, 6000)
        hk = rng.choice([1, 2, 4])
        return dict(op=op, tokens=tokens, segments=rng.randint(1, max(1, min(24, tokens // 48))), tail=rng.choice([0, 0, min(5, tokens - 1)]),
                    hq=hk * rng.choice([1, 2, 3, 4]), hk=hk, dk=rng.choice([40, 64, 64, 96, 128]))
    return dict(op=op, tokens=_log_uniform(rng, 1, 4000), dim=8 * rng.randint(8, 128), vocab=_log_uniform(rng, 300, 50304),
                ignored=rng.choice([0.0, 0.0, 0.2]))


def _lengths(case):
    """Lengths of the segments of a pack: equal where they divide the tokens and nothing is left over, else cut at places that
    depend on the case alone (a place drawn twice leaves an empty segment)."""
    live, n = case["tokens"] - case["tail"], case["segments"]
    if case["tail"] == 0 and live % n == 0:
        return [live // n] * n
    r = random.Random(1000003 * live + n)
    cuts = sorted(r.randint(0, live) for _ in range(n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [live])]


THETA, EPS = 10000.0, 1e-6


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    op, t = case["op"], {}
    if op.startswith("norm_rope"):
        n, hq, hk, dk = case["tokens"], case["hq"], case["hk"], case["dk"]
        t["q"], t["k"] = normal(n, hq, dk, std=1.7), normal(n, hk, dk, std=0.6)
        t["wq"], t["wk"] = 1.0 + normal(dk, std=0.1), 1.0 + normal(dk, std=0.1)
        t["positions"] = ((torch.arange(n, device="cuda") + 3001) % 8192).float()
        if op == "norm_rope_grad":
            t["gq"], t["gk"] = normal(n, hq, dk, std=1e-2), normal(n, hk, dk, std=1e-2)
    elif op.startswith("attention"):
        n, hq, hk, dk = case["tokens"], case["hq"], case["hk"], case["dk"]
        t["q"], t["k"], t["v"] = normal(n, hq, dk, std=1.2), normal(n, hk, dk, std=1.2), normal(n, hk, dk)
        ends = torch.tensor([0] + _lengths(case)).cumsum(0)
        t["starts"] = ends.float().cuda()
        if op == "attention_train":
            t["g"] = normal(n, hq, dk, std=1e-2)
    else:
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        t["x"], t["w"] = normal(n, d), normal(v, d, std=2.0 / math.sqrt(d))
        target = torch.randint(0, v, (n,), generator=g, device="cuda")
        left_out = torch.rand(n, generator=g, device="cuda") < case["ignored"]
        t["targets"] = torch.where(left_out, torch.full_like(target, -100), target).float()
        if op == "head_loss_train":
            t["g"] = torch.ones(1, device="cuda")
    state = dict(case=case, t=t)
    if own:  # the same values in memory of the library, where its users have them
        state["d"] = {name: _device_tensor(x) for name, x in t.items()}
        torch.cuda.synchronize()
    return state


def run(state):
    return (_own_pass if own else _plain_pass)(state)


# ---- the plain form ---------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, rot, interleaved):
    """x [tokens, heads, dk]; cos, sin [tokens, 1, rot / 2]: pairs (i, i + rot / 2), or (2 i, 2 i + 1) where interleaved."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2 : rot])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _angles(t, rot):
    # positions times frequencies in 64 bits: 32 lose the angle of far positions
    freq = THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = t["positions"].double()[:, None, None] * freq
    return angle.cos().float(), angle.sin().float()


def _plain_norm_rope(case, t):
    cos, sin = _angles(t, case["rot"])

    def one(x, w):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        return _rotate(y, cos, sin, case["rot"], case["interleaved"])

    return one(t["q"], t["wq"]), one(t["k"], t["wk"])


def _plain_norm_rope_grad(case, t):
    cos, sin = _angles(t, case["rot"])

    def one(x, w, g):
        g = _rotate(g, cos, -sin, case["rot"], case["interleaved"])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xhat = x * r
        gw = g * w
        return r * (gw - xhat * (gw * xhat).mean(-1, keepdim=True)), (g * xhat).sum((0, 1))

    gq, gwq = one(t["q"], t["wq"], t["gq"])
    gk, gwk = one(t["k"], t["wk"], t["gk"])
    return gq, gk, gwq, gwk


def _plain_attention(case, t):
    """Every segment padded to the longest: [segments, heads, length, ...]."""
    hq, hk, dk = case["hq"], case["hk"], case["dk"]
    lengths = torch.tensor(_lengths(case), device="cuda")
    first, longest = lengths.cumsum(0) - lengths, max(_lengths(case))
    place = first[:, None] + torch.arange(longest, device="cuda")
    live = torch.arange(longest, device="cuda") < lengths[:, None]
    place = torch.where(live, place, torch.full_like(place, case["tokens"]))  # one more row, of zeros

    def padded(x):
        x = torch.cat([x, torch.zeros_like(x[:1])])[place].transpose(1, 2)
        return x if x.shape[1] == hq else x.repeat_interleave(hq // hk, 1)

    q, k, v = padded(t["q"]), padded(t["k"]), padded(t["v"])
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(dk))
    s = s.masked_fill(torch.ones(longest, longest, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)

    def packed(x):  # the rows of the pack, the rows behind its last segment zero
        out = torch.zeros(case["tokens"] + 1, x.shape[1], dk, device="cuda")
        out[place.reshape(-1)] = x.transpose(1, 2).reshape(-1, x.shape[1], dk)
        return out[:-1].index_fill(0, torch.arange(case["tokens"] - case["tail"], case["tokens"], device="cuda"), 0.0) if case["tail"] else out[:-1]

    o = p @ v
    if "g" not in t:
        return (packed(o),)
    g = padded(t["g"]) * live[:, None, :, None]
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (g * o).sum(-1, keepdim=True)) * (1.0 / math.sqrt(dk))
    shared = lambda x: x.reshape(x.shape[0], hk, hq // hk, longest, dk).sum(2)  # noqa: E731
    return packed(o), packed(ds @ k), packed(shared(ds.transpose(-1, -2) @ q)), packed(shared(p.transpose(-1, -2) @ g))


def _plain_head_loss(case, t):
    target = t["targets"].long()
    live = target != -100
    logits = t["x"] @ t["w"].T
    top = logits.amax(-1, keepdim=True)
    e = (logits - top).exp()
    total = e.sum(-1, keepdim=True)
    row = target.clamp_min(0)[:, None]
    lse = (top + total.log())[:, 0]
    nll = lse - logits.gather(1, row)[:, 0]
    count = live.sum().clamp_min(1).float()
    loss = (torch.where(live, nll, torch.zeros_like(nll)).sum() / count)[None]
    if "g" not in t:
        return loss, lse
    d = e / total
    d = d.scatter_add(1, row, torch.full_like(nll, -1.0)[:, None]) * (live[:, None] * (t["g"] / count))
    return loss, d @ t["w"], d.T @ t["x"]


_PLAIN = dict(norm_rope=_plain_norm_rope, norm_rope_grad=_plain_norm_rope_grad, attention=_plain_attention,
              attention_train=_plain_attention, head_loss=_plain_head_loss, head_loss_train=_plain_head_loss)


def _plain_pass(state):
    return _PLAIN[state["case"]["op"]](state["case"], state["t"])


# ---- the framework's calls ----------------------------------------------------------------------------------------------------
class _Owned:
    """A tensor of the library that a torch tensor can look into; the slot is released with the last look."""

    def __init__(self, desc):
        import vearo_b200 as vb
        self.desc, self.lib = desc, vb.lib()
        at = C.c_void_p()
        vb.vb_check(self.lib.vb_ptr(desc.slot, C.byref(at)), "vb_ptr")
        n = range(desc.rank)
        self.__cuda_array_interface__ = dict(shape=tuple(desc.dims[i] for i in n), strides=tuple(4 * desc.strides[i] for i in n),
                                             typestr="<f4", data=((at.value or 0) + 4 * desc.offset, False), version=3)

    def __del__(self):
        self.lib.vb_release(self.desc.slot, None)


def _device_tensor(x):
    """A tensor of the library with the values of a torch tensor."""
    import vearo_b200 as vb
    if not vb._inited:
        vb.init(torch.cuda.current_device())
    slot = C.c_uint32()
    vb.vb_check(vb.lib().vb_alloc(x.numel(), 0, C.byref(slot)), "vb_alloc")
    mine = _Owned(vb.VbTensor.contiguous(slot.value, tuple(x.shape)))
    torch.as_tensor(mine, device="cuda").copy_(x)
    return mine


def _own_pass(state):
    import vearo_b200 as vb
    L, case, d = vb.lib(), state["case"], state["d"]
    ref = lambda name: C.byref(d[name].desc)  # noqa: E731
    op = case["op"]
    new = [vb.VbTensor() for _ in range(5)]
    at = [C.byref(x) for x in new]
    if op == "norm_rope":
        rc = L.vb_qk_norm_rope(ref("q"), ref("k"), ref("wq"), ref("wk"), ref("positions"), THETA, case["rot"], int(case["interleaved"]), EPS, at[0], at[1])
        kept = new[:2]
    elif op == "norm_rope_grad":
        rc = L.vb_qk_norm_rope_backward(ref("q"), ref("k"), ref("wq"), ref("wk"), ref("positions"), THETA, case["rot"], int(case["interleaved"]), EPS,
                                        ref("gq"), ref("gk"), at[0], at[1], at[2], at[3])
        kept = new[:4]
    elif op == "attention":
        rc = L.vb_segment_attention(ref("q"), ref("k"), ref("v"), ref("starts"), 1.0 / math.sqrt(case["dk"]), at[0], None)
        kept = new[:1]
    elif op == "attention_train":
        scale = 1.0 / math.sqrt(case["dk"])
        rc = L.vb_segment_attention(ref("q"), ref("k"), ref("v"), ref("starts"), scale, at[0], at[4])
        rc = rc or L.vb_segment_attention_backward(ref("q"), ref("k"), ref("v"), ref("starts"), scale, at[0], at[4], ref("g"), at[1], at[2], at[3])
        kept = new[:4]
    elif op == "head_loss":
        rc = L.vb_linear_cross_entropy(ref("x"), ref("w"), ref("targets"), -100, at[0], at[1])
        kept = new[:2]
    else:
        rc = L.vb_linear_cross_entropy(ref("x"), ref("w"), ref("targets"), -100, at[0], at[4])
        rc = rc or L.vb_linear_cross_entropy_backward(ref("x"), ref("w"), ref("targets"), -100, at[4], ref("g"), at[1], at[2])
        kept = new[:3]
    vb.vb_check(rc, op)
    if new[4].slot:
        L.vb_release(new[4].slot, None)
    return tuple(torch.as_tensor(_Owned(x), device="cuda") for x in kept)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------
def work(case):
    op, n = case["op"], case["tokens"]
    if op.startswith("norm_rope"):
        q, dk = n * (case["hq"] + case["hk"]) * case["dk"], case["dk"]
        if op == "norm_rope":
            return dict(bytes=4 * (2 * q + 2 * dk + n), flops=9 * q)
        return dict(bytes=4 * (3 * q + 4 * dk + n), flops=16 * q)
    if op.startswith("attention"):
        pairs = sum(m * (m + 1) // 2 for m in _lengths(case))
        q, k = n * case["hq"] * case["dk"], n * case["hk"] * case["dk"]
        if op == "attention":  # Q K^T and P V
            return dict(bytes=4 * (2 * q + 2 * k), flops=4 * pairs * case["hq"] * case["dk"])
        return dict(bytes=4 * (4 * q + 4 * k), flops=12 * pairs * case["hq"] * case["dk"])  # and dP, dV, dK, dQ
    d, v = case["dim"], case["vocab"]
    if op == "head_loss":
        return dict(bytes=4 * (n * d + v * d + 2 * n + 1), flops=2 * n * v * d)
    return dict(bytes=4 * (2 * n * d + 2 * v * d + n + 1), flops=6 * n * v * d)  # the logits and both gradients


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------------------------------
def _exact_rope(x, positions, rot, interleaved, sign):
    """Pairs as complex numbers, turned by e^(i sign position theta^(-2 j / rot))."""
    j = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(()).double().cuda(), sign * positions[:, None] * torch.exp(-2.0 * j / rot * math.log(THETA)))[:, None, :]
    out = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., : rot // 2], x[..., rot // 2 : rot]) * turn
        out[..., : rot // 2], out[..., rot // 2 : rot] = z.real, z.imag
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        t = {name: x.double() for name, x in prepare(case, seed)["t"].items()}
    finally:
        own = was
    op = case["op"]
    if op.startswith("norm_rope"):
        out = []
        for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
            size = torch.sqrt(t[x].square().sum(-1, keepdim=True) / case["dk"] + EPS)
            if op == "norm_rope":
                out.append(_exact_rope(t[x] / size * t[w], t["positions"], case["rot"], case["interleaved"], 1.0))
            else:
                back = _exact_rope(t[g], t["positions"], case["rot"], case["interleaved"], -1.0)
                inner = (back * t[w] * t[x]).sum(-1, keepdim=True)
                out.append((back * t[w] / size - t[x] * inner / (case["dk"] * size**3), (back * t[x] / size).sum((0, 1))))
        return tuple(out) if op == "norm_rope" else (out[0][0], out[1][0], out[0][1], out[1][1])
    if op.startswith("attention"):
        o, dq, dk, dv = (torch.zeros_like(t[x]) for x in ("q", "q", "k", "v"))
        scale, group, at = 1.0 / math.sqrt(case["dk"]), case["hq"] // case["hk"], 0
        for m in _lengths(case):
            rows = slice(at, at + m)
            at += m
            future = torch.ones(m, m, dtype=torch.bool, device="cuda").triu(1)
            for h in range(case["hq"]):
                q, k, v = t["q"][rows, h], t["k"][rows, h // group], t["v"][rows, h // group]
                p = torch.softmax((q @ k.T * scale).masked_fill(future, -math.inf), -1)
                o[rows, h] = p @ v
                if op == "attention_train":
                    g = t["g"][rows, h]
                    ds = g @ v.T
                    ds = p * (ds - (ds * p).sum(-1, keepdim=True)) * scale
                    dq[rows, h] = ds @ k
                    dk[rows, h // group] += ds.T @ q
                    dv[rows, h // group] += p.T @ g
        return (o,) if op == "attention" else (o, dq, dk, dv)
    target = t["targets"].long()
    live = (target != -100).double()
    count = live.sum().clamp_min(1.0)
    logits = t["x"] @ t["w"].T
    lse = torch.logsumexp(logits, -1)
    log_p = logits - lse[:, None]
    del logits
    loss = -(log_p.gather(1, target.clamp_min(0)[:, None])[:, 0] * live).sum().reshape(1) / count
    if op == "head_loss":
        return loss, lse
    d = log_p.exp_()
    d[torch.arange(len(target), device="cuda"), target.clamp_min(0)] -= 1.0
    d *= (live / count * t["g"])[:, None]
    return loss, d @ t["w"], d.T @ t["x"]
