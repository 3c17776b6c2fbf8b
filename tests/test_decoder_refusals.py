"""What the decoder-training entry points say without a device: every one refuses, names the reason and leaves its outputs alone."""
import ctypes as C
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Tensor(C.Structure):
    _fields_ = [("slot", C.c_uint32), ("rank", C.c_int32), ("offset", C.c_int64), ("dims", C.c_int64 * 8), ("strides", C.c_int64 * 8)]


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    lib = C.CDLL(os.path.join(ROOT, "vearo_b200", "libvearo_b200.so"))
    lib.vb_last_error.restype = C.c_char_p
    return lib


def tensor(*shape):
    t = Tensor(slot=1, rank=len(shape), offset=0)
    step = 1
    for i in reversed(range(len(shape))):
        t.dims[i], t.strides[i] = shape[i], step
        step *= shape[i]
    return t


def calls():
    q, k, w, pos, starts = tensor(4, 2, 8), tensor(4, 1, 8), tensor(8), tensor(4), tensor(2)
    x, head, targets, lse, one = tensor(4, 8), tensor(5, 8), tensor(4), tensor(2, 4), tensor(1)
    f, i, big = C.c_float, C.c_int, C.c_int64
    return {
        "vb_qk_norm_rope": ((q, k, w, w, pos, f(1e4), i(8), i(0), f(1e-6)), 2),
        "vb_qk_norm_rope_backward": ((q, k, w, w, pos, f(1e4), i(8), i(0), f(1e-6), q, k), 4),
        "vb_segment_attention": ((q, k, k, starts, f(0.5)), 2),
        "vb_segment_attention_backward": ((q, k, k, starts, f(0.5), q, lse, q), 3),
        "vb_linear_cross_entropy": ((x, head, targets, big(-100)), 2),
        "vb_linear_cross_entropy_backward": ((x, head, targets, big(-100), targets, one), 2),
    }


@pytest.mark.parametrize("name", sorted(calls()))
@pytest.mark.parametrize("null", [False, True])
def test_refused_without_a_device(lib, name, null):
    args, n = calls()[name]
    outs = [tensor(3, 7) for _ in range(n)]
    before = [bytes(o) for o in outs]
    passed = [None if null and isinstance(a, Tensor) else C.byref(a) if isinstance(a, Tensor) else a for a in args]
    assert getattr(lib, name)(*passed, *[C.byref(o) for o in outs]) == 3, lib.vb_last_error()      # VB_ERR_NOT_INIT
    assert b"vb_init" in lib.vb_last_error()
    assert [bytes(o) for o in outs] == before
