"""What the learning operators refuse, on the host: wrong arguments return before any device work."""
import ctypes

import pytest

VP = ctypes.c_void_p
P = VP(4096)  # an address that is never dereferenced: the calls below return before a launch
ONE = 0x3F800000
INVALID, OVERFLOW, WORKSPACE = 1, 2, 3


@pytest.fixture()
def lib(provider):
    return provider.library()


@pytest.fixture()
def word():
    return ctypes.byref(ctypes.c_uint64(0))


def _norm(lib, word, **change):
    a = dict(dtype=0, act=0, x=P, w=None, b=None, out=P, stats=P, n=2, s=3, c=8, g=2, xb=24, xs=8, ob=24, os=8, eps=0,
             ws=None, ws_bytes=0, status=word)
    a.update(change)
    return lib.pcu_b200_group_norm(a["dtype"], a["act"], a["x"], a["w"], a["b"], a["out"], a["stats"], a["n"], a["s"],
                                   a["c"], a["g"], a["xb"], a["xs"], a["ob"], a["os"], a["eps"], a["ws"], a["ws_bytes"],
                                   a["status"], None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=4), INVALID), (dict(dtype=-1), INVALID), (dict(act=4), INVALID), (dict(act=-1), INVALID),
    (dict(status=None), INVALID), (dict(x=None), INVALID), (dict(out=None), INVALID), (dict(stats=None), INVALID),
    (dict(g=0), INVALID), (dict(g=3), INVALID), (dict(xs=7), INVALID), (dict(xb=23), INVALID), (dict(os=7), INVALID),
    (dict(ob=23), INVALID), (dict(eps=0x7F800000), INVALID), (dict(eps=0xBF800000), INVALID), (dict(eps=0x7FC00000), INVALID),
    (dict(xs=9, xb=26), INVALID),  # in place (out is x), but not element for element
    (dict(n=1 << 31), OVERFLOW), (dict(s=1 << 41), OVERFLOW), (dict(c=1 << 31, g=1), OVERFLOW),
    (dict(xs=1 << 57), OVERFLOW), (dict(n=1 << 20, s=1 << 39, xb=1 << 50), OVERFLOW),
    (dict(x=VP(4098), out=VP(8192)), INVALID), (dict(out=VP(4097)), INVALID), (dict(w=VP(4097)), INVALID),
    (dict(b=VP(4098)), INVALID), (dict(stats=VP(4098)), INVALID), (dict(dtype=2, x=VP(4097), out=VP(8192)), INVALID),
    (dict(dtype=1, stats=VP(4100)), INVALID),
])
def test_group_norm(lib, word, change, code):
    assert _norm(lib, word, **change) == code


def test_group_norm_of_nothing(lib, word):
    assert _norm(lib, word, n=0, x=None, out=None, stats=None) == 0
    assert _norm(lib, word, c=0, x=None, out=None, stats=None) == 0


def _norm_backward(lib, word, **change):
    a = dict(dtype=0, act=0, x=P, dy=P, w=None, b=None, stats=P, dx=VP(8192), dw=None, db=None, n=2, s=3, c=8, g=2, xb=24,
             xs=8, yb=24, ys=8, ob=24, os=8, ws=P, ws_bytes=1 << 30, status=word)
    a.update(change)
    return lib.pcu_b200_group_norm_backward(*[a[k] for k in (
        "dtype", "act", "x", "dy", "w", "b", "stats", "dx", "dw", "db", "n", "s", "c", "g", "xb", "xs", "yb", "ys", "ob", "os",
        "ws", "ws_bytes", "status")], None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=4), INVALID), (dict(status=None), INVALID), (dict(x=None), INVALID), (dict(dy=None), INVALID),
    (dict(dx=None), INVALID), (dict(stats=None), INVALID), (dict(ys=7), INVALID), (dict(yb=20), INVALID),
    (dict(ys=1 << 57), OVERFLOW), (dict(ws=None), WORKSPACE), (dict(ws_bytes=3), WORKSPACE), (dict(ws=VP(4098)), WORKSPACE),
    (dict(dx=P, dy=VP(8192), xs=9, xb=27), INVALID), (dict(dy=VP(4097)), INVALID), (dict(dw=VP(4097)), INVALID),
    (dict(db=VP(4098)), INVALID),
])
def test_group_norm_backward(lib, word, change, code):
    assert _norm_backward(lib, word, **change) == code


def test_group_norm_backward_of_nothing(lib, word):
    assert _norm_backward(lib, word, n=0, x=None, dy=None, dx=None, stats=None, ws=None, ws_bytes=0) == 0
    for dtype in range(4):
        assert lib.pcu_b200_group_norm_workspace_size(dtype, 2, 3, 8, 2) % 8 == 0
        assert lib.pcu_b200_group_norm_backward_workspace_size(dtype, 2, 3, 8, 2) > 0
        # sizes that the call refuses have no workspace that could be allocated for them by mistake
        assert lib.pcu_b200_group_norm_backward_workspace_size(dtype, 2, 3, 8, 0) == 0
        assert lib.pcu_b200_group_norm_backward_workspace_size(dtype, 1 << 40, 1 << 40, 1 << 40, 1) == 0
    assert lib.pcu_b200_group_norm_backward_workspace_size(9, 2, 3, 8, 2) == 0


def _distill(lib, word, call, **change):
    a = dict(dtype=0, z=P, rows=2, vocab=10, stride=10, at=P, top=P, k=3, w=None, t=ONE, loss=P, stats=P, up=None, uni=0,
             g=VP(8192), gs=10, status=word)
    a.update(change)
    head = [a[k] for k in ("dtype", "z", "rows", "vocab", "stride", "at", "top", "k", "w", "t")]
    if call == "loss":
        return lib.pcu_b200_distill_loss(*head, a["loss"], a["stats"], a["status"], None)
    if call == "backward":
        return lib.pcu_b200_distill_loss_backward(*head, a["stats"], a["up"], a["uni"], a["g"], a["gs"], a["status"], None)
    return lib.pcu_b200_distill_loss_step(*head, a["loss"], a["stats"], a["up"], a["uni"], a["g"], a["gs"], a["status"], None)


@pytest.mark.parametrize("call", ["loss", "backward", "step"])
@pytest.mark.parametrize("change,code", [
    (dict(dtype=4), INVALID), (dict(status=None), INVALID), (dict(z=None), INVALID), (dict(vocab=0), INVALID),
    (dict(stride=9), INVALID), (dict(at=None), INVALID), (dict(top=None), INVALID), (dict(t=0), INVALID),
    (dict(t=0xBF800000), INVALID), (dict(t=0x7F800000), INVALID), (dict(t=0x7FC00000), INVALID), (dict(t=1), INVALID),
    (dict(k=1025), OVERFLOW), (dict(rows=1 << 31), OVERFLOW), (dict(vocab=1 << 31, stride=1 << 31, gs=1 << 31), OVERFLOW),
    (dict(stride=1 << 41), OVERFLOW), (dict(z=VP(4097)), INVALID), (dict(top=VP(4098)), INVALID),
    (dict(at=VP(4100)), INVALID), (dict(w=VP(4097)), INVALID), (dict(stats=VP(4098)), INVALID),
])
def test_distill(lib, word, call, change, code):
    assert _distill(lib, word, call, **change) == code


def test_distill_of_each_call(lib, word):
    assert _distill(lib, word, "loss", loss=None) == INVALID
    assert _distill(lib, word, "loss", stats=None) == INVALID
    assert _distill(lib, word, "step", loss=None) == INVALID
    for call in ("backward", "step"):
        assert _distill(lib, word, call, g=None) == INVALID
        assert _distill(lib, word, call, gs=9) == INVALID
        assert _distill(lib, word, call, gs=11, g=P) == INVALID  # in place with another stride
    assert _distill(lib, word, "backward", stats=None) == INVALID
    for call in ("loss", "backward", "step"):
        assert _distill(lib, word, call, rows=0, z=None, at=None, top=None, loss=None, stats=P, g=None) in (0, INVALID)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=1), INVALID), (dict(dtype=4), INVALID), (dict(high=2), INVALID), (dict(status=None), INVALID),
    (dict(x=None), INVALID), (dict(codes=None), INVALID), (dict(scales=None), INVALID), (dict(stride=9), INVALID),
    (dict(codes_stride=9), INVALID), (dict(rows=1 << 31), OVERFLOW), (dict(columns=1 << 31, stride=1 << 31, codes_stride=1 << 31), OVERFLOW),
    (dict(x=VP(4097)), INVALID), (dict(scales=VP(4098)), INVALID),
    (dict(stride=1 << 41), OVERFLOW), (dict(rows=0, x=None, codes=None, scales=None), 0),
])
def test_block_quantize(lib, word, change, code):
    a = dict(dtype=0, x=P, rows=4, columns=10, stride=10, high=1, codes=P, codes_stride=16, scales=P, status=word)
    a.update(change)
    assert lib.pcu_b200_block_quantize(a["dtype"], a["x"], a["rows"], a["columns"], a["stride"], a["high"], a["codes"],
                                       a["codes_stride"], a["scales"], a["status"], None) == code


@pytest.mark.parametrize("change,code", [
    (dict(dtype=1), INVALID), (dict(dtype=4), INVALID), (dict(status=None), INVALID), (dict(a=None), INVALID),
    (dict(b=None), INVALID), (dict(sa=None), INVALID), (dict(sb=None), INVALID), (dict(out=None), INVALID),
    (dict(lda=9), INVALID), (dict(ldb=9), INVALID), (dict(ldo=9), INVALID), (dict(m=1 << 31), OVERFLOW),
    (dict(out=VP(4098)), INVALID), (dict(sa=VP(4097)), INVALID), (dict(sb=VP(4098)), INVALID),
    (dict(k=1 << 31, lda=1 << 31, ldb=1 << 31), OVERFLOW), (dict(ldo=1 << 41), OVERFLOW),
    (dict(m=1 << 30, n=1 << 30, ldo=1 << 30), OVERFLOW), (dict(m=0, a=None, out=None), 0), (dict(n=0, b=None, out=None), 0),
])
def test_block_matmul(lib, word, change, code):
    a = dict(dtype=0, a=P, sa=P, b=P, sb=P, out=P, m=4, k=10, n=10, lda=16, ldb=16, ldo=10, status=word)
    a.update(change)
    assert lib.pcu_b200_block_matmul(*[a[k] for k in ("dtype", "a", "sa", "b", "sb", "out", "m", "k", "n", "lda", "ldb", "ldo",
                                                      "status")], None) == code


def test_guarded_forms_want_records(lib):
    assert lib.pcu_b200_guarded_group_norm(0, 0, P, None, None, P, P, 1, 1, 8, 2, 8, 8, 8, 8, 0, None, 0, None, 0, None) == INVALID
    assert lib.pcu_b200_guarded_group_norm_backward(0, 0, P, P, None, None, P, P, None, None, 1, 1, 8, 2, 8, 8, 8, 8, 8, 8, P,
                                                    64, None, 0, None) == INVALID
    assert lib.pcu_b200_guarded_distill_loss(0, P, 1, 8, 8, P, P, 1, None, ONE, P, P, None, 0, None) == INVALID
    assert lib.pcu_b200_guarded_distill_loss_backward(0, P, 1, 8, 8, P, P, 1, None, ONE, P, None, 0, P, 8, None, 0, None) == INVALID
    assert lib.pcu_b200_guarded_distill_loss_step(0, P, 1, 8, 8, P, P, 1, None, ONE, P, P, None, 0, P, 8, None, 0, None) == INVALID
    assert lib.pcu_b200_guarded_block_quantize(0, P, 1, 8, 8, 1, P, 16, P, None, 0, None) == INVALID
    assert lib.pcu_b200_guarded_block_matmul(0, P, P, P, P, P, 1, 8, 8, 16, 16, 8, None, 0, None) == INVALID
