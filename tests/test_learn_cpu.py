"""The trainer-side operators without a GPU: what the C boundary and the Python entry points refuse, before anything is
launched.  Pointers handed to the C boundary here are numbers that nothing reads."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

A = 1 << 20         # a "buffer" every 2^20 bytes


def _lib():
    from mpe_hip import _lib
    return _lib, _lib.load()


def _err(lib):
    return lib.mpe_last_error(None).decode()


def _forward(lib, dtype=0, act=1, m=8, n=4, k=3, x=1 * A, ldx=3, w=2 * A, ldw=3, bias=3 * A, res=4 * A, ldr=4, y=5 * A, ldy=4, pre=6 * A, ws=7 * A, wsb=1 << 19):
    return lib.mpe_linear_forward(0, dtype, act, m, n, k, x, ldx, w, ldw, bias, res, ldr, y, ldy, pre, ws, wsb, None)


def _backward(lib, dtype=0, act=1, m=8, n=4, k=3, dy=1 * A, lddy=4, x=2 * A, ldx=3, w=3 * A, ldw=3, pre=4 * A, dx=5 * A, lddx=3, dw=6 * A, db=7 * A, ws=8 * A, wsb=1 << 19):
    return lib.mpe_linear_backward(0, dtype, act, m, n, k, dy, lddy, x, ldx, w, ldw, pre, dx, lddx, dw, db, ws, wsb, None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(dtype=9), "dtype"), (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(m=-1), "sizes"), (dict(n=0), "sizes"),
    (dict(k=0), "sizes"), (dict(m=1 << 41), "2^40"), (dict(m=1 << 30, n=1 << 20), "2^40"), (dict(n=1 << 31), "2^31"), (dict(x=None), "NULL"),
    (dict(w=None), "NULL"), (dict(y=None), "NULL"), (dict(ldx=2), "stride"), (dict(ldw=2), "stride"), (dict(ldy=3), "stride"), (dict(ldr=3), "stride"),
    (dict(x=A + 2), "aligned"), (dict(bias=3 * A + 1), "aligned"), (dict(pre=6 * A + 2), "aligned"), (dict(y=1 * A + 64), "overlap"), (dict(y=2 * A), "overlap"),
    (dict(pre=5 * A + 4), "overlap"), (dict(y=4 * A + 4), "overlap"), (dict(y=4 * A, ldy=8), "overlap"), (dict(ldx=1 << 62), "stride")])
def test_linear_forward_refuses(kw, text):
    _, lib = _lib()
    assert _forward(lib, **kw) == -1
    assert text in _err(lib), _err(lib)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(act=7), "activation"), (dict(act=5, dtype=2), "TANH_OUT"), (dict(dy=None), "NULL"), (dict(pre=None), "NULL"), (dict(lddy=3), "stride"), (dict(lddx=2), "stride"),
    (dict(dx=2 * A), "overlap"), (dict(dw=5 * A + 8), "overlap"), (dict(db=1 * A + 124), "overlap"), (dict(dw=6 * A + 1), "aligned"), (dict(pre=4 * A + 2), "aligned"),
    (dict(m=1 << 20, ws=None, ldx=3), "workspace"), (dict(m=1 << 12, ws=8 * A + 8), "workspace"), (dict(m=1 << 12, wsb=0), "workspace")])
def test_linear_backward_refuses(kw, text):
    _, lib = _lib()
    big = dict(dy=1 << 32, x=2 << 32, w=3 << 32, pre=4 << 32, dx=5 << 32, dw=6 << 32, db=7 << 32, n=257, lddy=257) if "workspace" == text else {}
    assert _backward(lib, **{**big, **kw}) == -1
    assert text in _err(lib), _err(lib)


def test_linear_with_nothing_to_do_needs_no_buffer():
    _, lib = _lib()
    assert _forward(lib, m=0, x=None, w=None, y=None) == 0
    assert _backward(lib, dx=None, dw=None, db=None, dy=None) == 0
    f, b = C.c_int64(-1), C.c_int64(-1)
    assert lib.mpe_linear_workspace(0, 1, 1000, 64, 64, C.byref(f), C.byref(b)) == 0 and f.value >= 0 and b.value >= 0
    assert lib.mpe_linear_workspace(1, 1, 1000, 64, 64, C.byref(f), C.byref(b)) == -1 and "dtype" in _err(lib)


def _ppo(lib, dtype=0, rows=8, v=5, logits=1 * A, ld=5, actions=2 * A, ab=4, olp=3 * A, adv=4 * A, mask=None, ldm=0, weights=None, values=5 * A, old=6 * A, ret=7 * A,
         clip=0.2, vclip=-1.0, loss=8 * A, stats=9 * A, ws=10 * A, wsb=1 << 19):
    return lib.mpe_ppo_loss_forward(0, dtype, rows, v, logits, ld, actions, ab, olp, adv, mask, ldm, weights, values, old, ret, clip, vclip, 0.5, 0.01, loss, stats,
                                    ws, wsb, None)


def _ppo_back(lib, rows=8, v=5, logits=1 * A, ld=5, values=5 * A, old=6 * A, ret=7 * A, stats=9 * A, grad=10 * A, dl=11 * A, ldd=5, dv=12 * A):
    return lib.mpe_ppo_loss_backward(0, 0, rows, v, logits, ld, 2 * A, 4, 3 * A, 4 * A, None, 0, None, values, old, ret, 0.2, -1.0, 0.5, 0.01, stats, grad, dl, ldd, dv,
                                     None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(v=0), "sizes"), (dict(rows=-1), "sizes"), (dict(ab=2), "int32"), (dict(clip=-0.1), "clip"), (dict(clip=float("nan")), "clip"),
    (dict(values=None), "together"), (dict(ret=None), "together"), (dict(logits=None), "NULL"), (dict(adv=None), "NULL"), (dict(ld=4), "stride"),
    (dict(mask=13 * A, ldm=4), "stride"), (dict(olp=3 * A + 2), "aligned"), (dict(ab=8, actions=2 * A + 4), "aligned"), (dict(loss=None), "loss"),
    (dict(stats=9 * A + 1), "aligned"), (dict(ws=None), "workspace"), (dict(wsb=100), "workspace")])
def test_ppo_forward_refuses(kw, text):
    _, lib = _lib()
    assert _ppo(lib, **kw) == -1
    assert text in _err(lib), _err(lib)


@pytest.mark.parametrize("kw, text", [
    (dict(stats=None), "NULL"), (dict(grad=None), "NULL"), (dict(dl=None), "NULL"), (dict(values=None, old=None, ret=None), "without values"), (dict(ldd=4), "stride"),
    (dict(dl=1 * A), "overlap"), (dict(dl=9 * A), "overlap"), (dict(dv=5 * A), "overlap"), (dict(dv=11 * A), "overlap"), (dict(dl=10 * A), "overlap")])
def test_ppo_backward_refuses(kw, text):
    _, lib = _lib()
    assert _ppo_back(lib, **kw) == -1
    assert text in _err(lib), _err(lib)


def test_clip_refuses():
    _, lib = _lib()
    arr = lambda t, *v: (t * len(v))(*v)
    src, cnt, typ = arr(C.c_void_p, A, 2 * A), arr(C.c_int64, 10, 20), arr(C.c_int32, 0, 2)
    call = lambda n=2, src=src, dst=src, cnt=cnt, typ=typ, mx=1.0, norm=3 * A, ws=4 * A, wsb=1 << 19: lib.mpe_clip_grad_norm(0, n, src, dst, cnt, typ, mx, norm, ws, wsb, None)
    for kw, text in ((dict(n=-1), "NULL"), (dict(src=None), "NULL"), (dict(dst=None, norm=None), "neither"), (dict(mx=-1.0), "max_norm"), (dict(mx=float("nan")), "max_norm"),
                     (dict(typ=arr(C.c_int32, 0, 1)), "dtype"), (dict(cnt=arr(C.c_int64, 10, -1)), "count"), (dict(src=arr(C.c_void_p, A, None)), "NULL"),
                     (dict(src=arr(C.c_void_p, A + 2, 2 * A)), "misaligned"), (dict(dst=arr(C.c_void_p, A + 4, 2 * A)), "overlap"), (dict(norm=3 * A + 2), "aligned"),
                     (dict(ws=None), "workspace"), (dict(ws=4 * A + 8), "workspace"), (dict(wsb=8), "workspace")):
        assert call(**kw) == -1, kw
        assert text in _err(lib), (kw, _err(lib))


def test_clip_refuses_destinations_that_meet_other_tensors():
    _, lib = _lib()
    arr = lambda t, *v: (t * len(v))(*v)
    cnt, typ = arr(C.c_int64, 10, 20, 0), arr(C.c_int32, 0, 2, 0)
    call = lambda src, dst: lib.mpe_clip_grad_norm(0, 3, arr(C.c_void_p, *src), arr(C.c_void_p, *dst), cnt, typ, 1.0, 3 * A, 4 * A, 1 << 19, None)
    for src, dst, text in (((A, 2 * A, None), (2 * A, A, None), "overlaps the source"),                 # swapped
                           ((A, 2 * A, None), (5 * A, A + 36, None), "overlaps the source of tensor 0"),    # its last element
                           ((A, 2 * A, None), (5 * A, 5 * A + 38, None), "given twice"),
                           ((A, A, None), (A, A, None), "given twice"),
                           ((A, A, None), (A, 2 * A, None), "overlaps the source of tensor 1")):
        assert call(src, dst) == -1 and text in _err(lib), (src, dst, _err(lib))


@pytest.mark.parametrize("kw", [dict(m=(1 << 29) + 1, n=1, k=1), dict(m=1 << 20, n=(1 << 17) + 1, k=1), dict(m=1 << 20, n=1, k=(1 << 17) + 1)])
def test_linear_refuses_more_tiles_than_a_grid_has(kw):
    _, lib = _lib()
    far = {n: (i + 1) << 44 for i, n in enumerate(("x", "w", "bias", "res", "y", "pre"))}
    assert _forward(lib, **far, **kw, ldx=kw["k"], ldw=kw["k"], ldr=kw["n"], ldy=kw["n"]) == -1 and "2^29 rows" in _err(lib), _err(lib)
    far = {n: (i + 1) << 44 for i, n in enumerate(("dy", "x", "w", "pre", "dx", "dw", "db", "ws"))}
    assert _backward(lib, **far, **kw, lddy=kw["n"], ldx=kw["k"], ldw=kw["k"], lddx=kw["k"]) == -1 and "2^29 rows" in _err(lib), _err(lib)


def test_linear_workspace_counts_whole_strips_of_many_rows():
    """The column sums of a large 16-bit weight gradient: at most 32768 strips, whatever m."""
    _, lib = _lib()
    b = C.c_int64(-1)
    for m in (1 << 22, (1 << 22) + 1, 1 << 25, 1 << 29):
        assert lib.mpe_linear_workspace(2, 0, m, 128, 256, None, C.byref(b)) == 0
        assert b.value <= 4 * (512 * 128 * 256 + 32768 * 128), (m, b.value)


def test_python_entry_points_refuse_cpu_tensors_and_bad_arguments():
    import mpe_hip
    x, w = torch.zeros(4, 3), torch.zeros(2, 3)
    with pytest.raises(ValueError, match="no CPU path"):
        mpe_hip.linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        mpe_hip.linear(x, w, activation="elu")
    with pytest.raises(ValueError, match="activation"):
        mpe_hip.linear(x, w, activation=["tanh"])
    with pytest.raises(ValueError, match="no CPU path"):
        mpe_hip.ppo_loss(torch.zeros(4, 5), torch.zeros(4, dtype=torch.int32), torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="on the GPU"):
        mpe_hip.grad_norm([x])
    with pytest.raises(ValueError, match="no tensors"):
        mpe_hip.grad_norm([])
    with pytest.raises(ValueError, match="max_norm"):
        mpe_hip.clip_grad_norm([x], -1.0, out=[x])
    with pytest.raises(ValueError, match="in out"):
        mpe_hip.clip_grad_norm([x], 1.0, out=[x, w])
    with pytest.raises(ValueError, match="no parameter"):
        mpe_hip.clip_grad_norm_([torch.nn.Parameter(x)], 1.0)


def test_the_binding_agrees_with_the_header():
    import os
    import re
    _l, _ = _lib()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "mpe_hip.h")).read()
    define = dict(re.findall(r"#define\s+(MPE_\w+)\s+\(?(-?\d+)\)?", text))
    for name, value in (("MPE_BF16", _l.MPE_BF16), ("MPE_F16", _l.MPE_F16), ("MPE_ACT_NONE", _l.ACT_NONE), ("MPE_ACT_TANH", _l.ACT_TANH),
                        ("MPE_ACT_RELU", _l.ACT_RELU), ("MPE_ACT_GELU", _l.ACT_GELU), ("MPE_ACT_SILU", _l.ACT_SILU),
                        ("MPE_CLIP_WORKSPACE_BYTES", _l.CLIP_WORKSPACE_BYTES), ("MPE_PPO_WORKSPACE_BYTES", _l.PPO_WORKSPACE_BYTES)):
        assert int(define[name]) == value, name
