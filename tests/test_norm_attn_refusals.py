"""CPU: calls of group_norm_act / cross_attn that are refused -- by the library (before any HIP call) and by the launchers."""
import ctypes as C

import pytest
import torch

from underwater_image_restoration_amd import _lib, ops

P = 1 << 20     # stands for a device pointer: checks come before any access


def refused(rc, *words):
    msg = _lib.load().uwir_last_error().decode()
    assert rc == -1 and all(w in msg for w in words), (rc, msg)


def gn(**o):
    a = dict(x=P, xd=0, ldx=64, B=2, n=10, C=64, G=8, eps=1e-5, gamma=P, beta=P, ss=None, ld_ss=0, act=0, out=P << 4, od=0, ldo=64,
             mean=None, rstd=None, ws=P << 5, nb=1 << 20)
    a.update(o)
    return _lib.load().uwir_group_norm_act(*a.values(), None)


def gnb(**o):
    a = dict(dy=P, ldy=64, x=P << 3, ldx=64, dt=0, B=2, n=10, C=64, G=8, gamma=P, beta=P, mean=P, rstd=P, ss=None, ld_ss=0, act=0,
             dx=P << 4, ldd=64, dg=P, db=P, dss=None, ld_dss=0, ws=P << 5, nb=1 << 20)
    a.update(o)
    return _lib.load().uwir_group_norm_act_backward(*a.values(), None)


def ca(**o):
    a = dict(q=P, ldq=64, k=P << 1, ldk=64, v=P << 2, ldv=64, dt=1, B=2, nq=10, nk=20, H=2, KV=2, hd=32, scale=0.5, lens=None, mask=None,
             ldm=0, out=P << 4, ldo=64, lse=None, ws=None, nb=0)
    a.update(o)
    return _lib.load().uwir_cross_attn(*a.values(), None)


def cab(**o):
    a = dict(q=P, ldq=64, k=P << 1, ldk=64, v=P << 2, ldv=64, out=P << 3, ldo=64, lse=P, go=P << 4, ldg=64, dt=1, B=2, nq=10, nk=20, H=2,
             KV=2, hd=32, scale=0.5, lens=None, mask=None, ldm=0, dq=P << 5, ld_dq=64, dk=P << 6, ld_dk=64, dv=P << 7, ld_dv=64,
             ws=P << 8, nb=1 << 20)
    a.update(o)
    return _lib.load().uwir_cross_attn_backward(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(ws=None), "null"), (dict(B=0), "shape"), (dict(n=0), "shape"),
    (dict(C=2056, ldx=2056, ldo=2056), "shape"), (dict(G=7), "groups"), (dict(G=0), "groups"), (dict(act=2), "act"), (dict(xd=2), "dtype"),
    (dict(od=5), "dtype"), (dict(ldx=63), "stride"), (dict(ldo=0), "stride"), (dict(ss=P, ld_ss=127), "stride"), (dict(eps=0.0), "eps"),
    (dict(nb=16), "workspace"), (dict(ws=(P << 5) + 8), "aligned"), (dict(out=P + 256), "overlap"), (dict(out=P, od=1, ldo=128), "overlap"),
    (dict(out=P + 64 * 4 * 2), "overlap"), (dict(ws=P + 512), "workspace")])
def test_group_norm_act_refuses(kw, word):
    refused(gn(**kw), "group_norm_act", word)


@pytest.mark.parametrize("kw,word", [
    (dict(dy=None), "null"), (dict(mean=None), "null"), (dict(dg=None), "null"), (dict(G=9), "groups"), (dict(act=1), "act"), (dict(dt=3), "dtype"),
    (dict(ldd=60), "stride"), (dict(dss=P, ld_dss=128), "dscale_shift"), (dict(ss=P, ld_ss=128, dss=P, ld_dss=100), "stride"),
    (dict(nb=0), "workspace"), (dict(dx=P + 128), "overlap"), (dict(dx=(P << 3) + 256), "overlap")])
def test_group_norm_act_backward_refuses(kw, word):
    refused(gnb(**kw), "group_norm_act_backward", word)


COMMON = [(dict(q=None), "null"), (dict(v=None), "null"), (dict(dt=2), "dtype"), (dict(B=0), "shape"), (dict(nq=-1), "shape"), (dict(nk=-1), "shape"),
          (dict(KV=3), "kv_heads"), (dict(hd=0), "head size"), (dict(hd=36), "head size"), (dict(hd=136), "head size"), (dict(scale=0.0), "scale"),
          (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(ldq=56), "stride"),
          (dict(ldk=68), "aligned"), (dict(q=P + 8), "aligned"), (dict(mask=P, ldm=19), "mask"), (dict(B=40000), "too large"),
          (dict(nq=1 << 30), "too large")]


@pytest.mark.parametrize("kw,word", COMMON + [
    (dict(out=P), "overlap"), (dict(out=(P << 1) + 128), "overlap"), (dict(out=P + 64, ldo=72, ldq=72), "overlap"),
    (dict(nq=1, nk=100000, out=P << 8), "workspace")])
def test_cross_attn_refuses(kw, word):
    refused(ca(**kw), "cross_attn", word)


@pytest.mark.parametrize("kw,word", COMMON + [
    (dict(lse=None), "lse"), (dict(go=None), "null"), (dict(dk=None), "null"), (dict(dq=P), "overlap"), (dict(dv=P << 6), "overlap"),
    (dict(ws=None), "workspace"), (dict(nb=64), "workspace"), (dict(ws=(P << 8) + 4), "workspace")])
def test_cross_attn_backward_refuses(kw, word):
    refused(cab(**kw), "cross_attn_backward", word)


# operands apart from each other: what a call that is not refused would look like
GN_APART = dict(gamma=P << 6, beta=P << 7, ws=P << 8, out=P << 4)
GNB_APART = dict(GN_APART, dy=P, x=P << 3, dx=P << 4, mean=P << 9, rstd=P << 10, dg=P << 11, db=P << 12)
del GNB_APART["out"]


@pytest.mark.parametrize("kw,words", [
    (dict(mean=P << 9, rstd=P << 9), ("mean", "rstd")), (dict(mean=P << 6), ("mean", "gamma")), (dict(rstd=P << 8), ("workspace", "rstd")),
    (dict(ws=P << 7), ("workspace", "beta")), (dict(out=(P << 6) - 256), ("out", "gamma")), (dict(ss=P << 4, ld_ss=128), ("out", "scale_shift")),
    (dict(mean=P), ("mean", "x"))])
def test_group_norm_act_refuses_shared_memory(kw, words):
    refused(gn(**dict(GN_APART, **kw)), "overlaps", *words)


@pytest.mark.parametrize("kw,words", [
    (dict(db=P << 11), ("dgamma", "dbeta")), (dict(dg=P << 6), ("dgamma", "gamma")), (dict(db=(P << 7) + 128), ("dbeta", "beta")),
    (dict(ss=P << 13, ld_ss=128, dss=P << 13, ld_dss=128), ("dscale_shift", "scale_shift")), (dict(ws=P << 9), ("workspace", "mean")),
    (dict(dg=P << 3), ("dgamma", "x")), (dict(rstd=(P << 4) + 512), ("dx", "rstd")), (dict(dg=P), ("dgamma", "dy"))])
def test_group_norm_act_backward_refuses_shared_memory(kw, words):
    refused(gnb(**dict(GNB_APART, **kw)), "overlaps", *words)


SPLIT = dict(nq=1, nk=8192, ws=P << 9, nb=1 << 24)     # a call that needs a workspace


@pytest.mark.parametrize("kw,words", [
    (dict(SPLIT, ws=(P << 4) - 256), ("workspace", "out")), (dict(SPLIT, ws=P << 1), ("workspace", "k")),
    (dict(SPLIT, lse=P << 4), ("lse", "out")), (dict(lse=(P << 4) + 64), ("lse", "out")), (dict(lse=P), ("lse", "q")),
    (dict(SPLIT, lse=P << 9), ("workspace", "lse"))])
def test_cross_attn_refuses_shared_memory(kw, words):
    refused(ca(**kw), "overlaps", *words)


@pytest.mark.parametrize("kw,words", [
    (dict(ws=P << 4), ("workspace", "dout")), (dict(ws=P << 6), ("workspace", "dk")), (dict(ws=(P << 5) + 16), ("workspace", "dq")),
    (dict(lse=P << 7), ("lse", "dv")), (dict(lse=P << 8), ("workspace", "lse"))])
def test_cross_attn_backward_refuses_shared_memory(kw, words):
    refused(cab(**kw), "overlaps", *words)


def test_too_many_blocks_for_a_launch():
    Q = 1 << 40     # 64 GB of rows each
    refused(ca(B=1024, KV=32, H=32, hd=8, nq=1 << 17, nk=1, ldq=256, ldk=256, ldv=256, ldo=256, q=Q, k=2 * Q, v=3 * Q, out=4 * Q),
            "too many rows")


def test_nothing_to_do_is_no_error():
    assert ca(nq=0, q=None, out=None) == 0
    assert cab(nq=0, nk=0) == 0


def test_workspace_sizes():
    assert ops.cross_attn_workspace_bytes(8, 4096, 77, 8, 8, 32, torch.bfloat16) == 0
    assert ops.cross_attn_workspace_bytes(1, 1, 8192, 8, 8, 64, torch.bfloat16) > 0
    assert ops.group_norm_act_workspace_bytes(2, 10, 64, 8) > 0 and ops.group_norm_act_workspace_bytes(0, 10, 64, 8) == 0
    with pytest.raises(TypeError):
        ops.cross_attn_workspace_bytes(1, 1, 1, 1, 1, 32, torch.float16)


def test_launchers_check_shapes_types_and_devices():
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    x, w, ws = f(20, 64), f(64), f(100000)
    ok = dict(mean=None)
    for bad, err in (((f(20, 63), w, w, f(20, 64)), ValueError), ((x, f(63), w, f(20, 64)), ValueError), ((x, w.double(), w, f(20, 64)), ValueError),
                     ((x, w, w, f(21, 64)), ValueError), ((x.t().contiguous().t(), w, w, f(20, 64)), ValueError),
                     ((x.half(), w, w, f(20, 64)), TypeError)):
        with pytest.raises(err):
            ops.group_norm_act(bad[0], 2, 10, 64, 8, 1e-5, bad[1], bad[2], bad[3], ws, **ok)
    with pytest.raises(ValueError):
        ops.group_norm_act(x, 2, 10, 64, 8, 1e-5, w, w, f(20, 64), ws, act=ops.ACT_RELU)
    with pytest.raises(ValueError):
        ops.group_norm_act(x, 2, 10, 64, 8, 1e-5, w, w, f(20, 64), ws, mean=f(2, 9))
    with pytest.raises(ValueError):     # a device of its own for one operand
        ops.group_norm_act(x, 2, 10, 64, 8, 1e-5, w.to("meta"), w, f(20, 64), ws)
    with pytest.raises(TypeError):
        ops.group_norm_act_backward(x.bfloat16(), x, 2, 10, 64, 8, w, w, f(2, 8), f(2, 8), f(20, 64), f(64), f(64), ws)
    q, k = f(10, 64), f(20, 64)
    d = (2, 5, 10, 2, 2, 32, 0.5)
    for a, kw, err in (((f(10, 60), k, k), {}, ValueError), ((q, k.bfloat16(), k), {}, TypeError), ((q, f(21, 64), k), {}, ValueError),
                       ((q, k, k), dict(key_lens=torch.zeros(2)), ValueError), ((q, k, k), dict(key_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
                       ((q, k, k), dict(key_mask=f(2, 10)), TypeError), ((q, k, k), dict(key_mask=torch.ones(2, 9, dtype=torch.bool)), ValueError),
                       ((q, k, k), dict(lse=f(2, 5, 2)), ValueError), ((q, k, k.to("meta")), {}, ValueError)):
        with pytest.raises(err):
            ops.cross_attn(*a, *d, f(10, 64), None, **kw)
    with pytest.raises(TypeError):
        ops.cross_attn_backward(q, k, k, q, f(2, 2, 5), q.bfloat16(), *d, f(10, 64), f(20, 64), f(20, 64), ws)
    with pytest.raises((ValueError, RuntimeError, AssertionError)):     # host tensors never reach a kernel
        ops.cross_attn(q, k, k, *d, f(10, 64), None)


def test_argument_lists_match_the_header():
    """ctypes checks nothing: the signature table must have the header's argument counts."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "uwir.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    kinds = {"int": C.c_int, "size_t": C.c_size_t, "float": C.c_float}
    for name in ("uwir_group_norm_act", "uwir_group_norm_act_backward", "uwir_cross_attn", "uwir_cross_attn_backward",
                 "uwir_group_norm_act_workspace_bytes", "uwir_cross_attn_workspace_bytes", "uwir_cross_attn_backward_workspace_bytes"):
        decl = re.search(r"\b" + name + r"\s*\(([^;]*?)\)\s*;", text, flags=re.S).group(1)
        want = [C.c_void_p if "*" in a or "stream_t" in a else kinds[a.split()[0]] for a in decl.split(",")]
        assert want == _lib._SIGS[name][1], name
