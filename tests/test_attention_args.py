"""Refusals of the attention operators and the epilogue's backward pass: the C
ABI's without a device, the Python functions' on host tensors."""
import ctypes
import math

import pytest
import torch

from t2h import _build, _lib, ops

P = ctypes.c_void_p(256)       # never dereferenced: validation fails first
Q = ctypes.c_void_p(1 << 20)


@pytest.fixture(scope="module")
def lib():
    import os

    if not os.path.exists(_build.LIB_PATH):
        _build.build()
    return _lib.load()


def strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


def fwd(lib, q=P, k=P, v=P, out=Q, lse=None, st=None, rows=64, krows=64, h=4, kvh=4, d=64, dt=1, scale=0.125, qo=None,
        ko=None, kl=None, nb=1, ws=None, wb=0):
    return lib.t2h_attention(q, k, v, out, lse, st, rows, krows, h, kvh, d, dt, scale, qo, ko, kl, nb, ws, wb, None)


def bwd(lib, q=P, k=P, v=P, out=P, lse=P, dout=P, dq=Q, dk=Q, dv=Q, st=None, rows=64, krows=64, h=4, kvh=4, d=64, dt=1,
        scale=0.125, nb=1, ws=Q, wb=1 << 40):
    return lib.t2h_attention_backward(q, k, v, out, lse, dout, dq, dk, dv, st, rows, krows, h, kvh, d, dt, scale, None,
                                      None, None, nb, ws, wb, None)


BAD = [(dict(dt=0), -2, b"f16 or bf16"), (dict(dt=9), -1, b"f16 or bf16"), (dict(d=96), -2, b"64 or 128"),
       (dict(d=32), -2, b"64 or 128"), (dict(h=4, kvh=3), -1, b"multiple of kv_heads"), (dict(kvh=0), -1, b"bad shape"),
       (dict(h=0), -1, b"bad shape"), (dict(rows=-1), -1, b"bad shape"), (dict(krows=-2), -1, b"bad shape"),
       (dict(nb=0), -1, b"nbatch"), (dict(nb=3), -1, b"divide into nbatch"), (dict(scale=0.0), -1, b"scale"),
       (dict(scale=-1.0), -1, b"scale"), (dict(scale=math.inf), -1, b"scale"), (dict(scale=math.nan), -1, b"scale"),
       (dict(rows=1 << 31), -2, b"rows"), (dict(krows=(1 << 31) - 1), -2, b"rows"),
       (dict(rows=1 << 30, h=65535, kvh=1), -2, b"tiles"), (dict(q=None), -1, b"q is NULL"),
       (dict(k=None), -1, b"k is NULL"), (dict(v=None), -1, b"v is NULL"), (dict(out=None), -1, b"out is NULL"),
       (dict(q=ctypes.c_void_p(260)), -1, b"16-byte aligned"), (dict(v=ctypes.c_void_p(264)), -1, b"16-byte aligned")]


@pytest.mark.parametrize("call", [fwd, bwd])
@pytest.mark.parametrize("args,code,text", BAD, ids=lambda v: str(v)[:28])
def test_attention_refuses(lib, call, args, code, text):
    assert call(lib, **args) == code
    assert text in lib.t2h_last_error()


@pytest.mark.parametrize("i,name", enumerate(["q", "k", "v", "out", "dout", "dq", "dk", "dv"]))
@pytest.mark.parametrize("bad,code", [((60, 64), -1), ((256, 4), -1), ((-256, 64), -1), ((256, -64), -1),
                                      ((260, 64), -1), ((256, 68), -1), ((1 << 24, 64), -2), (((1 << 22) + 8, 64), -2)])
def test_attention_refuses_strides(lib, i, name, bad, code):
    st = [256, 64] * 8
    st[2 * i:2 * i + 2] = bad
    calls = [(bwd, 8)] + ([(fwd, 4)] if i < 4 else [])
    for call, n in calls:
        assert call(lib, st=strides(*st[:2 * n])) == code
        assert f"{name} ".encode() in lib.t2h_last_error()


def test_attention_refuses_aliases_and_workspaces(lib):
    assert fwd(lib, out=P) == -1 and b"alias" in lib.t2h_last_error()
    assert fwd(lib, ws=ctypes.c_void_p(8), wb=1 << 30) == -1 and b"workspace" in lib.t2h_last_error()
    for name in ("dq", "dk", "dv"):
        assert bwd(lib, **{name: P}) == -1 and b"alias" in lib.t2h_last_error()
    assert bwd(lib, lse=None) == -1 and b"lse is NULL" in lib.t2h_last_error()
    assert bwd(lib, ws=None) == -1 and b"needs a workspace of" in lib.t2h_last_error()
    assert bwd(lib, wb=16) == -1 and b"needs a workspace of" in lib.t2h_last_error()
    assert bwd(lib, ws=ctypes.c_void_p(24)) == -1 and b"16-byte aligned" in lib.t2h_last_error()


def test_gradients_that_alias_each_other(lib):
    """Their blocks run side by side: one would overwrite the other's."""
    R, S = ctypes.c_void_p(1 << 21), ctypes.c_void_p(1 << 22)
    for args in (dict(dq=R, dk=R, dv=S), dict(dq=R, dk=S, dv=R), dict(dq=R, dk=S, dv=S)):
        assert bwd(lib, **args) == -1 and b"alias each other" in lib.t2h_last_error()
    kw = dict(q=ctypes.c_void_p(512), k=ctypes.c_void_p(1024), dq=ctypes.c_void_p(2048), dk=ctypes.c_void_p(4096))
    for args in (dict(), dict(dqi=kw["dk"]), dict(dki=kw["dq"]), dict(dqi=kw["k"]), dict(dki=kw["q"]),
                 dict(dq=P, dk=P, dqi=P, dki=P)):
        assert qkb(lib, **{**kw, **args}) == -1 and b"must not alias" in lib.t2h_last_error()


def test_expanded_tensors_are_refused(monkeypatch):
    """A stride of 0 means contiguous to the C ABI: it would read past an
    expanded tensor's end. A dimension of one has no stride that counts."""
    full, one = torch.zeros((6, 2, 64)), torch.zeros((1, 1, 64))
    rows, heads = torch.zeros((1, 2, 64)).expand(6, 2, 64), torch.zeros((6, 1, 64)).expand(6, 2, 64)
    for bad in (rows, heads):
        with pytest.raises(ValueError, match="x must not be expanded"):
            ops._attn_operand(bad, bad.shape, bad.dtype, "f", "x")
    assert ops._attn_operand(full, full.shape, full.dtype, "f", "x") == (128, 64)
    assert ops._attn_operand(one.expand(1, 1, 64), one.shape, one.dtype, "f", "x") == (0, 0)
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    with pytest.raises(ValueError, match="rows must not overlap"):
        ops._heads_view(rows, "f")
    with pytest.raises(ValueError, match="heads must be contiguous"):
        ops._heads_view(heads, "f")
    assert ops._heads_view(full, "f") == (6, 2, 64, 128)
    assert ops._heads_view(torch.zeros((7, 64)).as_strided((1, 2, 64), (0, 64, 1)), "f") == (1, 2, 64, 128)


def test_attention_workspaces(lib):
    assert lib.t2h_attention_workspace(-1, 1, 1, 1, 64, 1) == -1
    assert lib.t2h_attention_workspace(1, 1, 1, 1, 60, 1) == -1
    assert lib.t2h_attention_backward_workspace(1, 1, 2, 3, 64, 1) == -1
    assert lib.t2h_attention_workspace(4096, 4096, 12, 12, 128, 1) == 0          # enough blocks without a split
    one = lib.t2h_attention_workspace(1, 1 << 20, 12, 12, 128, 1)                # parts' outputs and log-sum-exps
    assert one > 0 and one % (12 * 129 * 4) == 0
    # at least delta and lse2
    assert lib.t2h_attention_backward_workspace(1000, 1000, 12, 12, 128, 1) >= 2 * 1000 * 12 * 4
    assert lib.t2h_attention_workspace(0, 0, 1, 1, 64, 1) == 0
    assert lib.t2h_qk_rmsnorm_rope_backward_workspace(-1, 1, 64, 1) == -1
    assert lib.t2h_qk_rmsnorm_rope_backward_workspace(10, 1, 64, 3) == -1
    assert lib.t2h_qk_rmsnorm_rope_backward_workspace(4, 2, 64, 2) >= 2 * 2 * 2 * 64 * 4


def test_attention_of_nothing_is_a_noop(lib):
    assert fwd(lib, q=None, out=None, rows=0) == 0
    assert bwd(lib, q=None, k=None, v=None, out=None, lse=None, dout=None, dq=None, dk=None, dv=None, rows=0, krows=0,
               ws=None, wb=0) == 0
    assert lib.t2h_last_error() == b""


def qkb(lib, q=P, k=P, dq=P, dk=P, dqi=Q, dki=Q, rows=8, xs=0, ys=0, ds=0, h=2, d=64, dt=0, bq=None, bk=None, gq=P, gk=P,
        rope=0, dgq=None, dgk=None, dbq=None, dbk=None, ws=None, wb=0):
    return lib.t2h_qk_rmsnorm_rope_backward(q, k, dq, dk, dqi, dki, rows, xs, ys, ds, h, d, dt, bq, bk, gq, gk, rope,
                                            None, 0, 3, None, 0, None, 0, 0, dgq, dgk, dbq, dbk, ws, wb, None)


@pytest.mark.parametrize("args,code,text", [
    (dict(dt=5), -1, b"bad dtype"), (dict(d=63), -1, b"bad shape"), (dict(d=258), -2, b"head_dim"),
    (dict(h=0), -1, b"bad shape"), (dict(rows=-1), -1, b"bad shape"), (dict(xs=100), -1, b"row stride"),
    (dict(ys=127), -1, b"row stride"), (dict(ds=1), -1, b"row stride"), (dict(dqi=None), -1, b"NULL tensor"),
    (dict(dq=None), -1, b"NULL tensor"), (dict(q=None), -1, b"needs its input"),
    (dict(gq=None, dgq=P), -1, b"dgamma without gamma"), (dict(dq=None, dqi=None, dgq=P), -1, b"needs its tensor"),
    (dict(dq=None, dqi=None, dk=None, dki=None), -1, b"both NULL"), (dict(dqi=P, ys=128, ds=256), -1, b"in place"),
    (dict(dgq=Q), -1, b"needs a workspace"), (dict(dgq=Q, ws=P, wb=64), -1, b"needs a workspace"),
    (dict(dbq=Q, ws=ctypes.c_void_p(8), wb=1 << 30), -1, b"needs a workspace"),
    (dict(rope=1), -1, b"needs phases, coords or grid_res")], ids=lambda v: str(v)[:28])
def test_qk_backward_refuses(lib, args, code, text):
    assert qkb(lib, **args) == code
    assert text in lib.t2h_last_error()


def test_qk_backward_of_nothing_is_a_noop(lib):
    assert qkb(lib, q=None, k=None, dq=None, dk=None, dqi=None, dki=None, rows=0) == 0


def test_python_refuses_host_tensors():
    q = torch.zeros((4, 2, 64), dtype=torch.float16)
    for f in (lambda: ops.attention(q, q, q), lambda: ops.qk_rmsnorm_rope_backward(dq=q),
              lambda: ops.attention_backward(q, q, q, q, q, torch.zeros((2, 4)))):
        with pytest.raises(ValueError, match="device"):
            f()
    with pytest.raises(ValueError, match="both None"):
        ops.qk_rmsnorm_rope_backward()
    with pytest.raises(ValueError):
        ops.attention_workspace(1, 1, 3, 2, 64)


def test_tensors_of_another_device_are_refused(monkeypatch):
    """The launch goes to the current device's stream."""
    class OnDevice:
        def __init__(self, i):
            self.i = i

        def get_device(self):
            return self.i

    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    monkeypatch.setattr(ops, "_current", lambda: 0)
    ops._same_device(OnDevice(0), (OnDevice(0), None), "f")
    with pytest.raises(ValueError, match="f: tensors must be on the current device"):
        ops._same_device(OnDevice(1), (OnDevice(1),), "f")
    with pytest.raises(ValueError, match="f: tensors are on different devices"):
        ops._same_device(OnDevice(0), (None, OnDevice(1)), "f")
