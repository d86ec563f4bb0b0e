"""CPU: what the lookup, fp8 and AdamW entry points refuse.  Every check sits on the host in front of the first launch, so
the error codes come back without a GPU; pointers are made up and never followed."""
import ctypes as C

import pytest
import torch

from ddgani_amd import _lib, ops

OK, ARG, UNSUPPORTED, WORKSPACE = 0, -1, -2, -3
P = 1 << 20          # a pointer-like number, aligned to everything


def embed(**kw):
    a = dict(ids=P, i64=1, n=4, table=P, tt=0, V=10, D=8, ld=8, scale=1.0, out=P, ot=0, ldo=8, s=None)
    a.update(kw)
    return _lib.lib().ddg_embedding(*a.values())


@pytest.mark.parametrize("kw", [dict(ids=None), dict(table=None), dict(out=None), dict(n=-1), dict(V=0), dict(D=0), dict(ld=7),
                                dict(ldo=7), dict(tt=3), dict(ot=-1), dict(i64=2), dict(V=1 << 31)])
def test_embedding_refuses(kw):
    assert embed(**kw) == ARG


def test_embedding_empty():
    assert embed(n=0, ids=None, out=None) == OK
    assert embed(n=0, D=0) == ARG


def grad(**kw):
    a = dict(ids=P, i64=0, n=100, dy=P, dt=1, ldd=8, V=10, D=8, scale=1.0, pad=-1, acc=0, out=P, ot=0, ldo=8, ws=P, wsb=1 << 30,
             s=None)
    a.update(kw)
    return _lib.lib().ddg_embedding_grad(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(ids=None), ARG), (dict(dy=None), ARG), (dict(out=None), ARG), (dict(V=0), ARG),
                                   (dict(D=0), ARG), (dict(ldd=7), ARG), (dict(ldo=7), ARG), (dict(dt=9), ARG), (dict(ot=9), ARG),
                                   (dict(i64=-1), ARG), (dict(n=-1), ARG), (dict(n=1 << 31), UNSUPPORTED),
                                   (dict(V=(1 << 31) - 1), UNSUPPORTED), (dict(ws=None), WORKSPACE), (dict(wsb=100), WORKSPACE),
                                   (dict(ws=P + 8), ARG)])
def test_embedding_grad_refuses(kw, rc):
    assert grad(**kw) == rc


def test_embedding_grad_nothing_to_add():
    assert grad(n=0, acc=1, ids=None, dy=None, ws=None, wsb=0) == OK


def adamw(t=None, **kw):
    t = t or [dict()]
    arr = (_lib.AdamwTensor * len(t))(*[_lib.AdamwTensor(*{**dict(p=P, g=P, n=300, off=0, wd=0.0, pt=0, gt=0, r=0), **e}.values())
                                        for e in t])
    a = dict(tensors=arr, count=len(t), bits=32, m=P, v=P, ms=P, vs=P, master=None, length=512, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8,
             max_norm=1.0, control=P, ws=P, wsb=1 << 20, s=None)
    a.update(kw)
    return _lib.lib().ddg_adamw_step(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(bits=16), ARG), (dict(m=None), ARG), (dict(v=None), ARG), (dict(control=None), ARG),
                                   (dict(bits=8, ms=None), ARG), (dict(bits=8, vs=None), ARG), (dict(b1=1.0), ARG),
                                   (dict(b2=-0.1), ARG), (dict(eps=-1.0), ARG), (dict(lr=float("nan")), ARG),
                                   (dict(max_norm=float("nan")), ARG), (dict(ws=None), WORKSPACE), (dict(wsb=0), WORKSPACE),
                                   (dict(count=-1), ARG), (dict(tensors=None, count=2), ARG), (dict(length=299), ARG),
                                   (dict(m=P + 4), ARG), (dict(t=[dict(p=None)]), ARG), (dict(t=[dict(g=None)]), ARG),
                                   (dict(t=[dict(n=-1)]), ARG), (dict(t=[dict(off=128)]), ARG), (dict(t=[dict(off=-256)]), ARG),
                                   (dict(t=[dict(off=256)]), ARG), (dict(t=[dict(pt=3)]), ARG), (dict(t=[dict(gt=-1)]), ARG)])
def test_adamw_refuses(kw, rc):
    assert adamw(**kw) == rc


def fp8(**kw):
    a = dict(x=P, xt=0, ldx=64, rows=100, w=P, out=32, inn=64, bias=None, y=P, yt=0, ldy=32, ws=P, wsb=1 << 30, s=None)
    a.update(kw)
    return _lib.lib().ddg_fp8_linear(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(x=None), ARG), (dict(w=None), ARG), (dict(y=None), ARG), (dict(w=P + 16), ARG),
                                   (dict(out=0), ARG), (dict(inn=0), ARG), (dict(rows=-1), ARG), (dict(ldx=63), ARG),
                                   (dict(ldy=31), ARG), (dict(xt=3), ARG), (dict(yt=3), ARG), (dict(ws=None), WORKSPACE),
                                   (dict(wsb=64), WORKSPACE), (dict(ws=P + 16), ARG), (dict(rows=1 << 40), ARG)])
def test_fp8_linear_refuses(kw, rc):
    assert fp8(**kw) == rc


def test_fp8_reductions_that_are_too_long():
    """refused in front of the first launch: these pointers are followed nowhere"""
    assert fp8(rows=17, inn=1 << 24, ldx=1 << 24, wsb=1 << 62) == UNSUPPORTED
    assert fp8(rows=1, inn=1 << 24, ldx=1 << 24, wsb=1 << 62) == UNSUPPORTED
    g = lambda rows, out, inn: _lib.lib().ddg_fp8_linear_grads(P, 0, out, P, 0, inn, rows, P, out, inn, P, 0, inn, P, None, P, 1 << 62,
                                                               None)
    assert g(1 << 24, 32, 64) == UNSUPPORTED and g(50, 1 << 24, 64) == UNSUPPORTED


def test_fp8_linear_no_rows():
    assert fp8(rows=0, x=None, y=None, ws=None, wsb=0) == OK


@pytest.mark.parametrize("kw", [dict(W=None), dict(packed=None), dict(packed=P + 1), dict(packed_t=P + 128), dict(type=4),
                                dict(ld=63), dict(out=0), dict(inn=0)])
def test_fp8_pack_refuses(kw):
    a = dict(W=P, type=0, ld=64, out=32, inn=64, packed=P, packed_t=None, s=None)
    a.update(kw)
    assert _lib.lib().ddg_fp8_pack_weight(*a.values()) == ARG


@pytest.mark.parametrize("kw,rc", [(dict(dy=None), ARG), (dict(x=None), ARG), (dict(wt=None), ARG), (dict(dx=None), ARG),
                                   (dict(dw=None), ARG), (dict(rows=0), ARG), (dict(ldd=31), ARG), (dict(ldx=63), ARG),
                                   (dict(lddx=63), ARG), (dict(wt=P + 64), ARG), (dict(dxt=7), ARG), (dict(ws=None), WORKSPACE),
                                   (dict(wsb=1000), WORKSPACE), (dict(ws=P + 32), ARG)])
def test_fp8_grads_refuse(kw, rc):
    a = dict(dy=P, dyt=0, ldd=32, x=P, xt=0, ldx=64, rows=50, wt=P, out=32, inn=64, dx=P, dxt=0, lddx=64, dw=P, db=None, ws=P,
             wsb=1 << 30, s=None)
    a.update(kw)
    assert _lib.lib().ddg_fp8_linear_grads(*a.values()) == rc


def test_more_workgroups_than_a_launch_takes():
    """refused in front of the first launch as well"""
    assert embed(n=1 << 33, D=2048, ld=2048, ldo=2048) == UNSUPPORTED
    assert grad(V=(1 << 31) - 2, D=1 << 20, ldd=1 << 20, ldo=1 << 20, wsb=1 << 62) == UNSUPPORTED
    assert grad(n=(1 << 31) - 1, D=2048, ldd=2048, ldo=2048, wsb=1 << 62) == UNSUPPORTED
    big = 1 << 40
    assert adamw(t=[dict(n=big)], length=big, wsb=1 << 40) == UNSUPPORTED
    assert adamw(t=[dict(n=1 << 32, off=i << 32) for i in range(20)], length=20 << 32, wsb=1 << 40) == UNSUPPORTED
    assert fp8(rows=1 << 29, inn=128, ldx=128, wsb=1 << 62) == UNSUPPORTED               # tiles of the result
    assert fp8(rows=1 << 28, inn=128, ldx=128, wsb=1 << 62) == UNSUPPORTED               # groups of x
    g = lambda rows, out, inn: _lib.lib().ddg_fp8_linear_grads(P, 0, out, P, 0, inn, rows, P, out, inn, P, 0, inn, P, None, P, 1 << 62,
                                                               None)
    assert g(1 << 23, (1 << 24) - 256, (1 << 24) - 256) == UNSUPPORTED
    pack = lambda out, inn: _lib.lib().ddg_fp8_pack_weight(P, 1, inn, out, inn, P, None, None)
    assert pack(1 << 29, 1 << 20) == UNSUPPORTED


@pytest.mark.parametrize("decay", [-0.1, float("nan")])
def test_adamw_refuses_decay(decay):
    assert adamw(t=[dict(wd=decay)]) == ARG


def test_workspace_sizes_of_bad_shapes():
    L = _lib.lib()
    assert L.ddg_embedding_grad_workspace_bytes(-1, 4) == 0 and L.ddg_embedding_grad_workspace_bytes(4, 0) == 0
    assert L.ddg_fp8_operand_bytes(-1, 4) == 0 and L.ddg_fp8_linear_workspace_bytes(4, 4, 0) == 0
    assert L.ddg_fp8_linear_grads_workspace_bytes(4, 0, 4) == 0
    assert L.ddg_adamw_workspace_bytes(None, 3) == 0


def test_operand_layout_size():
    # codes: (rows up to 16) x (cols up to 128); scales: one word for four blocks and row, and 1 KB; each part up to 256 bytes
    assert _lib.lib().ddg_fp8_operand_bytes(3, 130) == 16 * 256 + 1280
    assert _lib.lib().ddg_fp8_operand_bytes(100, 513) == 112 * 640 + 2048      # 5 blocks: two words a row


def test_python_front_end_refuses_host_tensors():
    t, i = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ops.embedding(i, t), lambda: ops.embedding_grad(i, torch.zeros(3, 8), 4), lambda: ops.Fp8Weight(t),
                 lambda: ops.AdamW([t], [t])):
        with pytest.raises(_lib.DdgError):
            call()


def test_python_front_end_refuses_arguments():
    t = torch.zeros(4)
    for kw in (dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(lr=float("nan")), dict(max_norm=0.0),
               dict(weight_decay=[0.1, 0.2])):
        with pytest.raises(_lib.DdgError):
            ops.AdamW([t], [t], **kw)
    with pytest.raises(_lib.DdgError):
        ops.AdamW([], [])
    with pytest.raises(_lib.DdgError):
        ops.embedding(torch.zeros(3), torch.zeros(4, 8))          # ids of a floating type
