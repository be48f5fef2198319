"""Operators around a block, CPU part: the random numbers' definition, what the
C entries refuse before any launch, and each argument check by its message."""
import ctypes

import numpy as np
import pytest
import torch

from swiftrwkv_amd import _lib, train

from .philox import numbers, philox

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
D = 64   # a dummy, 16-byte aligned address: refused calls never reach a launch
OK, SHAPE, DTYPE, UNSUP, NULL = 0, 1, 2, 3, 6
DEVICE = "must live on a ROCm device"   # looked at last: what nothing else is wrong with reaches it


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


# ───────────────────────────── the generator ─────────────────────────────

@pytest.mark.parametrize("ctr,key,want", [
    ((0, 0, 0, 0), (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), "d16cfe09 94fdcceb 5001e420 24126ea1")])
def test_philox_is_the_published_one(ctr, key, want):
    assert " ".join(f"{int(x):08x}" for x in philox(ctr, key)) == want


def test_numbers_are_uniform():
    """65536 cells of 16 bits over 2^22 numbers: chi² within six of its standard deviations."""
    n = np.bincount(numbers(512, 8192, 12345, 1 << 40).ravel(), minlength=65536)
    chi = ((n - 64.0) ** 2 / 64).sum()
    assert abs(chi - 65535) < 6 * (2 * 65535) ** 0.5


# ───────────────────────────── C entries ─────────────────────────────

def refused(status, name, *args):
    assert getattr(_lib.lib(), name)(*args) == status, (name, _lib.lib().rwkv_last_error())


def drop(threshold=6554):
    return _lib.Drop(1, None, 0, threshold)


def test_dropout_entry_refuses():
    a = lambda **k: [k.get("x", D), k.get("xdt", 1), k.get("ldx", 8), k.get("res"), k.get("ldr", 0), k.get("y", D),  # noqa: E731
                     k.get("ydt", 1), k.get("drop", ctypes.byref(drop())), k.get("N", 2), k.get("D", 8), None]
    refused(DTYPE, "rwkv_dropout", *a(xdt=1, ydt=2))
    refused(DTYPE, "rwkv_dropout", *a(xdt=3, ydt=3))
    refused(SHAPE, "rwkv_dropout", *a(ldx=7))
    refused(SHAPE, "rwkv_dropout", *a(D=0))
    refused(SHAPE, "rwkv_dropout", *a(D=(1 << 22) + 1, ldx=1 << 23))
    refused(SHAPE, "rwkv_dropout", *a(N=(1 << 24) + 1))
    refused(SHAPE, "rwkv_dropout", *a(N=-1))
    refused(SHAPE, "rwkv_dropout", *a(res=D, ldr=7))
    refused(SHAPE, "rwkv_dropout", *a(ldx=1 << 32))
    refused(SHAPE, "rwkv_dropout", *a(res=D, ldr=1 << 32))
    refused(NULL, "rwkv_dropout", *a(x=None))
    refused(NULL, "rwkv_dropout", *a(y=None))
    refused(UNSUP, "rwkv_dropout", *a(drop=None))
    refused(UNSUP, "rwkv_dropout", *a(drop=ctypes.byref(drop(65537))))
    refused(UNSUP, "rwkv_dropout", *a(drop=ctypes.byref(drop(-1))))
    refused(OK, "rwkv_dropout", *a(N=0, x=None, y=None))


def join(**k):
    v = dict(x=D, o=D, gate=None, ldx=8, ldo=8, ldg=0, x_dt=0, dt=1, w_dt=0, post_weight=None, post_bias=None, scale=None,
             weight=D, bias=None, post_eps=1e-5, eps=1e-5, drop=drop(0), N=2, D=8)
    v.update(k)
    return ctypes.byref(_lib.Join(**v))


def test_join_entries_refuse():
    fwd = lambda j, xs=D, h=D, st=None: refused_join("rwkv_join_fwd", j, xs, h, st, None)  # noqa: E731

    def refused_join(name, *args):
        return getattr(_lib.lib(), name)(*args)

    assert fwd(join(x_dt=2)) == DTYPE and fwd(join(w_dt=2)) == DTYPE and fwd(join(dt=5)) == DTYPE
    assert fwd(join(x_dt=1, dt=0)) == DTYPE   # a 16-bit stream with an fp32 branch
    for bad in (dict(D=0), dict(D=8193, ldx=9000, ldo=9000), dict(ldx=7), dict(ldo=7), dict(gate=D, ldg=7), dict(N=-1),
                dict(N=(1 << 24) + 1)):
        assert fwd(join(**bad)) == SHAPE, bad
    assert fwd(join(x=None)) == NULL and fwd(join(weight=None)) == NULL and fwd(join(), xs=None) == NULL
    assert fwd(join(post_bias=D)) == NULL and fwd(None) == NULL
    assert fwd(join(), st=D + 4) == SHAPE
    assert fwd(join(drop=drop(65537))) == UNSUP
    assert fwd(join(N=0, x=None, o=None)) == OK

    def bwd(j, xs=D, st=D, dx=None, do=None, dg=None, dw=None, db=None, dpw=None, dpb=None, dsc=None, ws=D, wsn=1 << 20):
        return _lib.lib().rwkv_join_bwd(j, xs, st, D, D, dx, do, dg, dw, db, dpw, dpb, dsc, ws, wsn, None)

    need = _lib.lib().rwkv_join_bwd_workspace(2, 8)
    assert need >= 5 * 8 * 4 and need % 5 == 0
    one = need // 5
    assert bwd(join(), dw=D, wsn=one - 1) == SHAPE and bwd(join(), dw=D, ws=None) == SHAPE and bwd(join(), dw=D, ws=D + 4) == SHAPE
    assert bwd(join(), dg=D) == NULL and bwd(join(), dsc=D) == NULL and bwd(join(), dpw=D) == NULL and bwd(join(), dpb=D) == NULL
    assert bwd(join(o=None, scale=D), dw=D) == NULL and bwd(join(), xs=None, dw=D) == NULL and bwd(join(), st=None) == NULL
    assert bwd(join(x_dt=1, x=None), dw=D) == NULL and bwd(join(x_dt=1, o=None), dw=D) == NULL and bwd(join(x_dt=1, ldx=7), dw=D) == SHAPE
    assert bwd(join(x_dt=2), dw=D) == DTYPE and bwd(join(ldo=7), dw=D) == SHAPE and bwd(None) == NULL
    assert bwd(join(), st=D + 8) == SHAPE
    assert [_lib.lib().rwkv_join_bwd_workspace(*a) for a in ((-1, 8), (2, 0), (2, 8193))] == [0, 0, 0]


def tail(**k):
    v = dict(o=D, r=D, k=D, v=D, gate=D, ldo=64, ldr=64, ldk=64, ldv=64, ldg=64, o_dt=0, dt=1, w_dt=0, r_k=D, weight=D, bias=D,
             eps=64e-5, N=2, H=1)
    v.update(k)
    return ctypes.byref(_lib.Tail(**v))


def test_tail_entries_refuse():
    fwd = lambda j, y=D: _lib.lib().rwkv_tail_fwd(j, y, None)  # noqa: E731
    assert fwd(tail(o_dt=2)) == DTYPE and fwd(tail(w_dt=2)) == DTYPE and fwd(tail(dt=0, o_dt=1)) == DTYPE
    for n in ("ldo", "ldr", "ldk", "ldv", "ldg"):
        assert fwd(tail(**{n: 63})) == SHAPE, n
    assert fwd(tail(H=0)) == SHAPE and fwd(tail(H=1025)) == SHAPE and fwd(tail(N=-1)) == SHAPE
    for n in ("o", "r", "k", "v", "gate", "r_k", "weight", "bias"):
        assert fwd(tail(**{n: None})) == NULL, n
    assert fwd(tail(), None) == NULL and fwd(None) == NULL and fwd(tail(N=0, o=None), None) == OK

    def bwd(j, dy=D, ld=64, drk=D, dw=D, db=D, ws=D, wsn=1 << 20):
        return _lib.lib().rwkv_tail_bwd(j, dy, ld, D, D, D, D, D, drk, dw, db, ws, wsn, None)

    need = _lib.lib().rwkv_tail_bwd_workspace(2, 1)
    assert need >= 3 * 64 * 4 and _lib.lib().rwkv_tail_bwd_workspace(2, 0) == 0
    assert bwd(tail(), wsn=need - 1) == SHAPE and bwd(tail(), ws=None) == SHAPE and bwd(tail(), ws=D + 4) == SHAPE
    assert bwd(tail(), ld=63) == SHAPE and bwd(tail(), dy=None) == NULL and bwd(tail(), dw=None) == NULL
    assert bwd(tail(r=None)) == NULL and bwd(tail(o_dt=2)) == DTYPE and bwd(None) == NULL


# ───────────────────────────── arguments ─────────────────────────────

SEED2 = torch.zeros(2, dtype=torch.int64)


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, DEVICE), (dict(x=t(8)), ValueError, DEVICE), (dict(residual=t(2, 8, dtype=F32)), ValueError, DEVICE),
    (dict(p=0), ValueError, DEVICE), (dict(p=1.0), ValueError, DEVICE), (dict(seed=(1 << 64) - 1, offset=1 << 63), ValueError, DEVICE),
    (dict(seed=torch.zeros(1, dtype=torch.int64)), ValueError, DEVICE), (dict(seed=torch.tensor(5)), ValueError, DEVICE),
    (dict(seed=np.int64(5), offset=np.uint64(7)), ValueError, DEVICE),
    (dict(p=-0.1), ValueError, "p must be 0 to 1"), (dict(p=1.01), ValueError, "p must be 0 to 1"),
    (dict(p=float("nan")), ValueError, "p must be 0 to 1"), (dict(p="a"), TypeError, "real number"),
    (dict(seed=-1), ValueError, "seed must be an integer of 0"), (dict(seed=1 << 64), ValueError, "seed must be an integer of 0"),
    (dict(seed=1.0), TypeError, "seed must be an integer"), (dict(seed=None), TypeError, "seed must be an integer"),
    (dict(offset=-1), ValueError, "offset must be an integer"), (dict(offset=torch.tensor(1)), TypeError, "offset must be an integer"),
    (dict(seed=SEED2), TypeError, "one int64"), (dict(seed=torch.zeros(1)), TypeError, "one int64"),
    (dict(x=t(2, 0)), ValueError, r"1 to 2\^22 values"), (dict(x=t()), ValueError, r"1 to 2\^22"),
    (dict(x=t(2, 8, dtype=torch.float64)), TypeError, "got Double"),
    (dict(residual=t(2, 7)), ValueError, r"residual must be \(2, 8\), got \(2, 7\)"),
    (dict(residual=t(8)), ValueError, r"residual must be \(2, 8\), got \(8,\)"),
    (dict(residual=t(2, 8, dtype=HF)), TypeError, "residual must be bfloat16 or float32, got float16")])
def test_dropout_checks(kw, err, msg):
    args = dict(x=t(2, 8), p=0.1, seed=3)
    args.update(kw)
    with pytest.raises(err, match=msg):
        train.dropout(**args)


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, DEVICE), (dict(x=t(2, 8)), ValueError, DEVICE), (dict(gate=t(2, 8), scale=t(8, dtype=F32)), ValueError, DEVICE),
    (dict(post_weight=t(8, dtype=F32), post_bias=t(8, dtype=F32), bias=t(8, dtype=F32), p=0.5), ValueError, DEVICE),
    (dict(weight=t(8)), ValueError, DEVICE),
    (dict(x=t(2, 8, dtype=HF)), TypeError, "x must be float32 or bfloat16 as o, got float16"),
    (dict(o=t(2, 8, dtype=F32), x=t(2, 8)), TypeError, "x must be float32 or float32 as o"),
    (dict(o=t(2, 7)), ValueError, r"o \(2, 7\) must be \(2, 8\) as x"),
    (dict(gate=t(8)), ValueError, r"gate \(8,\) must be \(2, 8\)"),
    (dict(gate=t(2, 8, dtype=F32)), TypeError, "gate is float32, o bfloat16"),
    (dict(weight=t(7, dtype=F32)), ValueError, r"weight must be \[8\], got \(7,\)"),
    (dict(weight=t(8, dtype=HF)), TypeError, "weight is float16; the vectors share float32 or bfloat16"),
    (dict(scale=t(8)), TypeError, "scale is bfloat16; the vectors share"),
    (dict(scale=t(1, dtype=F32)), ValueError, r"scale must be \[8\], got \(1,\)"),
    (dict(bias=t(2, 8, dtype=F32)), ValueError, r"bias must be \[8\]"),
    (dict(post_bias=t(8, dtype=F32)), ValueError, "post_bias without post_weight"),
    (dict(p=2), ValueError, "p must be 0 to 1"), (dict(seed=-5), ValueError, "seed must be an integer"),
    (dict(x=t(2, 8193, dtype=F32), o=t(2, 8193)), ValueError, "1 to 8192 values"),
    (dict(x=t(2, 0, dtype=F32), o=t(2, 0)), ValueError, "1 to 8192 values"),
    (dict(weight=None), TypeError, "weight must be a tensor"), (dict(eps=None), TypeError, "real number")])
def test_block_join_checks(kw, err, msg):
    args = dict(x=t(2, 8, dtype=F32), o=t(2, 8), weight=t(8, dtype=F32))
    args.update(kw)
    with pytest.raises(err, match=msg):
        train.block_join(**args)


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, DEVICE), (dict(o=t(2, 128)), ValueError, DEVICE), (dict(r_k=t(2, 64, dtype=F32)), ValueError, DEVICE),
    (dict(o=t(2, 100)), ValueError, "1 to 1024 heads of 64"), (dict(o=t(2, 0)), ValueError, "heads of 64"),
    (dict(o=t(2, 65600)), ValueError, "heads of 64"),
    (dict(k=t(2, 64)), ValueError, r"k must be \(2, 128\) as o, got \(2, 64\)"),
    (dict(gate=t(3, 128)), ValueError, r"gate must be \(2, 128\)"),
    (dict(v=t(2, 128, dtype=F32)), TypeError, "v is float32, r bfloat16"),
    (dict(o=t(2, 128, dtype=HF)), TypeError, "o must be float32 or bfloat16 as r, got float16"),
    (dict(r_k=t(64, 2, dtype=F32)), ValueError, r"r_k must be \[128\], got \(64, 2\)"),
    (dict(bias=t(128)), TypeError, "bias is bfloat16; the vectors share"),
    (dict(weight=t(64, dtype=F32)), ValueError, r"weight must be \[128\]"),
    (dict(bias=None), TypeError, "bias must be a tensor")])
def test_wkv_tail_checks(kw, err, msg):
    args = dict(o=t(2, 128, dtype=F32), r=t(2, 128), k=t(2, 128), v=t(2, 128), r_k=t(128, dtype=F32), gate=t(2, 128),
                weight=t(128, dtype=F32), bias=t(128, dtype=F32))
    args.update(kw)
    with pytest.raises(err, match=msg):
        train.wkv_tail(**args)


CALLS = {"gated_linear": lambda a: train.gated_linear(a, t(4, 64)), "dropout": lambda a: train.dropout(a, 0.1, 1),
         "block_join": lambda a: train.block_join(a, t(2, 64), t(64))[0],
         "wkv_tail": lambda a: train.wkv_tail(t(2, 64), a, t(2, 64), t(2, 64), t(64), t(2, 64), t(64), t(64))}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_transforms_and_tracing_are_refused(name):
    f = CALLS[name]
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
            f(torch.autograd.forward_ad.make_dual(t(2, 64), torch.ones_like(t(2, 64))))
    with pytest.raises(NotImplementedError, match=f"{name}: .*transforms"):
        torch.vmap(f)(t(3, 2, 64))
    with pytest.raises(NotImplementedError, match=f"{name}: .*transforms"):
        torch.func.vjp(f, t(2, 64))
    with pytest.raises(NotImplementedError, match=f"{name}: .*tracing"):
        torch.jit.trace(f, t(2, 64), check_trace=False)
    with torch._subclasses.FakeTensorMode() as m:
        with pytest.raises(NotImplementedError, match=f"{name}: .*tracing"):
            f(m.from_tensor(t(2, 64)))


# ───────────────────────────── gated products ─────────────────────────────

def test_gated_entries_refuse():
    lib = _lib.lib()
    fwd = lambda **k: [k.get("x", D), k.get("ldx", 8), D, k.get("ldw", 8), k.get("h", D), k.get("aux"), k.get("rem"), k.get("act", 2),  # noqa: E731
                       k.get("dt", 1), k.get("M", 2), k.get("F", 4), k.get("K", 8), k.get("ws"), k.get("wsn", 0), None]
    refused(DTYPE, "rwkv_gated_fwd", *fwd(dt=0))
    refused(UNSUP, "rwkv_gated_fwd", *fwd(act=4))
    refused(UNSUP, "rwkv_gated_fwd", *fwd(act=-1))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(K=0))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(F=0))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(F=(1 << 19) + 1))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(F=1 << 62))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(M=-1))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(ldx=7))
    refused(SHAPE, "rwkv_gated_fwd", *fwd(ldw=1 << 22))
    refused(NULL, "rwkv_gated_fwd", *fwd(x=None))
    refused(NULL, "rwkv_gated_fwd", *fwd(h=None))
    refused(NULL, "rwkv_gated_fwd", *fwd(aux=D))
    refused(NULL, "rwkv_gated_fwd", *fwd(rem=D))
    refused(OK, "rwkv_gated_fwd", *fwd(M=0, x=None))
    need = lib.rwkv_gated_fwd_workspace(256, 64, 16384)
    assert need > 0 and lib.rwkv_gated_fwd_workspace(1, 64, 64) == 0 and lib.rwkv_gated_fwd_workspace(-1, 64, 64) == 0
    for ws in ((None, need), (D, need - 1), (D + 4, need)):
        refused(SHAPE, "rwkv_gated_fwd", *fwd(M=256, F=64, K=16384, ldx=16384, ldw=16384, ws=ws[0], wsn=ws[1]))
    dact = lambda **k: [k.get("dy", D), k.get("lddy", 4), k.get("kept", D), k.get("rem", D), k.get("act", 2), k.get("dz", D),  # noqa: E731
                        k.get("ldz", 8), k.get("dt", 1), k.get("M", 2), k.get("F", 4), None]
    refused(DTYPE, "rwkv_gated_dact", *dact(dt=0))
    refused(UNSUP, "rwkv_gated_dact", *dact(act=7))
    refused(SHAPE, "rwkv_gated_dact", *dact(lddy=3))
    refused(SHAPE, "rwkv_gated_dact", *dact(ldz=7))
    refused(SHAPE, "rwkv_gated_dact", *dact(ldz=16))
    refused(SHAPE, "rwkv_gated_dact", *dact(F=0))
    for n in ("dy", "kept", "rem", "dz"):
        refused(NULL, "rwkv_gated_dact", *dact(**{n: None}))
    refused(OK, "rwkv_gated_dact", *dact(M=0, dy=None))


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, DEVICE), (dict(x=t(8)), ValueError, DEVICE), (dict(activation="relu2"), ValueError, DEVICE),
    (dict(x=t(2, 8, dtype=F32), weight=t(4, 8, dtype=F32)), TypeError, "x must be bfloat16 or float16, got float32"),
    (dict(weight=t(5, 8)), ValueError, r"weight \(5, 8\) must be \[..., K\] and \[2F, K\]"),
    (dict(weight=t(4, 7)), ValueError, r"weight \(4, 7\) must be"), (dict(weight=t(0, 8)), ValueError, r"weight \(0, 8\) must be"),
    (dict(weight=t(4)), ValueError, r"weight \(4,\) must be"), (dict(x=t()), ValueError, "must be"),
    (dict(weight=t(4, 8, dtype=HF)), TypeError, "weight is float16, x bfloat16"),
    (dict(activation="gelu"), ValueError, "'gelu' is none of"), (dict(activation=None), ValueError, "is none of"),
    (dict(weight=None), TypeError, "weight must be a tensor")])
def test_gated_linear_checks(kw, err, msg):
    args = dict(x=t(2, 8), weight=t(4, 8))
    args.update(kw)
    with pytest.raises(err, match=msg):
        train.gated_linear(**args)
