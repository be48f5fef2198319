"""Training-side operators, CPU part: what the C entries and the Python
wrappers refuse (before any launch), and the 8-bit format's definition."""
import pytest
import torch

from swiftrwkv_amd import _lib, train

D = 64   # a dummy, 16-byte aligned address: refused calls never reach a launch


def refused(status, name, *args):
    assert getattr(_lib.lib(), name)(*args) == status, (name, args, _lib.lib().rwkv_last_error())


SHAPE, DTYPE, UNSUP, NULL = 1, 2, 3, 6


def test_act8_entries_refuse():
    lib = _lib.lib()
    assert [lib.rwkv_act8_width(d) for d in (-1, 0, 1, 32, 33)] == [0, 0, 32, 32, 64]
    refused(DTYPE, "rwkv_act8_pack", D, 3, 8, D, D, 1, 8, None)
    refused(SHAPE, "rwkv_act8_pack", D, 0, 7, D, D, 1, 8, None)       # pitch below the width
    refused(SHAPE, "rwkv_act8_pack", D, 0, 8, D, D, -1, 8, None)
    refused(SHAPE, "rwkv_act8_pack", D, 0, 8, D, D, 1, 0, None)
    refused(NULL, "rwkv_act8_pack", D, 0, 8, None, D, 1, 8, None)
    refused(NULL, "rwkv_act8_unpack", D, None, D, 0, 1, 8, None)
    refused(0, "rwkv_act8_pack", None, 0, 8, None, None, 0, 8, None)  # no rows: nothing to do
    refused(0, "rwkv_act8_unpack", None, None, None, 0, 0, 8, None)


def test_norm_entries_refuse():
    fwd = lambda **k: [k.get("x", D), k.get("xdt", 0), k.get("ldx", 8), D, D, k.get("wdt", 0), D, k.get("ydt", 0), D,  # noqa: E731
                       k.get("codes"), k.get("scales"), k.get("N", 1), k.get("D", 8), 1e-5, None]
    refused(DTYPE, "rwkv_norm_fwd", *fwd(xdt=1, ydt=0))      # bf16 rows into fp32
    refused(DTYPE, "rwkv_norm_fwd", *fwd(xdt=1, ydt=1, wdt=2))
    refused(DTYPE, "rwkv_norm_fwd", *fwd(xdt=5))
    refused(SHAPE, "rwkv_norm_fwd", *fwd(D=65537, ldx=65537))
    refused(SHAPE, "rwkv_norm_fwd", *fwd(D=0))
    refused(SHAPE, "rwkv_norm_fwd", *fwd(ldx=7))
    refused(NULL, "rwkv_norm_fwd", *fwd(x=None))
    refused(NULL, "rwkv_norm_fwd", *fwd(codes=D))            # without scales
    refused(0, "rwkv_norm_fwd", *fwd(N=0, x=None))
    bwd = lambda **k: [D, k.get("ydt", 0), k.get("x", D), k.get("xdt", 0), 8, None, None, D, D, 0, D, k.get("dw", D),  # noqa: E731
                       k.get("db", D), k.get("N", 4), 8, k.get("ws", D), k.get("wsn", 1 << 20), None]
    refused(DTYPE, "rwkv_norm_bwd", *bwd(xdt=2, ydt=1))
    refused(NULL, "rwkv_norm_bwd", *bwd(x=None))             # neither x nor a checkpoint
    refused(NULL, "rwkv_norm_bwd", *bwd(dw=None))            # db without dw
    need = _lib.lib().rwkv_norm_bwd_workspace(4, 8)
    assert need >= 2 * 8 * 4
    refused(SHAPE, "rwkv_norm_bwd", *bwd(wsn=need - 1))
    refused(SHAPE, "rwkv_norm_bwd", *bwd(ws=None))
    refused(SHAPE, "rwkv_norm_bwd", *bwd(ws=D + 4))          # misaligned


def test_linear_entries_refuse():
    lib = _lib.lib()
    fwd = lambda **k: [k.get("x", D), k.get("ldx", 8), D, k.get("ldw", 8), None, k.get("res"), k.get("ldr", 0), D,  # noqa: E731
                       k.get("ydt", 1), k.get("aux"), k.get("rem"), k.get("codes"), None, k.get("act", 0), k.get("dt", 1), k.get("M", 2),
                       k.get("N", 4), k.get("K", 8), k.get("ws"), k.get("wsn", 0), None]
    refused(DTYPE, "rwkv_linear_fwd", *fwd(dt=0, ydt=0))
    refused(DTYPE, "rwkv_linear_fwd", *fwd(ydt=2))
    refused(UNSUP, "rwkv_linear_fwd", *fwd(act=4))
    refused(UNSUP, "rwkv_linear_fwd", *fwd(act=-1))
    refused(SHAPE, "rwkv_linear_fwd", *fwd(K=0))
    refused(SHAPE, "rwkv_linear_fwd", *fwd(N=0))
    refused(SHAPE, "rwkv_linear_fwd", *fwd(ldx=7))
    refused(SHAPE, "rwkv_linear_fwd", *fwd(ldw=1 << 22))
    refused(SHAPE, "rwkv_linear_fwd", *fwd(res=D, ldr=3))
    refused(NULL, "rwkv_linear_fwd", *fwd(x=None))
    refused(NULL, "rwkv_linear_fwd", *fwd(codes=D))
    refused(NULL, "rwkv_linear_fwd", *fwd(aux=D))            # without remainders
    refused(UNSUP, "rwkv_linear_fwd", *fwd(rem=D, ydt=0))    # remainders of an fp32 y
    refused(UNSUP, "rwkv_linear_fwd", *fwd(rem=D, res=D, ldr=4))
    refused(0, "rwkv_linear_fwd", *fwd(M=0, x=None))
    # a shape that sums ranges of K refuses a workspace that is short
    M, N, K = 256, 64, 16384
    need = lib.rwkv_linear_wgrad_workspace(K, M, N)
    assert need > 0 and need % 4 == 0
    for name in ("dgrad", "wgrad"):
        entry = "rwkv_linear_" + name
        refused(DTYPE, entry, D, 8, D, 8, D, 0, 8, 8, 8, None, 0, None)
        refused(SHAPE, entry, D, 7, D, 8, D, 1, 8, 8, 8, None, 0, None)
        refused(NULL, entry, None, 8, D, 8, D, 1, 8, 8, 8, None, 0, None)
    refused(SHAPE, "rwkv_linear_wgrad", D, 8, D, 8, D, 1, 0, 8, 8, None, 0, None)   # no rows to sum
    refused(SHAPE, "rwkv_linear_pad", D, 6, D, 2, 7, None)
    refused(SHAPE, "rwkv_linear_pad", D, 7, D, -1, 7, None)
    refused(NULL, "rwkv_linear_pad", D, 7, D + 8, 2, 7, None)      # misaligned output
    refused(0, "rwkv_linear_pad", None, 7, None, 0, 7, None)
    refused(SHAPE, "rwkv_linear_wgrad", D, M, D, N, D, 1, K, M, N, D, need // 2 - 4, None)
    dact = lambda **k: [D, k.get("ld", 8), k.get("dydt", 1), k.get("kept"), k.get("rem", k.get("kept")), k.get("isy", 0), k.get("codes"), k.get("scales"),  # noqa: E731
                        k.get("act", 0), D, k.get("ldz", 8), k.get("db"), 1, 2, 8, None, 0, None]
    refused(NULL, "rwkv_linear_dact", *dact(act=1))                      # nothing kept
    refused(NULL, "rwkv_linear_dact", *dact(act=1, kept=D, rem=None))
    refused(NULL, "rwkv_linear_dact", *dact(act=1, kept=D, codes=D, scales=D))
    refused(UNSUP, "rwkv_linear_dact", *dact(act=2, kept=D, isy=1))
    refused(SHAPE, "rwkv_linear_dact", *dact(ldz=16))
    refused(SHAPE, "rwkv_linear_dact", *dact(ld=7))
    refused(DTYPE, "rwkv_linear_dact", *dact(dydt=2))
    refused(SHAPE, "rwkv_linear_dact", *dact(db=D))                      # no workspace


def test_wrappers_refuse():
    h = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match="ROCm device"):
        train.layer_norm(torch.zeros(2, 8), torch.ones(8))
    with pytest.raises(ValueError, match="ROCm device"):
        train.linear(h(2, 8), h(4, 8))
    with pytest.raises(ValueError, match="ROCm device"):
        train.checkpoint8(torch.zeros(2, 8))
    with pytest.raises(TypeError, match="tensor"):
        train.checkpoint8([1.0])
    with pytest.raises(ValueError, match=r"\[B, T, D\]"):
        train.channel_mix(h(2, 8), h(8), h(8), h(8), h(16, 8), h(8, 16))


class Fake(torch.Tensor):
    """A CPU tensor that says it is on the device, for checks before a launch."""
    @property
    def device(self):
        return torch.device("cuda:0")


def fake(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype).as_subclass(Fake)


@pytest.mark.parametrize("kw,err", [
    (dict(weight=fake(7)), ValueError), (dict(weight=fake(8, dtype=torch.float16)), TypeError),
    (dict(bias=fake(8, dtype=torch.float32)), TypeError),        # another type than the weight's
    (dict(out_dtype=torch.float16), TypeError), (dict(x=fake(2, 0), weight=fake(0)), ValueError),
    (dict(x=fake(2, 65537), weight=fake(65537)), ValueError), (dict(x=fake(2, 8, dtype=torch.float64)), TypeError)])
def test_layer_norm_refuses(kw, err):
    args = dict(x=fake(2, 8), weight=fake(8))
    args.update(kw)
    with pytest.raises(err):
        train.layer_norm(**args)


@pytest.mark.parametrize("kw,err", [
    (dict(x=fake(2, 8, dtype=torch.float32)), TypeError), (dict(weight=fake(4, 7)), ValueError),
    (dict(weight=fake(4, 8, dtype=torch.float16)), TypeError), (dict(weight=fake(4, 8, 1)), ValueError),
    (dict(bias=fake(5)), ValueError), (dict(bias=fake(4, dtype=torch.float32)), TypeError),
    (dict(activation="gelu"), ValueError), (dict(residual=fake(2, 5)), ValueError),
    (dict(residual=fake(2, 4, dtype=torch.float16)), TypeError), (dict(x=fake(2, 0), weight=fake(4, 0)), ValueError)])
def test_linear_refuses(kw, err):
    args = dict(x=fake(2, 8), weight=fake(4, 8))
    args.update(kw)
    with pytest.raises(err):
        train.linear(**args)
