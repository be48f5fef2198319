"""Training-side operators, CPU part: each argument check by its own message,
and what is refused because no derivative would come of it."""
import pytest
import torch

from swiftrwkv_amd import train

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def t(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


# The device is looked at last: a message other than the device's comes of the
# check that it names, and arguments that nothing else is wrong with reach it.
DEVICE = "must live on a ROCm device"


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, DEVICE), (dict(bias=t(8)), ValueError, DEVICE), (dict(x=t(8)), ValueError, DEVICE),
    (dict(x=t(2, 8, dtype=F32), weight=t(8, dtype=F32), out_dtype=HF), ValueError, DEVICE),
    (dict(x=t(2, 65536), weight=t(65536)), ValueError, DEVICE),
    (dict(weight=t(7)), ValueError, r"weight must be \[8\], got \(7,\)"),
    (dict(weight=t(8, 1)), ValueError, r"weight must be \[8\], got \(8, 1\)"),
    (dict(weight=t(8, dtype=HF)), TypeError, "weight and bias must share float32 or bfloat16, got float16"),
    (dict(bias=t(9)), ValueError, r"bias must be \[8\], got \(9,\)"),
    (dict(bias=t(8, dtype=F32)), TypeError, "weight and bias must share .* got float32"),
    (dict(weight=t(8, dtype=F32), bias=t(8)), TypeError, "weight and bias must share .* got bfloat16"),
    (dict(out_dtype=HF), TypeError, "bfloat16 rows give bfloat16, not float16"),
    (dict(x=t(2, 8, dtype=F32), out_dtype=torch.float64), TypeError, "float32 rows give"),
    (dict(out_dtype="bf16"), TypeError, "out_dtype must be a torch.dtype"),
    (dict(x=t(2, 0), weight=t(0)), ValueError, r"1 to 65536 values, got \(2, 0\)"),
    (dict(x=t(2, 65537), weight=t(65537)), ValueError, "1 to 65536 values"),
    (dict(x=t()), ValueError, "1 to 65536 values"),
    (dict(x=t(2, 8, dtype=torch.float64)), TypeError, "x must be float32, bfloat16 or float16, got Double"),
    (dict(x=[1.0]), TypeError, "x must be a tensor, got list"), (dict(weight=None), TypeError, "weight must be a tensor")])
def test_layer_norm_checks(kw, err, msg):
    args = dict(x=t(2, 8), weight=t(8))
    args.update(kw)
    with pytest.raises(err, match=msg):
        train.layer_norm(**args)


@pytest.mark.parametrize("kw,err,msg", [
    ({}, ValueError, DEVICE), (dict(x=t(8)), ValueError, DEVICE), (dict(x=t(3, 2, 8)), ValueError, DEVICE),
    (dict(bias=t(4), residual=t(2, 4, dtype=F32), activation="tanh"), ValueError, DEVICE),
    (dict(x=t(2, 8, dtype=F32)), TypeError, "x must be bfloat16 or float16, got float32"),
    (dict(weight=t(4, 7)), ValueError, r"x \(2, 8\) and weight \(4, 7\) must be"),
    (dict(weight=t(8)), ValueError, r"and weight \(8,\) must be"),
    (dict(weight=t(4, 8, 1)), ValueError, r"and weight \(4, 8, 1\) must be"),
    (dict(weight=t(0, 8)), ValueError, r"and weight \(0, 8\) must be"),
    (dict(x=t(2, 0), weight=t(4, 0)), ValueError, r"and weight \(4, 0\) must be"),
    (dict(weight=t(4, 8, dtype=HF)), TypeError, "weight is float16, x bfloat16"),
    (dict(bias=t(5)), ValueError, r"bias must be \[4\], got \(5,\)"),
    (dict(bias=t(4, 1)), ValueError, r"bias must be \[4\], got \(4, 1\)"),
    (dict(bias=t(4, dtype=F32)), TypeError, "bias is float32, x bfloat16"),
    (dict(activation="gelu"), ValueError, "'gelu' is none of"), (dict(activation=None), ValueError, "is none of"),
    (dict(residual=t(2, 5)), ValueError, r"residual must be \(2, 4\), got \(2, 5\)"),
    (dict(residual=t(1, 4)), ValueError, r"residual must be \(2, 4\), got \(1, 4\)"),
    (dict(residual=t(4)), ValueError, r"residual must be \(2, 4\), got \(4,\)"),
    (dict(residual=t(2, 4, dtype=HF)), TypeError, "residual must be bfloat16 or float32, got float16")])
def test_linear_checks(kw, err, msg):
    args = dict(x=t(2, 8), weight=t(4, 8))
    args.update(kw)
    with pytest.raises(err, match=msg):
        train.linear(**args)


@pytest.mark.parametrize("args,err,msg", [
    ((t(2, 8),), ValueError, DEVICE), ((t(),), ValueError, "last axis of at least 1"),
    ((t(2, 0),), ValueError, r"last axis of at least 1, got \(2, 0\)"), ((t(2, 8, dtype=torch.int8),), TypeError, "got Char")])
def test_checkpoint_checks(args, err, msg):
    with pytest.raises(err, match=msg):
        train.checkpoint8(*args)


def test_restore_checks():
    codes, scales = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.uint8)
    make = lambda c=codes, s=scales, shape=(3, 40), dt=BF: train.Checkpoint8(c, s, shape, dt)  # noqa: E731
    with pytest.raises(ValueError, match="codes must live on a ROCm device"):
        make().restore()
    for bad in (make(shape=(3, 65)), make(shape=(3, 32)), make(shape=(4, 40)), make(shape=()), make(c=codes[:, :32]),
                make(s=scales[:2]), make(s=scales.to(torch.int8)), make(c=codes.to(torch.int16)),
                make(c=torch.zeros(64, 3, dtype=torch.int8).t())):
        with pytest.raises(ValueError, match="does not hold"):
            bad.restore()
    with pytest.raises(TypeError, match="restore to float32"):
        make().restore(torch.float64)


CALLS = {"layer_norm": lambda a, b: train.layer_norm(a, b[0]), "linear": lambda a, b: train.linear(a, b)}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_derivatives_are_refused(name, which):
    """A result without a tangent would read as a derivative of zero."""
    args = [t(2, 8), t(4, 8)]
    with torch.autograd.forward_ad.dual_level():
        args[which] = torch.autograd.forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
            CALLS[name](*args)
    with pytest.raises(ValueError, match=DEVICE):   # the level is closed
        CALLS[name](t(2, 8), t(4, 8))


TRACED = {**CALLS, "checkpoint8": lambda a, b: train.checkpoint8(a).codes}


@pytest.mark.parametrize("name", TRACED)
def test_transforms_and_tracing_are_refused(name):
    """A traced call would be a constant, a transformed one has no memory."""
    f = lambda a: TRACED[name](a, t(4, 8))  # noqa: E731
    with pytest.raises(NotImplementedError, match=f"{name}: .*transforms"):
        torch.vmap(f)(t(3, 2, 8))
    with pytest.raises(NotImplementedError, match=f"{name}: .*transforms"):
        torch.func.vjp(f, t(2, 8))
    with pytest.raises(NotImplementedError, match=f"{name}: .*tracing"):
        torch.jit.trace(f, t(2, 8), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    for mode in ("real", "fake"):
        with pytest.raises(NotImplementedError, match=f"{name}: .*tracing"):
            make_fx(f, tracing_mode=mode)(t(2, 8))
    with torch._subclasses.FakeTensorMode() as m:
        with pytest.raises(NotImplementedError, match=f"{name}: .*tracing"):
            f(m.from_tensor(t(2, 8)))


def test_keep8_has_to_have_a_truth_value():
    """An argument whose truth value raises: its own error, no call."""
    for f in (lambda k: train.layer_norm(t(2, 8), t(8), keep8=k), lambda k: train.linear(t(2, 8), t(4, 8), keep8=k)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            f(torch.zeros(2))
