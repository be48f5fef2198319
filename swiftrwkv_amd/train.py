"""Differentiable operators around the WKV-7 recurrence, for training on
MI355X: layer norm, dense products with bias / activation / residual, and
8-bit activation checkpoints that their backward passes read.

The reference forms these from MLX operations and differentiates them with
MLX's autograd (RWKVBlock.rwkvTmixForward / rwkvCmixForward,
Sources/RWKVModel/RWKVBlock.swift:163-307); here each is hand-written kernels
behind the C ABI.  channel_mix runs them together as one block half.

Tensors live on a ROCm device; results and gradients come back in the types
of the arguments.  Leading axes are rows; a last axis that is not contiguous is
copied first.  There is no CPU fallback: a missing library raises.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DT = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_HALF = (torch.bfloat16, torch.float16)
ACTIVATIONS = {"none": 0, "relu2": 1, "tanh": 2, "sigmoid": 3}
_RELU2 = ACTIVATIONS["relu2"]

_stream = _lib.stream


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, what: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise ValueError(f"{what} must live on a ROCm device, got {t.device}")
    if t.dtype not in _DT:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")


def _same_device(a: torch.Tensor, b: torch.Tensor, what: str) -> None:
    if a.device != b.device:
        raise ValueError(f"{what} is on {b.device}, the input on {a.device}")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """t as rows [N, D] with their pitch: a view where the last axis is
    contiguous and the rows are evenly apart, else a copy."""
    D = t.shape[-1]
    t2 = t if t.dim() == 2 else t.reshape(-1, D)
    if t2.shape[0] <= 1:
        return (t2, D) if t2.stride(1) == 1 or D == 1 else (t2.contiguous(), D)
    if (t2.stride(1) != 1 and D > 1) or t2.stride(0) < D:
        t2 = t2.contiguous()
    return t2, t2.stride(0)


def _workspace(nbytes: int, device) -> Tuple[Optional[torch.Tensor], int]:
    return (torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes) if nbytes else (None, 0)


# ───────────────────────────── 8-bit checkpoints ─────────────────────────────

class Checkpoint8:
    """An activation in 8 bits (MXINT8: groups of 32 values along the last axis
    share a power of two): codes int8 [rows, width], scales uint8
    [rows, width/32], with the shape and type of what it stands for."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, torch.Size(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def restore(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values the codes stand for, in `dtype` (default: the type they
        were taken from).  Exact in float32 and bfloat16; float16 rounds steps
        under 2^-24."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DT:
            raise TypeError(f"checkpoints restore to float32, bfloat16 or float16, not {dtype}")
        y = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        _lib.call("rwkv_act8_unpack", _p(self.codes), _p(self.scales), _p(y), _DT[dtype], self.codes.shape[0],
                  self.shape[-1], _stream(self.codes))
        return y


def _codes(N: int, D: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    W = (D + 31) // 32 * 32
    return (torch.empty((N, W), dtype=torch.int8, device=device),
            torch.empty((N, W // 32), dtype=torch.uint8, device=device))


def checkpoint8(x: torch.Tensor) -> Checkpoint8:
    """x [..., D] (float32, bfloat16 or float16) in 8 bits.  With 2^e the
    largest power of two not above a group's largest magnitude, a value is
    kept to half a step of 2^(e-6) (one step at the group's very top); a group
    holding an infinity or a NaN restores as NaN.  Not differentiable: it is
    what a backward pass keeps."""
    _need(x, "checkpoint8: x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"checkpoint8: x must have a last axis of at least 1, got {tuple(x.shape)}")
    xr, ld = _rows(x.detach())
    N, D = xr.shape
    codes, scales = _codes(N, D, x.device)
    _lib.call("rwkv_act8_pack", _p(xr), _DT[x.dtype], ld, _p(codes), _p(scales), N, D, _stream(xr))
    return Checkpoint8(codes, scales, x.shape, x.dtype)


# ───────────────────────────── layer norm ─────────────────────────────

def _norm_forward(x, weight, bias, eps, out_dtype, stats, keep8):
    xr, ld = _rows(x)
    N, D = xr.shape
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    st = torch.empty((N, 2), dtype=torch.float32, device=x.device) if stats else None
    codes, scales = _codes(N, D, x.device) if keep8 else (None, None)
    _lib.call("rwkv_norm_fwd", _p(xr), _DT[x.dtype], ld, _p(weight), _p(bias), _DT[weight.dtype], _p(y),
              _DT[out_dtype], _p(st), _p(codes), _p(scales), N, D, eps, _stream(xr))
    return y, xr, st, codes, scales


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype, keep8):
        y, xr, st, codes, scales = _norm_forward(x, weight, bias, eps, out_dtype, True, keep8)
        ctx.shape, ctx.x_dtype, ctx.has_bias = x.shape, x.dtype, bias is not None
        ctx.save_for_backward(None if keep8 else xr, codes, scales, st, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, codes, scales, st, w = ctx.saved_tensors
        D = ctx.shape[-1]
        N = st.shape[0]
        dy = dy.reshape(N, D).contiguous()
        dev = dy.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        need_b = need_b and ctx.has_bias
        dx = torch.empty((N, D), dtype=ctx.x_dtype, device=dev) if need_x else None
        dw = torch.empty(D, dtype=w.dtype, device=dev) if need_w or need_b else None
        db = torch.empty(D, dtype=w.dtype, device=dev) if need_b else None
        ws, wsn = _workspace(_lib.lib().rwkv_norm_bwd_workspace(N, D) if dw is not None else 0, dev)
        ld = D if x is None or N <= 1 else x.stride(0)
        _lib.call("rwkv_norm_bwd", _p(dy), _DT[dy.dtype], _p(x), _DT[ctx.x_dtype], ld, _p(codes), _p(scales), _p(st),
                  _p(w), _DT[w.dtype], _p(dx), _p(dw), _p(db), N, D, _p(ws), wsn, _stream(dy))
        return (None if dx is None else dx.reshape(ctx.shape)), (dw if need_w else None), db, None, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
               out_dtype: Optional[torch.dtype] = None, keep8: bool = False) -> torch.Tensor:
    """Layer norm over the last axis (width at most 65536), differentiable in
    x, weight and bias.  x float32, bfloat16 or float16; weight and bias [D]
    float32 or x's type; the result in `out_dtype` (default x's type; any of
    the three for float32 x).  Statistics and sums are fp32.  keep8: the
    backward pass reads x from an 8-bit checkpoint that the forward pass writes
    beside y (1.03 bytes per value kept), with the exact row's mean and
    deviation.  With no gradient needed nothing is kept."""
    _need(x, "layer_norm: x")
    _need(weight, "layer_norm: weight")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 65536:
        raise ValueError(f"layer_norm: the last axis must hold 1 to 65536 values, got {tuple(x.shape)}")
    D = x.shape[-1]
    if out_dtype not in _DT or (out_dtype != x.dtype and x.dtype != torch.float32):
        raise TypeError(f"layer_norm: {x.dtype} rows give {x.dtype}, not {out_dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _need(t, f"layer_norm: {name}")
        _same_device(x, t, f"layer_norm: {name}")
        if tuple(t.shape) != (D,):
            raise ValueError(f"layer_norm: {name} must be [{D}], got {tuple(t.shape)}")
        if t.dtype not in (torch.float32, x.dtype) or t.dtype != weight.dtype:
            raise TypeError(f"layer_norm: weight and bias must share float32 or {x.dtype}, got {t.dtype}")
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps), out_dtype, bool(keep8))
    return _norm_forward(x, weight, bias, float(eps), out_dtype, False, False)[0]


# ───────────────────────────── dense products ─────────────────────────────

def _linear_forward(x, w, bias, act, residual, aux, keep8):
    """(y, x rows, x pitch, w, w pitch, aux, z codes, z scales)"""
    xr, ldx = _rows(x)
    wr, ldw = _rows(w)
    M, K = xr.shape
    N = wr.shape[0]
    dev = x.device
    res, ldr = (None, 0) if residual is None else _rows(residual)
    y_dt = x.dtype if residual is None else residual.dtype
    y = torch.empty((*x.shape[:-1], N), dtype=y_dt, device=dev)
    ax = torch.empty((M, N), dtype=x.dtype, device=dev) if aux else None
    codes, scales = _codes(M, N, dev) if keep8 else (None, None)
    ws, wsn = _workspace(_lib.lib().rwkv_linear_fwd_workspace(M, N, K), dev)
    _lib.call("rwkv_linear_fwd", _p(xr), ldx, _p(wr), ldw, _p(bias), _p(res), ldr, _p(y), _DT[y_dt], _p(ax), _p(codes),
              _p(scales), act, _DT[x.dtype], M, N, K, _p(ws), wsn, _stream(xr))
    return y, xr, ldx, wr, ldw, ax, codes, scales


class _Linear(torch.autograd.Function):
    """Keeps x (or its checkpoint), W, and of the activation: nothing for
    "none"; y for bfloat16 relu² without a residual (relu(z) = √y, half of y's
    rounding); tanh or σ where y is that; else an extra buffer of relu(z),
    tanh(z) or σ(z) (float16 relu² too: its squares underflow early); or with
    keep8 the 8-bit checkpoint of z."""

    @staticmethod
    def forward(ctx, x, w, bias, residual, act, keep8):
        z8 = keep8 and act != 0
        from_y = not z8 and act != 0 and residual is None and not (act == _RELU2 and x.dtype == torch.float16)
        aux = act != 0 and not z8 and not from_y
        y, xr, ldx, wr, ldw, ax, codes, scales = _linear_forward(x, w, bias, act, residual, aux, z8)
        x8 = checkpoint8(xr) if keep8 and ctx.needs_input_grad[1] else None
        keep_x = xr if not keep8 and ctx.needs_input_grad[1] else None
        ctx.x_shape, ctx.dtype, ctx.act, ctx.from_y = x.shape, x.dtype, act, from_y
        ctx.MNK, ctx.ldx, ctx.ldw, ctx.y_dtype = (xr.shape[0], wr.shape[0], xr.shape[1]), ldx, ldw, y.dtype
        ctx.res_shape = None if residual is None else residual.shape
        ctx.save_for_backward(keep_x, None if x8 is None else x8.codes, None if x8 is None else x8.scales, wr,
                              y if from_y else ax, codes, scales)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, xc, xs, w, kept, zc, zs = ctx.saved_tensors
        M, N, K = ctx.MNK
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dev, dt, lib = dy.device, ctx.dtype, _lib.lib()
        d_res = dy.reshape(ctx.res_shape) if need_r else None
        dyr, lddy = _rows(dy.reshape(M, N))
        s = _stream(dy)
        need_z = need_x or need_w
        db = torch.empty(N, dtype=dt, device=dev) if need_b else None
        dz, ldz = dyr, lddy
        # dy itself serves as dz unless it has to be multiplied, narrowed, or
        # laid out in whole 16-byte chunks (with zeros behind an odd N)
        if need_z and (ctx.act != 0 or dyr.dtype != dt or N % 8 or lddy % 8):
            ldz = (N + 7) // 8 * 8
            dz = torch.empty((M, ldz), dtype=dt, device=dev)
        if dz is not dyr or need_b:
            ws, wsn = _workspace(lib.rwkv_linear_dact_workspace(M, N) if need_b else 0, dev)
            _lib.call("rwkv_linear_dact", _p(dyr), lddy, _DT[dyr.dtype], _p(kept),
                      int(ctx.from_y and ctx.act == _RELU2), _p(zc), _p(zs), ctx.act, None if dz is dyr else _p(dz),
                      ldz, _p(db), _DT[dt], M, N, _p(ws), wsn, s)
        dx = dw = None
        if need_x:
            dx = torch.empty((M, K), dtype=dt, device=dev)
            ws, wsn = _workspace(lib.rwkv_linear_dgrad_workspace(M, N, K), dev)
            _lib.call("rwkv_linear_dgrad", _p(dz), ldz, _p(w), ctx.ldw, _p(dx), _DT[dt], M, N, K, _p(ws), wsn, s)
            dx = dx.reshape(ctx.x_shape)
        if need_w:
            if M == 0:
                dw = torch.zeros((N, K), dtype=dt, device=dev)
            else:
                ldx = ctx.ldx
                if xc is not None:
                    x, ldx = Checkpoint8(xc, xs, (M, K), dt).restore(), K
                dw = torch.empty((N, K), dtype=dt, device=dev)
                ws, wsn = _workspace(lib.rwkv_linear_wgrad_workspace(M, N, K), dev)
                _lib.call("rwkv_linear_wgrad", _p(dz), ldz, _p(x), ldx, _p(dw), _DT[dt], M, N, K, _p(ws), wsn, s)
        return dx, dw, db, d_res, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, *, keep8: bool = False) -> torch.Tensor:
    """act(x·weightᵀ + bias) + residual, differentiable in all four.

    x [..., K] and weight [N, K], bias [N]: bfloat16 or float16, all alike.
    activation "none", "relu2" (relu(z)², the channel mix's), "tanh" or
    "sigmoid" (the low-rank branches').  residual [..., N] of x's type or
    float32 is added after the activation; the result has its type (x's
    without one).  Products accumulate in fp32 and the result is rounded once.
    The gradient of z is rounded to x's type before its two products, as they
    run on the matrix cores.  keep8: for the backward pass x and, under an
    activation, z are kept in 8 bits instead of 16.  With no gradient needed
    nothing is kept."""
    _need(x, "linear: x")
    _need(weight, "linear: weight")
    if x.dtype not in _HALF:
        raise TypeError(f"linear: x must be bfloat16 or float16, got {x.dtype}")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"linear: activation {activation!r} is none of {', '.join(ACTIVATIONS)}")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError(f"linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} must be [..., K] and [N, K]")
    N = weight.shape[0]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _need(t, f"linear: {name}")
        _same_device(x, t, f"linear: {name}")
        if t.dtype != x.dtype:
            raise TypeError(f"linear: {name} is {t.dtype}, x {x.dtype}")
    if bias is not None and tuple(bias.shape) != (N,):
        raise ValueError(f"linear: bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None:
        _need(residual, "linear: residual")
        _same_device(x, residual, "linear: residual")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"linear: residual must be {x.dtype} or float32, got {residual.dtype}")
        if tuple(residual.shape) != (*x.shape[:-1], N):
            raise ValueError(f"linear: residual must be {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, residual, act, bool(keep8))
    return _linear_forward(x, weight, bias, act, residual, False, False)[0]


# ───────────────────────────── together ─────────────────────────────

def channel_mix(x: torch.Tensor, ln_weight: torch.Tensor, ln_bias: torch.Tensor, x_k: torch.Tensor,
                key: torch.Tensor, value: torch.Tensor, shift: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
                keep8: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The channel-mix half of a block, differentiable (rwkvCmixForward with
    its ln2 and residual, RWKVBlock.swift:275-307): xl = LN(x), the token shift
    xx = previous token's xl − xl, xk = xl + xx·x_k, x + relu(xk·keyᵀ)²·valueᵀ.

    x [B, T, D] float32 (the residual stream) or the weights' type; ln_weight,
    ln_bias [D] float32 or x's type; x_k [D]; key [F, D], value [D, F] bfloat16
    or float16; shift [B, D]: the normed row before the first token (None:
    zeros).  keep8 keeps the norm's x, both products' inputs and the key's
    pre-activation in 8 bits for the backward pass.  Returns (x', the last
    normed row [B, D])."""
    if x.dim() != 3:
        raise ValueError(f"channel_mix: x must be [B, T, D], got {tuple(x.shape)}")
    B, T, D = x.shape
    if T < 1:
        raise ValueError("channel_mix: T must be at least 1")
    xl = layer_norm(x, ln_weight, ln_bias, eps, out_dtype=key.dtype, keep8=keep8)
    first = xl.new_zeros((B, 1, D)) if shift is None else shift.to(xl.dtype).reshape(B, 1, D)
    xk = torch.lerp(xl, torch.cat([first, xl[:, :-1]], dim=1), x_k.to(xl.dtype))
    h = linear(xk, key, activation="relu2", keep8=keep8)
    return linear(h, value, residual=x, keep8=keep8), xl[:, -1]
