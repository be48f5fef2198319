"""Differentiable operators around the WKV-7 recurrence, for training on
MI355X: layer norm, dense products with bias / activation / residual, and
8-bit activation checkpoints that their backward passes read.

The reference forms these from MLX operations and differentiates them with
MLX's autograd (RWKVBlock.rwkvTmixForward / rwkvCmixForward,
Sources/RWKVModel/RWKVBlock.swift:163-307); here each is hand-written kernels
behind the C ABI.  channel_mix runs them together as one block half.

Tensors live on a ROCm device; results and gradients come back in the types
of the arguments.  Leading axes are rows, at most 2^24; a last axis that is not
contiguous is copied first.  Checks, allocations and autograd nodes are native code
(csrc/train_ext.cpp).  Gradients of gradients, forward-mode derivatives, tracing
and function transforms raise.  There is no CPU fallback: a missing library raises.
"""
from __future__ import annotations

import importlib
import os
from typing import Optional, Tuple

import torch

from . import _lib

ACTIVATIONS = ("none", "relu2", "tanh", "sigmoid")

_ext = None


def extension():
    """The native module behind this one (raises if it has not been built)."""
    global _ext
    if _ext is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_train.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -m swiftrwkv_amd.build` "
                               "(there is no CPU fallback for the HIP path)")
        _lib.lib()
        _ext = importlib.import_module("swiftrwkv_amd._train")
        _ext.set_error(_lib.RwkvHipError)
    return _ext


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
        return (_ext or extension()).restore8(self.codes, self.scales, self.shape, dtype or self.dtype)


def checkpoint8(x: torch.Tensor) -> Checkpoint8:
    """x [..., D] (float32, bfloat16 or float16) in 8 bits.  With 2^e the
    largest power of two not above a group's largest magnitude, a value is
    kept to half a step of 2^(e-6) (one step at the group's very top); a group
    holding an infinity or a NaN restores as NaN.  Not differentiable: it is
    what a backward pass keeps."""
    codes, scales = (_ext or extension()).checkpoint8(x)
    return Checkpoint8(codes, scales, x.shape, x.dtype)


# ───────────────────────────── layer norm ─────────────────────────────

def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5, *,
               out_dtype: Optional[torch.dtype] = None, keep8: bool = False) -> torch.Tensor:
    """Layer norm over the last axis (width at most 65536), differentiable in
    x, weight and bias.  x float32, bfloat16 or float16; weight and bias [D]
    float32 or x's type; the result in `out_dtype` (default x's type; any of
    the three for float32 x).  Statistics and sums are fp32.  keep8: the
    backward pass reads x from an 8-bit checkpoint that the forward pass writes
    beside y (1.03 bytes per value kept), with the exact row's mean and
    deviation.  With no gradient needed nothing is kept."""
    return (_ext or extension()).layer_norm(x, weight, bias, eps, out_dtype, keep8)


# ───────────────────────────── dense products ─────────────────────────────

def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, *, keep8: bool = False) -> torch.Tensor:
    """act(x·weightᵀ + bias) + residual, differentiable in all four.

    x [..., K] and weight [N, K], bias [N]: bfloat16 or float16, all alike.
    activation "none", "relu2" (relu(z)², the channel mix's), "tanh" or
    "sigmoid" (the low-rank branches').  residual [..., N] of x's type or
    float32 is added after the activation; the result has its type (x's
    without one).  Products accumulate in fp32 and the result is rounded once.
    The gradient of z is rounded to x's type before its two products, as they
    run on the matrix cores.  For it an activation keeps 3 bytes per value
    (bfloat16 relu² without a residual 1, beside y).  keep8:
    x and, under an activation, z are kept in 8 bits instead.  With no gradient
    needed nothing is kept.  With more than 128 rows and from M·N·K = 2^30 on, x and
    weight whose rows are not whole 16-byte chunks (K not a multiple of 8, or
    misaligned) are copied into such rows first, and a backward pass keeps the
    copies."""
    return (_ext or extension()).linear(x, weight, bias, activation, residual, keep8)


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
