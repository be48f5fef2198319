"""Differentiable operators around the WKV-7 recurrence, for training on
MI355X: layer norm, dense products with bias / activation / residual, gated
products, 8-bit activation checkpoints that their backward passes read,
dropout, the join of a block with the next, and the recurrence's tail.

The reference forms the norms, the dense products, the residual sums and the
recurrence's tail from MLX operations and differentiates them with MLX's autograd
(RWKVBlock.rwkvTmixForward / rwkvCmixForward,
Sources/RWKVModel/RWKVBlock.swift:163-307); here each is hand-written kernels
behind the C ABI.  The others are for training on blocks beside the reference's own.
channel_mix and mix_tail run them together as the halves of RWKV-7's block,
gated_mix as the half of one with a gated feed-forward.

Tensors live on a ROCm device; results and gradients come back in the types
of the arguments.  Leading axes are rows, at most 2^24; a last axis that is not
contiguous is copied first.  Checks, allocations and autograd nodes are native code
(csrc/train_ext.cpp).  Gradients of gradients, forward-mode derivatives, tracing
and function transforms raise.  There is no CPU fallback: a missing library raises.
"""
from __future__ import annotations

import importlib
import os
from typing import Optional, Tuple, Union

import torch

from . import _lib

ACTIVATIONS = ("none", "relu2", "tanh", "sigmoid")
GATES = ("relu2", "sigmoid", "silu", "gelu_tanh")

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
    (bfloat16 relu² without a residual 1, beside y); float16 pre-activations past
    65504 are infinities there, as is their relu²'s gradient.  keep8:
    x and, under an activation, z are kept in 8 bits instead.  With no gradient
    needed nothing is kept.  With more than 128 rows and from M·N·K = 2^30 on, x and
    weight whose rows are not whole 16-byte chunks (K not a multiple of 8, or
    misaligned) are copied into such rows first, and a backward pass keeps the
    copies."""
    return (_ext or extension()).linear(x, weight, bias, activation, residual, keep8)


def gated_linear(x: torch.Tensor, weight: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """act(x·Wgᵀ)·(x·Wuᵀ), differentiable in both: the gated half of a
    feed-forward in one product.

    x [..., K] and weight [2F, K], Wg's rows and then Wu's, bfloat16 or float16
    alike; the result [..., F] has their type.  activation "silu" (z·σ(z)),
    "gelu_tanh" (the gelu's tanh form), "sigmoid" or "relu2".  Products
    accumulate in fp32 and the result is rounded once; of a backward pass's two
    products the gradients of both factors are rounded to x's type.  For it 6
    bytes per value of the result are kept (both pre-activations to 16
    significant bits, with fp32's range).  With no gradient needed nothing is kept.  Rows that are
    not whole 16-byte chunks are copied as linear does."""
    return (_ext or extension()).gated_linear(x, weight, activation)


# ───────────────────────────── around a block ─────────────────────────────

def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], *, offset: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """drop(x) + residual, differentiable in both.  x float32, bfloat16 or
    float16 (last axis at most 2^22); residual of x's type or float32; the
    result has its type (x's without one).

    A value is dropped, and then zero whatever it was, where its 16-bit random
    number is under t = round(65536·p); the others are multiplied by
    65536/(65536 − t).  The numbers come from Philox4x32-10 with the key `seed`
    and a counter of the value's row and column in [rows, last axis] and
    `offset`: the same (seed, offset) gives the same mask whatever the type,
    strides or device, so every call of a step has an offset of its own.  The
    mask is never stored; the backward pass draws it again.  seed 0 to 2^64 − 1,
    or an int64 tensor of one value on x's device, which the kernels read as
    they run (a captured graph: what it holds at the replay), and which must
    not change between a forward pass and its backward pass."""
    return (_ext or extension()).dropout(x, p, seed, offset, residual)


def block_join(x: torch.Tensor, o: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
               post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
               gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, p: float = 0.0,
               seed: Union[int, torch.Tensor] = 0, offset: int = 0, eps: float = 1e-5,
               post_eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """The end of one block and the start of the next, in one pass:

        x' = x + scale·drop(gate·LN(o; post_weight, post_bias, post_eps))
        h  = LN(x'; weight, bias, eps)

    differentiable in all eight tensors.  x [..., D] the residual stream
    (float32 or o's type), o the block's result and gate [..., D] of one type
    (float32, bfloat16 or float16), the vectors [D] of one type (float32 or
    o's); D at most 8192.  Without post_weight o is not normed; gate, scale and
    p = 0 leave their factors out; drop as `dropout` has it.  Returns (x' of x's
    type, h of o's).  Statistics and sums are fp32; h comes from x' before its
    rounding.  The backward pass keeps x' (the result), four numbers a row, and
    o and gate where they reach a gradient; with an x of 16 bits x and o, from
    which x' is formed again, unrounded."""
    return (_ext or extension()).block_join(x, o, weight, bias, post_weight, post_bias, gate, scale, p, seed, offset, eps,
                                            post_eps)


def wkv_tail(o: torch.Tensor, r: torch.Tensor, k: torch.Tensor, v: torch.Tensor, r_k: torch.Tensor, gate: torch.Tensor,
             weight: torch.Tensor, bias: torch.Tensor, eps: float = 64e-5) -> torch.Tensor:
    """The time mix's tail (ln_x, the bonus and the gate, RWKVBlock.swift:249-270),
    differentiable in all eight: (LN(o) of every head of 64 · weight + bias +
    (Σ r·k·r_k)·v)·gate.

    o [..., 64 H] the recurrence's result (float32 or r's type); r, k, v, gate
    [..., 64 H] of one type (float32, bfloat16 or float16), which the result
    has; r_k [64 H] or [H, 64], weight and bias [64 H] of one type (float32 or
    r's).  H at most 1024.  Sums are fp32; the backward pass keeps the inputs
    alone.  kernel.wkv_tail is the decode step's, fp32 without gradients."""
    return (_ext or extension()).wkv_tail(o, r, k, v, r_k, gate, weight, bias, eps)


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


def gated_mix(x: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, next_weight: torch.Tensor,
              next_bias: Optional[torch.Tensor] = None, *, activation: str = "silu", post_weight: Optional[torch.Tensor] = None,
              post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
              scale: Optional[torch.Tensor] = None, p: float = 0.0, seed: Union[int, torch.Tensor] = 0, offset: int = 0,
              eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """A gated feed-forward half of a block, differentiable: from the stream x
    [..., D] (float32 or h's type) and its norm h (as the join before returned
    it), o = gated_linear(h, weight, activation)·downᵀ and the block_join of x
    and o.  weight [2F, D], down [D, F] of h's type; the rest as block_join
    has it, next_weight and next_bias the norm of what follows.  Returns
    (x', h')."""
    o = linear(gated_linear(h, weight, activation), down)
    return block_join(x, o, next_weight, next_bias, post_weight=post_weight, post_bias=post_bias, gate=gate, scale=scale, p=p,
                      seed=seed, offset=offset, eps=eps, post_eps=eps)


def mix_tail(x: torch.Tensor, o: torch.Tensor, r: torch.Tensor, k: torch.Tensor, v: torch.Tensor, r_k: torch.Tensor,
             gate: torch.Tensor, ln_weight: torch.Tensor, ln_bias: torch.Tensor, output: torch.Tensor,
             next_weight: torch.Tensor, next_bias: Optional[torch.Tensor] = None, *, scale: Optional[torch.Tensor] = None,
             p: float = 0.0, seed: Union[int, torch.Tensor] = 0, offset: int = 0, eps: float = 1e-5,
             head_eps: float = 64e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """The end of a time-mix half, differentiable (rwkvTmixForward from the
    recurrence's result on, RWKVBlock.swift:249-273): wkv_tail, the output
    projection, and the block_join with the stream x.  o [..., 64 H] from
    kernel.wkv7_train (reshaped), r, k, v, gate [..., 64 H] and output
    [D, 64 H] of one 16-bit type, ln_weight, ln_bias the heads' norm,
    next_weight, next_bias the norm of the half that follows.  Returns
    (x', h)."""
    y = linear(wkv_tail(o, r, k, v, r_k, gate, ln_weight, ln_bias, head_eps), output)
    return block_join(x, y, next_weight, next_bias, scale=scale, p=p, seed=seed, offset=offset, eps=eps)
