"""The training-side operators around the recurrence, as measurable cases over their public entry points.

Three operators (swiftrwkv_amd.train):

  norm    layer norm, forward alone or with its gradients (train.layer_norm); keep8: the backward pass reads the
          row from its 8-bit checkpoint
  ckpt    an activation into its 8-bit checkpoint and back (train.checkpoint8)
  linear  act(x Wᵀ + b) + residual, forward alone or with its gradients (train.linear); keep8: the weight's gradient
          reads x, and the activation's derivative the pre-activation, from 8-bit checkpoints

An 8-bit checkpoint holds groups of 32 values along the row: with 2^e the largest power of two that is not above the
group's largest magnitude, the codes are the values over 2^(e-6), rounded to the nearest integer (ties to even) and
clamped to ±127 (MXINT8 of the OCP microscaling formats).
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
GROUP = 32


# ───────────────────────────── the cases ─────────────────────────────

def listed():
    return [
        # one token's norm of a 0.4B-wide model while it answers: the smallest call there is
        {"name": "norm_token", "kind": "norm", "rows": 1, "width": 1024, "dtype": "f32", "out": "f32", "weights": "f32",
         "bias": True, "keep8": False, "train": False},
        # a training batch of the 1.5B width, bf16 with fp32 weights
        {"name": "norm_train", "kind": "norm", "rows": 8192, "width": 2048, "dtype": "bf16", "out": "bf16",
         "weights": "f32", "bias": True, "keep8": False, "train": True},
        # a ragged batch of an odd width, all in fp16, no bias
        {"name": "norm_odd", "kind": "norm", "rows": 1001, "width": 1531, "dtype": "f16", "out": "f16",
         "weights": "f16", "bias": False, "keep8": False, "train": True},
        # a long batch of the 7B-class width from an fp32 residual stream into bf16, the row kept in 8 bits
        {"name": "norm_long_keep8", "kind": "norm", "rows": 32768, "width": 4096, "dtype": "f32", "out": "bf16",
         "weights": "f32", "bias": True, "keep8": True, "train": True},
        # one sequence's activations parked in 8 bits and taken back
        {"name": "ckpt_seq", "kind": "ckpt", "rows": 512, "width": 1024, "dtype": "bf16"},
        # a training batch's ffn activations of the 1.5B width parked in 8 bits and taken back
        {"name": "ckpt_batch", "kind": "ckpt", "rows": 16384, "width": 8192, "dtype": "bf16"},
        # one token through a 0.4B ffn key: relu² of a matrix-vector product
        {"name": "linear_token", "kind": "linear", "rows": 1, "in": 1024, "out": 4096, "dtype": "f16", "act": "relu2",
         "bias": False, "residual": "", "keep8": False, "train": False},
        # sixteen sequences decoded together through a 7B-class ffn value, added to the fp32 residual stream
        {"name": "linear_tokens", "kind": "linear", "rows": 16, "in": 14336, "out": 4096, "dtype": "bf16",
         "act": "none", "bias": False, "residual": "f32", "keep8": False, "train": False},
        # the first half of a low-rank branch (decay) in training: a narrow product under tanh
        {"name": "linear_lowrank", "kind": "linear", "rows": 8192, "in": 2048, "out": 96, "dtype": "bf16",
         "act": "tanh", "bias": True, "residual": "", "keep8": False, "train": True},
        # a ragged batch with odd widths on every side
        {"name": "linear_odd", "kind": "linear", "rows": 1003, "in": 1019, "out": 517, "dtype": "f16",
         "act": "sigmoid", "bias": True, "residual": "f16", "keep8": False, "train": True},
        # a training batch through the 1.5B ffn key with both its activations kept in 8 bits
        {"name": "linear_keep8", "kind": "linear", "rows": 8192, "in": 2048, "out": 8192, "dtype": "bf16",
         "act": "relu2", "bias": False, "residual": "", "keep8": True, "train": True},
        # a long training batch through the 7B-class ffn key: the largest products
        {"name": "linear_train", "kind": "linear", "rows": 16384, "in": 4096, "out": 14336, "dtype": "bf16",
         "act": "relu2", "bias": False, "residual": "", "keep8": False, "train": True},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of the time a multiple of 64."""
    n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    return min(hi, max(64, n // 64 * 64)) if n >= 64 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(("norm", "norm", "ckpt", "linear", "linear", "linear"))
    if kind == "linear":
        dt = rng.choice(("bf16", "f16"))
        c = {"kind": kind, "rows": _spread(rng, 1, 16384), "in": _spread(rng, 16, 14336),
             "out": _spread(rng, 16, 14336), "dtype": dt, "act": rng.choice(("none", "relu2", "tanh", "sigmoid")),
             "bias": rng.random() < 0.5, "residual": rng.choice(("", "", dt, "f32")), "keep8": False,
             "train": rng.random() < 0.7}
        c["keep8"] = c["train"] and rng.random() < 0.4
        return c
    rows, width = _spread(rng, 1, 65536), _spread(rng, 32, 8192)
    while rows * width > 1 << 27:
        rows //= 2
    if kind == "ckpt":
        return {"kind": kind, "rows": rows, "width": width, "dtype": rng.choice(("f32", "bf16", "f16"))}
    dt, out = rng.choice((("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")))
    c = {"kind": kind, "rows": rows, "width": width, "dtype": dt, "out": out, "weights": rng.choice(("f32", dt)),
         "bias": rng.random() < 0.7, "keep8": False, "train": rng.random() < 0.7}
    c["keep8"] = c["train"] and rng.random() < 0.5
    return c


# ───────────────────────────── inputs ─────────────────────────────

def _stream_rows(gen, rows, width, dtype):
    """Rows of a residual stream: a row scale and offset of their own, and a few channels far larger than the rest."""
    x = torch.randn((rows, width), generator=gen, device=DEVICE)
    loud = torch.rand(width, generator=gen, device=DEVICE) < 0.01
    x *= torch.where(loud, 12.0, 1.0)
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device=DEVICE))
    x += 0.3 * torch.randn((rows, 1), generator=gen, device=DEVICE)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPE[case["dtype"]]
    rows = case["rows"]
    s = {"case": case}
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)  # noqa: E731
    if case["kind"] == "linear":
        k, n = case["in"], case["out"]
        s["x"] = rand(rows, k).to(dt)
        s["w"] = (rand(n, k) / math.sqrt(k)).to(dt)
        s["b"] = (0.3 * rand(n)).to(dt) if case["bias"] else None
        s["res"] = rand(rows, n).to(DTYPE[case["residual"]]) if case["residual"] else None
        if case["train"]:
            s["dy"] = rand(rows, n).to(DTYPE[case["residual"]] if case["residual"] else dt)
        leaves = [t for t in (s["x"], s["w"], s["b"], s["res"]) if t is not None]
    else:
        d = case["width"]
        s["x"] = _stream_rows(gen, rows, d, dt)
        leaves = []
        if case["kind"] == "norm":
            wdt = DTYPE[case["weights"]]
            s["w"] = (1 + 0.2 * rand(d)).to(wdt)
            s["b"] = (0.2 * rand(d)).to(wdt) if case["bias"] else None
            if case["train"]:
                s["dy"] = rand(rows, d).to(DTYPE[case["out"]])
            leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
    if case.get("train"):
        for t in leaves:
            t.requires_grad_(True)
    s["leaves"] = leaves
    return s


# ───────────────────────────── the operators ─────────────────────────────

def run(state):
    return _call(state) if own else _plain(state)


def _call(s):
    """The calls that a training or serving program makes."""
    from swiftrwkv_amd import train

    c = s["case"]
    if c["kind"] == "ckpt":
        return {"x": train.checkpoint8(s["x"]).restore()}
    if c["kind"] == "norm":
        y = train.layer_norm(s["x"], s["w"], s["b"], EPS, out_dtype=DTYPE[c["out"]], keep8=c["keep8"])
    else:
        y = train.linear(s["x"], s["w"], s["b"], activation=c["act"], residual=s["res"], keep8=c["keep8"])
    if not c["train"]:
        return {"y": y}
    names = [n for n, t in (("dx", s["x"]), ("dw", s["w"]), ("db", s["b"]), ("dres", s.get("res"))) if t is not None]
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, s["leaves"], s["dy"])))}


def _through8(x):
    """The values that the 8-bit checkpoint of the fp32 rows x [rows, width] stands for."""
    rows, width = x.shape
    pad = -width % GROUP
    v = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, GROUP)
    e = torch.frexp(v.abs().amax(-1, keepdim=True)).exponent.clamp(min=-119) - 7
    step = torch.ldexp(torch.ones((), device=x.device), e)
    return (torch.round(v / step).clamp(-127, 127) * step).reshape(rows, -1)[:, :width]


def _act(name, z):
    if name == "relu2":
        return torch.relu(z) * torch.relu(z)
    if name == "tanh":
        return torch.tanh(z)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_slope(name, z):
    if name == "relu2":
        return 2 * torch.relu(z)
    if name == "tanh":
        return 1 - torch.tanh(z) * torch.tanh(z)
    if name == "sigmoid":
        return _act(name, z) * _act(name, -z)
    return torch.ones_like(z)


@torch.no_grad()
def _plain(s):
    """The same from elementary operations in 32 bits, rounded once at the end."""
    c = s["case"]
    x = s["x"].float()
    if c["kind"] == "ckpt":
        return {"x": _through8(x).to(s["x"].dtype)}
    out = {}
    if c["kind"] == "norm":
        w, b = s["w"].float(), s["b"]
        mean = x.mean(-1, keepdim=True)
        rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
        y = (x - mean) * rstd * w
        out["y"] = (y if b is None else y + b.float()).to(DTYPE[c["out"]])
        if c["train"]:
            dy = s["dy"].float()
            xh = ((_through8(x) if c["keep8"] else x) - mean) * rstd
            g = dy * w
            dx = (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * rstd
            out["dx"] = dx.to(s["x"].dtype)
            out["dw"] = (dy * xh).sum(0).to(s["w"].dtype)
            if b is not None:
                out["db"] = dy.sum(0).to(b.dtype)
        return out
    w, b, res = s["w"].float(), s["b"], s["res"]
    z = x @ w.t()
    if b is not None:
        z = z + b.float()
    y = _act(c["act"], z)
    out["y"] = (y if res is None else y + res.float()).to(s["x"].dtype if res is None else res.dtype)
    if c["train"]:
        kept = c["keep8"] and c["act"] != "none"
        dz = s["dy"].float() * _act_slope(c["act"], _through8(z) if kept else z)
        out["dx"] = (dz @ w).to(s["x"].dtype)
        out["dw"] = (dz.t() @ (_through8(x) if c["keep8"] else x)).to(s["w"].dtype)
        if b is not None:
            out["db"] = dz.sum(0).to(b.dtype)
        if res is not None:
            out["dres"] = s["dy"].to(res.dtype)
    return out


# ───────────────────────────── 64 bits ─────────────────────────────

def _kept64(v):
    """The 8-bit checkpoint's values by their definition, in 64 bits: the exponent from the logarithm, put right where
    its rounding crosses a power of two."""
    rows, width = v.shape
    groups = -(-width // GROUP)
    padded = v.new_zeros(rows, groups * GROUP)
    padded[:, :width] = v
    padded = padded.view(rows, groups, GROUP)
    top = padded.abs().max(dim=-1, keepdim=True).values.clamp(min=2.0 ** -120)
    e = torch.floor(torch.log2(top))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
    scaled = padded * torch.exp2(6 - e)
    low = torch.floor(scaled)
    rest = scaled - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
    code = torch.where(up, low + 1, low).clamp(-127, 127)
    return (code * torch.exp2(e - 6)).view(rows, -1)[:, :width]


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda t: None if t is None else t.detach().double()  # noqa: E731
    x = d(s["x"])
    if case["kind"] == "ckpt":
        return {"x": _kept64(x)}
    w, b = d(s["w"]), d(s["b"])
    dy = d(s.get("dy"))
    out = {}
    if case["kind"] == "norm":
        n = x.shape[1]
        dev = x - x.sum(-1, keepdim=True) / n
        std = torch.sqrt((dev * dev).sum(-1, keepdim=True) / n + EPS)
        out["y"] = dev / std * w + (0 if b is None else b)
        if case["train"]:
            xh = (_kept64(x) - (x - dev)) / std if case["keep8"] else dev / std
            g = dy * w
            out["dx"] = (n * g - g.sum(-1, keepdim=True) - xh * (g * xh).sum(-1, keepdim=True)) / (n * std)
            out["dw"] = torch.einsum("rd,rd->d", dy, xh)
            if b is not None:
                out["db"] = dy.sum(0)
        return out
    res = d(s["res"])
    z = torch.mm(x, w.t()) + (0 if b is None else b)
    act = {"none": lambda t: t, "relu2": lambda t: t.clamp(min=0) ** 2, "tanh": torch.tanh,
           "sigmoid": torch.sigmoid}[case["act"]]
    out["y"] = act(z) + (0 if res is None else res)
    if case["train"]:
        at = (_kept64(z) if case["keep8"] and case["act"] != "none" else z).requires_grad_(True)
        dz, = torch.autograd.grad(act(at), at, dy) if case["act"] != "none" else (dy,)
        out["dx"] = torch.mm(dz, w)
        out["dw"] = torch.mm(dz.t(), _kept64(x) if case["keep8"] else x)
        if b is not None:
            out["db"] = dz.sum(0)
        if res is not None:
            out["dres"] = dy
    return out


# ───────────────────────────── what a pass cannot do without ─────────────────────────────

def work(case):
    size = lambda t: DTYPE[t].itemsize  # noqa: E731
    m = case["rows"]
    if case["kind"] == "linear":
        k, n, e = case["in"], case["out"], size(case["dtype"])
        y = size(case["residual"]) if case["residual"] else e
        b = e * n if case["bias"] else 0
        moved = e * (m * k + n * k) + y * m * n * (2 if case["residual"] else 1) + b
        flops = 2 * m * n * k
        if case["train"]:   # dy in; dx, dw, db and the residual's gradient out
            moved += y * m * n * (2 if case["residual"] else 1) + e * (m * k + n * k) + b
            flops *= 3
        return {"bytes": moved, "flops": flops}
    d, e = case["width"], size(case["dtype"])
    if case["kind"] == "ckpt":
        return {"bytes": 2 * e * m * d, "flops": 4 * m * d}
    o, wb = size(case["out"]), size(case["weights"]) * d * (2 if case["bias"] else 1)
    moved = m * d * (e + o) + wb
    if case["train"]:
        moved += m * d * (o + e) + wb
    return {"bytes": moved, "flops": m * d * (20 if case["train"] else 8)}
