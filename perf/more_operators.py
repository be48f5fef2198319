"""What a training block does around its recurrence and its products, as measurable cases over the public entry points.

Four operators (swiftrwkv_amd.train), forward alone or with their gradients:

  dropout  x with its values dropped by a counter-based generator, added to a residual (train.dropout)
  join     the end of a block and the start of the next: x' = x + scale·drop(gate·LN(o)), h = LN(x') (train.block_join)
  tail     the recurrence's head norm, bonus and gate: (LN64(o) + (Σ r·k·r_k)·v)·gate (train.wkv_tail)
  gated    act(x·Wgᵀ)·(x·Wuᵀ) with the rows of Wg and Wu in one weight (train.gated_linear)

The dropped values are those whose 16-bit random number is under t = round(65536·p); the others are multiplied by
65536/(65536 − t).  The numbers of columns 8c .. 8c + 7 of row r are the 128 bits of Philox4x32-10 (Salmon, Moraes, Dror
and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) for the key `seed` and the counter (c, r, offset).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
HEAD, HEAD_EPS = 64, 64e-5
OFFSET = 3 << 32 | 7   # of the calls' random numbers, past 32 bits
GATES = ("relu2", "sigmoid", "silu", "gelu_tanh")


# ───────────────────────────── the cases ─────────────────────────────

def listed():
    return [
        # a short fine-tuning sequence's low-rank input: the smallest call that trains
        {"name": "dropout_small", "kind": "dropout", "rows": 16, "width": 1024, "dtype": "bf16", "residual": "",
         "p": 0.1, "train": True},
        # a ragged batch of an odd width added to an fp32 stream
        {"name": "dropout_odd", "kind": "dropout", "rows": 1001, "width": 1531, "dtype": "f16", "residual": "f32",
         "p": 0.25, "train": True},
        # a long training batch of the 7B-class width added to its fp32 residual stream
        {"name": "dropout_stream", "kind": "dropout", "rows": 32768, "width": 4096, "dtype": "bf16", "residual": "f32",
         "p": 0.1, "train": True},
        # one token of a 0.4B-wide model while it answers: a block's result into the stream, and the next norm
        {"name": "join_token", "kind": "join", "rows": 1, "width": 1024, "stream": "f32", "dtype": "f32",
         "weights": "f32", "bias": True, "post": False, "gate": False, "scale": False, "p": 0.0, "train": False},
        # a ragged batch of an odd width with everything on, all in fp16
        {"name": "join_odd", "kind": "join", "rows": 1003, "width": 1531, "stream": "f16", "dtype": "f16",
         "weights": "f16", "bias": True, "post": True, "gate": True, "scale": True, "p": 0.1, "train": True},
        # a training batch of the 1.5B width: fp32 stream, bf16 branches, norms on both sides, gate, scale and dropout
        {"name": "join_train", "kind": "join", "rows": 16384, "width": 2048, "stream": "f32", "dtype": "bf16",
         "weights": "f32", "bias": True, "post": True, "gate": True, "scale": True, "p": 0.1, "train": True},
        # one token's tail of a 0.4B model
        {"name": "tail_token", "kind": "tail", "rows": 1, "heads": 16, "state": "f32", "dtype": "f32", "weights": "f32",
         "train": False},
        # eight sequences of 4096 tokens of the 1.5B model: fp32 from the recurrence, the rest bf16
        {"name": "tail_train", "kind": "tail", "rows": 32768, "heads": 32, "state": "f32", "dtype": "bf16",
         "weights": "f32", "train": True},
        # one token through the gated half of a 0.4B-wide feed-forward
        {"name": "gated_token", "kind": "gated", "rows": 1, "in": 1024, "out": 4096, "dtype": "f16", "act": "silu",
         "train": False},
        # sixteen sequences decoded together through a 7B-class one
        {"name": "gated_tokens", "kind": "gated", "rows": 16, "in": 4096, "out": 14336, "dtype": "bf16",
         "act": "gelu_tanh", "train": False},
        # a ragged batch with odd widths on every side
        {"name": "gated_odd", "kind": "gated", "rows": 1003, "in": 1019, "out": 517, "dtype": "f16", "act": "relu2",
         "train": True},
        # a long training batch through the 7B-class one: the largest products
        {"name": "gated_train", "kind": "gated", "rows": 16384, "in": 4096, "out": 14336, "dtype": "bf16",
         "act": "silu", "train": True},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, spread over its logarithm; half of the time a multiple of 64."""
    n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    return min(hi, max(64, n // 64 * 64)) if n >= 64 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(("dropout", "join", "join", "tail", "gated", "gated"))
    train = rng.random() < 0.7
    if kind == "gated":
        c = {"kind": kind, "rows": _spread(rng, 1, 16384), "in": _spread(rng, 16, 8192), "out": _spread(rng, 16, 14336),
             "dtype": rng.choice(("bf16", "f16")), "act": rng.choice(GATES), "train": train}
        while c["rows"] * c["in"] * c["out"] > 16384 * 4096 * 14336:
            c["rows"] //= 2
        return c
    rows = _spread(rng, 1, 65536)
    dt = rng.choice(("f32", "bf16", "f16"))
    wide = rng.choice(("f32", dt))
    if kind == "tail":
        heads = round(math.exp(rng.uniform(0, math.log(64))))
        while rows * heads * HEAD > 1 << 26:
            rows //= 2
        return {"kind": kind, "rows": rows, "heads": heads, "state": wide, "dtype": dt, "weights": rng.choice(("f32", dt)),
                "train": train}
    width = _spread(rng, 8, 8192)
    p = round(rng.uniform(0.02, 0.6), 3)
    while rows * width > 1 << (27 if kind == "dropout" else 26):
        rows //= 2
    if kind == "dropout":
        return {"kind": kind, "rows": rows, "width": width, "dtype": dt, "residual": rng.choice(("", "f32", dt)), "p": p,
                "train": train}
    return {"kind": kind, "rows": rows, "width": width, "stream": wide, "dtype": dt, "weights": rng.choice(("f32", dt)),
            "bias": rng.random() < 0.7, "post": rng.random() < 0.5, "gate": rng.random() < 0.5,
            "scale": rng.random() < 0.6, "p": p if train and rng.random() < 0.7 else 0.0, "train": train}


# ───────────────────────────── inputs ─────────────────────────────

def _stream_rows(rand, rows, width):
    """Rows of a residual stream: a size and an offset of their own, and a few channels far larger than the rest."""
    x = rand(rows, width) * torch.exp(0.5 * rand(rows, 1)) + 0.3 * rand(rows, 1)
    return x * torch.where(rand(width).abs() > 2.6, 12.0, 1.0)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)  # noqa: E731
    dt, rows, kind = DTYPE[case["dtype"]], case["rows"], case["kind"]
    leaves, dy = {}, {}   # what gradients are asked for, and what they come from
    if kind == "dropout":
        d = case["width"]
        leaves["x"] = rand(rows, d).to(dt)
        leaves["residual"] = _stream_rows(rand, rows, d).to(DTYPE[case["residual"]]) if case["residual"] else None
        dy["y"] = rand(rows, d).to(DTYPE[case["residual"]] if case["residual"] else dt)
    elif kind == "join":
        d, wdt = case["width"], DTYPE[case["weights"]]
        leaves["x"] = _stream_rows(rand, rows, d).to(DTYPE[case["stream"]])
        leaves["o"] = (0.7 * rand(rows, d) * torch.exp(0.3 * rand(rows, 1))).to(dt)
        leaves["weight"] = (1 + 0.2 * rand(d)).to(wdt)
        leaves["bias"] = (0.2 * rand(d)).to(wdt) if case["bias"] else None
        leaves["post_weight"] = (1 + 0.2 * rand(d)).to(wdt) if case["post"] else None
        leaves["post_bias"] = (0.2 * rand(d)).to(wdt) if case["post"] and case["bias"] else None
        leaves["gate"] = torch.sigmoid(rand(rows, d)).to(dt) if case["gate"] else None
        leaves["scale"] = (0.5 + 0.1 * rand(d)).to(wdt) if case["scale"] else None
        dy["x"], dy["h"] = rand(rows, d).to(DTYPE[case["stream"]]), rand(rows, d).to(dt)
    elif kind == "tail":
        d, wdt = case["heads"] * HEAD, DTYPE[case["weights"]]
        leaves["o"] = (0.4 * rand(rows, d)).to(DTYPE[case["state"]])
        for n in ("r", "k", "v"):
            leaves[n] = (0.6 * rand(rows, d)).to(dt)
        leaves["r_k"] = (0.3 * rand(d)).to(wdt)
        leaves["gate"] = rand(rows, d).to(dt)
        leaves["weight"], leaves["bias"] = (1 + 0.2 * rand(d)).to(wdt), (0.2 * rand(d)).to(wdt)
        dy["y"] = rand(rows, d).to(dt)
    else:
        k, n = case["in"], case["out"]
        leaves["x"] = rand(rows, k).to(dt)
        leaves["weight"] = (rand(2 * n, k) / math.sqrt(k)).to(dt)
        dy["y"] = rand(rows, n).to(dt)
    leaves = {n: t for n, t in leaves.items() if t is not None}
    if case["train"]:
        for t in leaves.values():
            t.requires_grad_(True)
    return {"case": case, "leaves": leaves, "dy": dy if case["train"] else {}, "seed": (seed * 0x9E3779B97F4A7C15) % (1 << 62)}


# ───────────────────────────── the operators ─────────────────────────────

def run(state):
    return _call(state) if own else _plain(state)


def _call(s):
    """The calls that a training or serving program makes."""
    from swiftrwkv_amd import train

    c, t = s["case"], s["leaves"]
    if c["kind"] == "dropout":
        out = {"y": train.dropout(t["x"], c["p"], s["seed"], offset=OFFSET, residual=t.get("residual"))}
    elif c["kind"] == "join":
        xs, h = train.block_join(t["x"], t["o"], t["weight"], t.get("bias"), post_weight=t.get("post_weight"),
                                 post_bias=t.get("post_bias"), gate=t.get("gate"), scale=t.get("scale"), p=c["p"],
                                 seed=s["seed"], offset=OFFSET, eps=EPS)
        out = {"x": xs, "h": h}
    elif c["kind"] == "tail":
        out = {"y": train.wkv_tail(t["o"], t["r"], t["k"], t["v"], t["r_k"], t["gate"], t["weight"], t["bias"],
                                   eps=HEAD_EPS)}
    else:
        out = {"y": train.gated_linear(t["x"], t["weight"], c["act"])}
    if not c["train"]:
        return out
    grads = torch.autograd.grad(tuple(out.values()), tuple(t.values()), tuple(s["dy"].values()))
    return {**{n: v.detach() for n, v in out.items()}, **{"d" + n: g for n, g in zip(t, grads)}}


def _numbers(rows, width, seed):
    """The 16-bit random numbers of [rows, width], as int32."""
    low = 0xFFFFFFFF
    chunks = -(-width // 8)
    c0 = torch.arange(chunks, device=DEVICE).expand(rows, chunks)
    c1 = torch.arange(rows, device=DEVICE)[:, None].expand(rows, chunks)
    c2, c3 = torch.full_like(c0, OFFSET & low), torch.full_like(c0, OFFSET >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57   # 64 bits, of which the sign bit is one
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    halves = [h for w in (c0, c1, c2, c3) for h in ((w & 0xFFFF).int(), (w >> 16).int())]
    return torch.stack(halves, -1).reshape(rows, 8 * chunks)[:, :width]


def _kept(c, seed, shape):
    """The factor of every value: zero, or what the kept ones are multiplied by."""
    t = round(65536 * c["p"])
    if t == 0:
        return None
    return torch.where(_numbers(*shape, seed) >= t, 65536 / (65536 - t), 0.0)


def _norm(x, eps):
    dev = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(dev.square().mean(-1, keepdim=True) + eps)
    return dev * r, r


def _norm_back(g, xh, r):
    return (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * r


def _gate_act(name, z):
    """The gate's activation and its slope."""
    if name == "relu2":
        return torch.relu(z).square(), 2 * torch.relu(z)
    if name == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        u, du = a * (z + 0.044715 * z * z * z), a * (1 + 3 * 0.044715 * z * z)
    else:
        u, du = z, 1.0
    s, rest = 1 / (1 + torch.exp(-u)), 1 / (1 + torch.exp(u))
    if name == "sigmoid":
        return s, s * rest
    return z * s, s + z * s * rest * du


@torch.no_grad()
def _plain(s):
    """The same from elementary operations in 32 bits, rounded once at the end."""
    c, leaves = s["case"], s["leaves"]
    t = {n: v.float() for n, v in leaves.items()}
    d = {n: v.float() for n, v in s["dy"].items()}
    out, g = {}, {}   # results; gradients
    if c["kind"] == "dropout":
        kept = _kept(c, s["seed"], t["x"].shape)
        y = t["x"] if kept is None else torch.where(kept > 0, t["x"] * kept, 0.0)
        res = leaves.get("residual")
        out["y"] = (y if res is None else y + t["residual"]).to((leaves["x"] if res is None else res).dtype)
        if c["train"]:
            g["x"] = d["y"] if kept is None else torch.where(kept > 0, d["y"] * kept, 0.0)
            if res is not None:
                g["residual"] = d["y"]
    elif c["kind"] == "join":
        kept = _kept(c, s["seed"], t["x"].shape) if c["p"] else None
        n = t["o"]
        if c["post"]:
            oh, r1 = _norm(t["o"], EPS)
            n = oh * t["post_weight"] + t.get("post_bias", 0.0)
        u = n * t["gate"] if c["gate"] else n
        m = u if kept is None else torch.where(kept > 0, u * kept, 0.0)
        xs = t["x"] + (m * t["scale"] if c["scale"] else m)
        xh, r2 = _norm(xs, EPS)
        out["x"] = xs.to(leaves["x"].dtype)
        out["h"] = (xh * t["weight"] + t.get("bias", 0.0)).to(leaves["o"].dtype)
        if c["train"]:
            dx = d["x"] + _norm_back(d["h"] * t["weight"], xh, r2)
            du = dx * t["scale"] if c["scale"] else dx
            if kept is not None:
                du = torch.where(kept > 0, du * kept, 0.0)
            dn = du * t["gate"] if c["gate"] else du
            g = {"x": dx, "o": _norm_back(dn * t["post_weight"], oh, r1) if c["post"] else dn,
                 "weight": (d["h"] * xh).sum(0), "bias": d["h"].sum(0), "gate": du * n, "scale": (dx * m).sum(0)}
            if c["post"]:
                g["post_weight"], g["post_bias"] = (dn * oh).sum(0), dn.sum(0)
    elif c["kind"] == "tail":
        rows, heads = c["rows"], c["heads"]
        by_head = lambda v: v.reshape(-1, heads, HEAD)  # noqa: E731
        o, r, k, v, gate = (by_head(t[n]) for n in ("o", "r", "k", "v", "gate"))
        rk, w, b = (by_head(t[n]) for n in ("r_k", "weight", "bias"))
        oh, inv = _norm(o, HEAD_EPS)
        dot = (r * k * rk).sum(-1, keepdim=True)
        q = oh * w + b + dot * v
        out["y"] = (q * gate).reshape(rows, -1).to(leaves["r"].dtype)
        if c["train"]:
            dy = by_head(d["y"])
            dq = dy * gate
            ddot = (dq * v).sum(-1, keepdim=True)
            g = {"o": _norm_back(dq * w, oh, inv), "r": ddot * k * rk, "k": ddot * r * rk, "v": dq * dot,
                 "r_k": (ddot * r * k).sum(0), "gate": dy * q, "weight": (dq * oh).sum(0), "bias": dq.sum(0)}
            g = {n: x.reshape(leaves[n].shape) for n, x in g.items()}
    else:
        wg, wu = t["weight"].chunk(2)
        zg, zu = t["x"] @ wg.t(), t["x"] @ wu.t()
        act, slope = _gate_act(c["act"], zg)
        out["y"] = (act * zu).to(leaves["x"].dtype)
        if c["train"]:
            dg, du = d["y"] * zu * slope, d["y"] * act
            g["x"] = dg @ wg + du @ wu
            g["weight"] = torch.cat([dg.t() @ t["x"], du.t() @ t["x"]])
    out.update(("d" + n, g[n].to(v.dtype)) for n, v in leaves.items() if c["train"])
    return out


# ───────────────────────────── 64 bits ─────────────────────────────

def _drops(c, seed, shape):
    """Which values are kept, by the generator's definition on the host."""
    rows, width = shape
    chunks, mask, half = -(-width // 8), np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = [np.tile(np.arange(chunks, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), chunks),
           np.uint64(OFFSET & 0xFFFFFFFF), np.uint64(OFFSET >> 32)]
    for i in range(10):
        keys = [np.uint64((k + i * w) & 0xFFFFFFFF) for k, w in ((seed, 0x9E3779B9), (seed >> 32, 0xBB67AE85))]
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> half) ^ ctr[1] ^ keys[0], b & mask, (a >> half) ^ ctr[3] ^ keys[1], a & mask]
    numbers = np.stack(ctr, 1).astype("<u4").view("<u2").reshape(rows, 8 * chunks)[:, :width]
    return torch.from_numpy(numbers >= round(65536 * c["p"])).to(DEVICE)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    t = {n: v.detach().double().requires_grad_(c["train"]) for n, v in s["leaves"].items()}

    def drop(v):
        if not c["p"]:
            return v
        return v.masked_fill(~_drops(c, s["seed"], v.shape), 0) * (65536 / (65536 - round(65536 * c["p"])))

    def norm(v, eps):
        var, mean = torch.var_mean(v, -1, correction=0, keepdim=True)
        return (v - mean) * torch.rsqrt(var + eps)

    if c["kind"] == "dropout":
        y = drop(t["x"])
        out = {"y": y + t["residual"] if "residual" in t else y}
    elif c["kind"] == "join":
        u = t["o"]
        if c["post"]:
            u = norm(u, EPS) * t["post_weight"]
            u = u + t["post_bias"] if "post_bias" in t else u
        for n in ("gate", "scale"):
            u = u * t[n] if n in t else u
        xs = t["x"] + drop(u)
        h = norm(xs, EPS) * t["weight"]
        out = {"x": xs, "h": h + t["bias"] if "bias" in t else h}
    elif c["kind"] == "tail":
        shape = (c["rows"], c["heads"], HEAD)
        bonus = torch.einsum("nhd,nhd,hd->nh", t["r"].view(shape), t["k"].view(shape), t["r_k"].view(shape[1:]))
        q = norm(t["o"].view(shape), HEAD_EPS).flatten(1) * t["weight"] + t["bias"]
        out = {"y": (q + (bonus[..., None] * t["v"].view(shape)).flatten(1)) * t["gate"]}
    else:
        z = t["x"] @ t["weight"].t()
        gate, up = z[:, :c["out"]], z[:, c["out"]:]
        act = {"relu2": lambda v: v.clamp(min=0) ** 2, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu,
               "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[c["act"]]
        out = {"y": act(gate) * up}
    if not c["train"]:
        return out
    grads = torch.autograd.grad(tuple(out.values()), tuple(t.values()), tuple(v.double() for v in s["dy"].values()))
    return {**{n: v.detach() for n, v in out.items()}, **{"d" + n: v for n, v in zip(t, grads)}}


# ───────────────────────────── what a pass cannot do without ─────────────────────────────

def work(case):
    size = lambda t: DTYPE[t].itemsize  # noqa: E731
    m, e, train, kind = case["rows"], size(case["dtype"]), case["train"], case["kind"]
    if kind == "gated":
        k, n = case["in"], case["out"]
        moved = e * (m * k + 2 * n * k + m * n)   # x, W and y; then dy, dx and dW
        return {"bytes": moved * (2 if train else 1), "flops": 4 * m * n * k * (3 if train else 1)}
    if kind == "dropout":
        y = size(case["residual"]) if case["residual"] else e
        forward = e + y * (2 if case["residual"] else 1)   # x and the residual in, y out; then dy in and their gradients
        return {"bytes": m * case["width"] * forward * (2 if train else 1), "flops": m * case["width"] * (4 if train else 2)}
    w = size(case["weights"])
    if kind == "tail":
        d, o = case["heads"] * HEAD, size(case["state"])
        forward = m * d * (o + 5 * e) + 3 * d * w   # o, r, k, v, gate in, y out; then dy in and theirs
        return {"bytes": forward * (2 if train else 1), "flops": m * d * (50 if train else 14)}
    d, x = case["width"], size(case["stream"])
    vectors = w * d * sum((1, case["bias"], case["post"], case["post"] and case["bias"], case["scale"]))
    forward = m * d * (2 * x + e * (3 if case["gate"] else 2)) + vectors   # x, o, gate in, x', h out; then theirs
    return {"bytes": forward * (2 if train else 1), "flops": m * d * (44 if train else 16)}
