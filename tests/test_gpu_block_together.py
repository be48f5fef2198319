"""The operators around a block run together, as a training step uses them."""
import sys

import pytest
import torch

from swiftrwkv_amd import kernel, train

from .philox import kept

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def case(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def norm(v, w, b, eps):
    m = v.mean(-1, keepdim=True)
    return (v - m) / torch.sqrt((v - m).square().mean(-1, keepdim=True) + eps) * w + b


def inputs(B, T, H, F, dt, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, scale=1.0, dtype=F32: (scale * torch.randn(s, generator=g, device=DEV)).to(dtype)  # noqa: E731
    D = 64 * H
    t = {"x": r(B, T, D)}
    for n in ("r", "k", "v", "gate"):
        t[n] = r(B, T, D, scale=0.5, dtype=dt)
    t["r_k"] = r(H, 64, scale=0.3)
    for n in ("ln", "next", "last"):
        t[n + "_w"], t[n + "_b"] = 1 + 0.1 * r(D), 0.1 * r(D)
    t["output"] = r(D, D, scale=D ** -0.5, dtype=dt)
    t["weight"] = r(2 * F, D, scale=D ** -0.5, dtype=dt)
    t["down"] = r(D, F, scale=F ** -0.5, dtype=dt)
    t["scale"] = 0.5 + 0.1 * r(D)
    t["w"] = torch.exp(-0.6 * torch.rand(B, T, H, 64, generator=g, device=DEV))
    return t, r(B, T, D), r(B, T, D, dtype=dt)


def step(t, B, T, H, p, seed):
    """Recurrence, tail, output projection, join; gated feed-forward, join."""
    heads = lambda v: v.reshape(B, T, H, 64).float()  # noqa: E731
    kk = torch.nn.functional.normalize(heads(t["k"]), dim=-1)
    o = kernel.wkv7_train(heads(t["r"]), t["w"], heads(t["k"]), heads(t["v"]), -kk, 0.5 * kk)
    x, h = train.mix_tail(t["x"], o.reshape(B, T, -1), t["r"], t["k"], t["v"], t["r_k"], t["gate"], t["ln_w"], t["ln_b"], t["output"],
                          t["next_w"], t["next_b"], p=p, seed=seed, offset=1)
    return train.gated_mix(x, h, t["weight"], t["down"], t["last_w"], t["last_b"], scale=t["scale"], p=p, seed=seed, offset=2)


def step64(t, B, T, H, p, seed):
    heads = lambda v: v.reshape(B, T, H, 64)  # noqa: E731
    r, w, k, v = heads(t["r"]), heads(t["w"]), heads(t["k"]), heads(t["v"])
    kk = torch.nn.functional.normalize(k, dim=-1)
    S = torch.zeros(B, H, 64, 64, dtype=torch.float64, device=DEV)
    outs = []
    for i in range(T):
        sa = (S * -kk[:, i, :, None, :]).sum(-1)
        S = S * w[:, i, :, None, :] + v[:, i, :, :, None] * k[:, i, :, None, :] + sa[..., None] * (0.5 * kk[:, i, :, None, :])
        outs.append((S * r[:, i, :, None, :]).sum(-1))
    o = torch.stack(outs, 1)
    bonus = (r * k * t["r_k"]).sum(-1, keepdim=True) * v
    m = o.mean(-1, keepdim=True)
    oh = (o - m) / torch.sqrt((o - m).square().mean(-1, keepdim=True) + 64e-5)
    y = (oh.flatten(2) * t["ln_w"] + t["ln_b"] + bonus.flatten(2)) * t["gate"]
    D, q = 64 * H, round(65536 * p)
    drop = lambda a, off: a * torch.from_numpy(kept(B * T, D, p, seed, off)).to(DEV).reshape(B, T, D) * 65536 / (65536 - q)  # noqa: E731
    x = t["x"] + drop(y @ t["output"].t(), 1)
    h = norm(x, t["next_w"], t["next_b"], 1e-5)
    zg, zu = (h @ t["weight"].t()).chunk(2, -1)
    x = x + t["scale"] * drop((zg * torch.sigmoid(zg) * zu) @ t["down"].t(), 2)
    return x, norm(x, t["last_w"], t["last_b"], 1e-5)


@pytest.mark.parametrize("B,T,H,F,dt", [(2, 32, 2, 320, BF), (1, 16, 3, 100, HF), (3, 48, 1, 96, HF)])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_block(B, T, H, F, dt, p):
    """Both halves against 64-bit autograd of their formulas: relative 2-norms,
    24 half steps of the 16-bit type for its at most twelve rounded values in a
    row, each met on the way there and back."""
    case(f"block {B} x {T} x {H} heads x {F} {dt} p {p}")
    t, dx, dh = inputs(B, T, H, F, dt, B + T + F)
    leaves = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    out = step(leaves, B, T, H, p, 99)
    grads = torch.autograd.grad(out, list(leaves.values()), (dx, dh))
    big = {n: v.detach().double().requires_grad_(True) for n, v in t.items()}
    ref = step64(big, B, T, H, p, 99)
    want = torch.autograd.grad(ref, list(big.values()), (dx.double(), dh.double()))
    tol = 24 * torch.finfo(dt).eps / 2
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    assert out[0].dtype == F32 and out[1].dtype == dt
    assert rel(out[0].detach(), ref[0].detach()) <= tol and rel(out[1].detach(), ref[1].detach()) <= tol
    for n, a, b in zip(leaves, grads, want):
        print(f"  d{n}: {rel(a, b):.2e}", flush=True)
        assert a.shape == b.shape and rel(a, b) <= tol, n


def test_steps_with_a_seed_each():
    """backward() into .grad, step after step, the seed in a tensor: each step's
    gradients are those of a call with that seed as a number; a graph captured
    with its own leaves replays the same."""
    case("training steps of a block, eager and captured")
    B, T, H, F, dt = 2, 16, 2, 128, BF
    t, dx, dh = inputs(B, T, H, F, dt, 7)
    leaves = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    seed = torch.zeros(1, dtype=torch.int64, device=DEV)

    def grads_of(sd):
        own = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        return torch.autograd.grad(step(own, B, T, H, 0.3, sd), list(own.values()), (dx, dh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads_of(seed)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = grads_of(seed)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        seed.fill_(40 + k)
        out = step(leaves, B, T, H, 0.3, seed)
        torch.autograd.backward(out, (dx, dh))
        want = grads_of(40 + k)
        assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves.values(), want)), k
        for leaf in leaves.values():
            leaf.grad = None
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(captured, want)), k


def test_a_token_at_a_time():
    """With no gradient, a row alone gives what it gives in a batch."""
    case("gated_mix and mix_tail, one token of a batch")
    B, T, H, F, dt = 1, 5, 4, 512, HF
    t, _, _ = inputs(B, T, H, F, dt, 3)
    with torch.no_grad():
        o = t["x"] * 0.3
        go = lambda i: train.mix_tail(t["x"][0, i], o[0, i], t["r"][0, i], t["k"][0, i], t["v"][0, i], t["r_k"], t["gate"][0, i],  # noqa: E731
                                      t["ln_w"], t["ln_b"], t["output"], t["next_w"])
        x, h = go(slice(None))
        for i in range(T):
            a, b = go(slice(i, i + 1))
            assert torch.equal(a[0], x[i]) and torch.equal(b[0], h[i])
        x2, h2 = train.gated_mix(x, h, t["weight"], t["down"], t["last_w"])
        for i in range(T):
            a, b = train.gated_mix(x[i], h[i], t["weight"], t["down"], t["last_w"])
            assert torch.equal(a, x2[i]) and torch.equal(b, h2[i])


def captured(f):
    """f() in a graph on a stream of its own: its results and the graph."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        out = f()
    torch.cuda.current_stream().wait_stream(side)
    return out, graph


def leaves_of(dt=BF, D=128):
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s, dtype=dt: (0.3 * torch.randn(s, generator=g, device=DEV)).to(dtype)  # noqa: E731
    return {"x": r(24, D), "m": r(D, D), "w2": r(64, D), "down": r(D, 32), "v": 1 + r(D, dtype=F32), "key": r(160, D), "value": r(D, 160)}


def test_captured_backward_refuses_every_held_leaf():
    """Each operator, and the halves of a block where the held leaf is next to a
    product in their middle: refused by the operator that meets it."""
    case("captured backward passes over held leaves")
    t = leaves_of()
    x, m, w2, down, v = (t[n] for n in ("x", "m", "w2", "down", "v"))
    on = lambda a: a.detach().requires_grad_(True)  # noqa: E731
    stream = x.float()
    calls = {
        "layer_norm x": ("layer_norm", x, lambda a: train.layer_norm(a, v, v)),
        "layer_norm bias": ("layer_norm", v, lambda a: train.layer_norm(x, v, a)),
        "linear x": ("linear", x, lambda a: train.linear(a, m, activation="tanh")),
        "linear weight": ("linear", m, lambda a: train.linear(x, a)),
        "linear residual": ("linear", x, lambda a: train.linear(x, m, residual=a)),
        "gated_mix down": ("linear", down, lambda a: train.gated_mix(stream, x, w2, a, v)[0]),
        "gated_mix weight": ("gated_linear", w2, lambda a: train.gated_mix(stream, x, a, down, v)[1]),
        "mix_tail output": ("linear", m, lambda a: train.mix_tail(stream, x, x, x, x, v, x, v, v, a, v)[0]),
        "mix_tail gate": ("wkv_tail", x, lambda a: train.mix_tail(stream, x, x, x, x, v, a, v, v, m, v)[1]),
        "channel_mix key": ("linear", t["key"], lambda a: train.channel_mix(stream.reshape(2, 12, 128), v, v, v, a, t["value"])[0]),
        "channel_mix norm": ("layer_norm", v, lambda a: train.channel_mix(stream.reshape(2, 12, 128), a, v, v, t["key"], t["value"])[0])}
    for name, (what, leaf, f) in calls.items():
        print(f"  {name}", flush=True)
        held = on(leaf)
        eager = f(held)
        dy = torch.ones_like(eager)

        def refused():
            y = f(held)
            with pytest.raises(RuntimeError, match=f"^{what}: its captured backward pass reaches a leaf"):
                torch.autograd.grad(y, held, dy)

        captured(refused)

        def go():
            own = on(leaf)
            return torch.autograd.grad(f(own), own, dy)[0]

        got, graph = captured(go)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, go()), name
        assert torch.equal(torch.autograd.grad(eager, held, dy)[0], got), name


def test_captured_backward_past_leaves_that_it_does_not_reach():
    """A leaf that another graph holds, and whose gradient is not asked for, is no reason to refuse."""
    case("captured backward passes beside held leaves")
    t = leaves_of()
    held = {n: a.detach().requires_grad_(True) for n, a in t.items()}
    x, m, w2, v = (held[n] for n in ("x", "m", "w2", "v"))
    calls = {"layer_norm": lambda a: train.layer_norm(a, v, v), "linear": lambda a: train.linear(a, m, activation="sigmoid", residual=x),
             "gated_linear": lambda a: train.gated_linear(a, w2), "dropout": lambda a: train.dropout(a, 0.3, 5, residual=x),
             "block_join": lambda a: train.block_join(x, a, v, v, post_weight=v, gate=x, scale=v)[1],
             "wkv_tail": lambda a: train.wkv_tail(x, a, x, x, v, x, v, v)}
    for name, f in calls.items():
        print(f"  {name}", flush=True)
        eager = f(t["x"])   # holds the nodes of the other leaves
        assert eager.requires_grad
        dy = torch.ones_like(eager)

        def go():
            own = t["x"].detach().requires_grad_(True)
            return torch.autograd.grad(f(own), own, dy)[0]

        got, graph = captured(go)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, go()), name
        del eager


@pytest.mark.parametrize("B,T,H,F,dt", [(2, 32, 2, 320, BF), (1, 16, 3, 100, HF)])
@pytest.mark.parametrize("act", train.GATES)
def test_every_part_of_both_halves(B, T, H, F, dt, act):
    """mix_tail and gated_mix with every argument they take, an eps of their own
    for each norm, large enough that one in another's place shows.  Relative
    2-norms: at most 24 values are rounded on the way there and back, each off by
    0.43 half steps in the quadratic mean (a third of the square, over a
    mantissa's octave); independent, √24·0.43 = 2.1 half steps together.  Twice
    that, as norms and activations pass some of it on enlarged: 4 half steps."""
    case(f"block, every part: {B} x {T} x {H} heads x {F} {dt} {act}")
    D, p, seed = 64 * H, 0.25, 123
    eps = {"head": 0.3, "next": 0.05, "last": 0.6}
    t, dx, dh = inputs(B, T, H, F, dt, 5)
    del t["w"]
    g = torch.Generator(device=DEV).manual_seed(6)
    r = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    t["o"] = 0.4 * r(B, T, D)
    t["post_w"], t["post_b"], t["scale1"] = 1 + 0.1 * r(D), 0.1 * r(D), 0.5 + 0.1 * r(D)
    t["gate2"] = torch.sigmoid(r(B, T, D)).to(dt)
    leaves = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    a = leaves
    x, h = train.mix_tail(a["x"], a["o"], a["r"], a["k"], a["v"], a["r_k"], a["gate"], a["ln_w"], a["ln_b"], a["output"], a["next_w"],
                          a["next_b"], scale=a["scale1"], p=p, seed=seed, offset=3, eps=eps["next"], head_eps=eps["head"])
    out = train.gated_mix(x, h, a["weight"], a["down"], a["last_w"], a["last_b"], activation=act, post_weight=a["post_w"],
                          post_bias=a["post_b"], gate=a["gate2"], scale=a["scale"], p=p, seed=seed, offset=4, eps=eps["last"])
    grads = torch.autograd.grad(out, list(leaves.values()), (dx, dh))

    b = {n: v.detach().double().requires_grad_(True) for n, v in t.items()}
    q = round(65536 * p)
    drop = lambda v, off: v * torch.from_numpy(kept(B * T, D, p, seed, off)).to(DEV).reshape(B, T, D) * 65536 / (65536 - q)  # noqa: E731
    heads = lambda v: v.reshape(B, T, H, 64)  # noqa: E731
    y = norm(heads(b["o"]), 1.0, 0.0, eps["head"]).flatten(2) * b["ln_w"] + b["ln_b"]
    y = (y + ((heads(b["r"]) * heads(b["k"]) * b["r_k"]).sum(-1, keepdim=True) * heads(b["v"])).flatten(2)) * b["gate"]
    x = b["x"] + b["scale1"] * drop(y @ b["output"].t(), 3)
    zg, zu = (norm(x, b["next_w"], b["next_b"], eps["next"]) @ b["weight"].t()).chunk(2, -1)
    f = {"relu2": lambda v: v.clamp(min=0) ** 2, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu,
         "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[act]
    n = norm((f(zg) * zu) @ b["down"].t(), b["post_w"], b["post_b"], eps["last"])
    x = x + b["scale"] * drop(b["gate2"] * n, 4)
    ref = x, norm(x, b["last_w"], b["last_b"], eps["last"])
    want = torch.autograd.grad(ref, list(b.values()), (dx.double(), dh.double()))
    tol = 4 * torch.finfo(dt).eps / 2
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    for n, got, w in (("x", out[0].detach(), ref[0].detach()), ("h", out[1].detach(), ref[1].detach()),
                      *(("d" + n, got, w) for n, got, w in zip(leaves, grads, want))):
        print(f"  {n}: {rel(got, w):.2e} of {tol:.2e}", flush=True)
        assert got.shape == w.shape and rel(got, w) <= tol, n
