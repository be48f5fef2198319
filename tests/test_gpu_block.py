"""Dropout, block joins and the recurrence's tail on the GPU against plain
64-bit forms, whose running error analysis (bounds.py) gives every value's
tolerance.  Masks have to be the generator's, exactly."""
import ctypes
import sys

import pytest
import torch

from swiftrwkv_amd import _lib, kernel, train

from .bounds import E, U, norm, norm_back, worst
from .philox import kept, numbers

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
SEED, OFF = 0x9E3779B97F4A7C15, (5 << 32) + 77


def case(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def check(what, got, want):
    w = worst(got, want)
    print(f"  {what}: worst error {w:.3f} of its bound", flush=True)
    assert w <= 1.0, (what, w)


def mask_of(rows, width, p, seed=SEED, offset=OFF):
    return torch.from_numpy(kept(rows, width, p, seed, offset)).to(DEV)


def scale_of(p):
    t = round(65536 * p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


# ───────────────────────────── dropout ─────────────────────────────

def run_dropout(x, p, res=None, dy=None, seed=SEED, offset=OFF):
    N, D = x.numel() // x.shape[-1], x.shape[-1]
    m = mask_of(N, D, p, seed, offset).reshape(x.shape)
    leaves = [v.detach().requires_grad_(True) for v in (x, res) if v is not None]
    y = train.dropout(leaves[0], p, seed, offset=offset, residual=leaves[1] if res is not None else None)
    v = (E(x) * E(scale_of(p), U)).where(m)
    check("y", y.detach(), v + E(res) if res is not None else v)
    dy = torch.ones_like(y) if dy is None else dy
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(a.dtype == b.dtype and a.shape == b.shape for a, b in zip(grads, leaves))
    check("dx", grads[0], (E(dy) * E(scale_of(p), U)).where(m))
    assert not grads[0][~m].any()
    if res is None:
        assert not y[~m].any()
    else:
        assert torch.equal(grads[1], dy) and torch.equal(y.detach()[~m], res[~m])
    return y


@pytest.mark.parametrize("N,D", [(1, 1), (1, 7), (3, 8), (5, 9), (700, 1), (300, 8), (2, 8191), (3, 8192), (2, 8200), (1, 70001),
                                 (129, 1000), (1, 1024), (4097, 33), (65, 4096)])
def test_dropout_sizes(N, D):
    case(f"dropout {N} x {D}")
    run_dropout(randn(gen(N + D), N, D), 0.3)


@pytest.mark.parametrize("xdt,rdt", [(F32, None), (F32, F32), (BF, None), (BF, BF), (BF, F32), (HF, None), (HF, HF), (HF, F32)])
@pytest.mark.parametrize("N,D", [(3, 64), (33, 517)])
def test_dropout_types(N, D, xdt, rdt):
    case(f"dropout {N} x {D} {xdt}, residual {rdt}")
    g = gen(N)
    x, res = randn(g, N, D, dtype=xdt), randn(g, N, D, dtype=rdt) if rdt else None
    run_dropout(x, 0.1, res, randn(g, N, D, dtype=rdt or xdt))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 2.0 ** -16, 0.5, 1 - 2.0 ** -16, 1 - 2.0 ** -18, 1.0])
def test_dropout_probabilities(p):
    case(f"dropout p {p}")
    x = randn(gen(1), 257, 1031)
    y = run_dropout(x, p)
    if round(65536 * p) == 0:
        assert torch.equal(y, x)
    if round(65536 * p) == 65536:
        assert not y.any()


@pytest.mark.parametrize("seed,offset", [(0, 0), ((1 << 64) - 1, (1 << 64) - 1), (1 << 32, 0), (1, 1 << 32), (1 << 63, 1 << 63)])
def test_dropout_seeds(seed, offset):
    case(f"dropout seed {seed} offset {offset}")
    run_dropout(randn(gen(2), 40, 100), 0.5, seed=seed, offset=offset)
    if seed < 1 << 63:
        x = randn(gen(2), 40, 100)
        t = torch.tensor([seed], device=DEV)
        assert torch.equal(train.dropout(x, 0.5, t, offset=offset), train.dropout(x, 0.5, seed, offset=offset))


def test_dropout_views():
    """Any strides: the mask goes by the value's place, not by its address."""
    case("dropout of views")
    big = randn(gen(3), 12, 200, dtype=BF)
    for v in (big[:, 3:103], big[::2, :64], big.t(), big[:, 1::2], big[4], big.reshape(3, 4, 200), big.reshape(3, 4, 200).transpose(0, 1),
              big[:1, 7:8], big[:1].expand(6, 200), big[:, :1].expand(12, 50)):
        run_dropout(v, 0.4, residual_of(v))
    for empty in (big[:0], big.reshape(3, 4, 200)[:, :0]):
        e = empty.detach().requires_grad_(True)
        y = train.dropout(e, 0.4, 1)
        assert y.shape == empty.shape and torch.autograd.grad(y, e, torch.ones_like(y))[0].shape == empty.shape


def residual_of(v):
    return torch.stack([v, v], -1)[..., 0].float()   # strided by two: copied first


def test_dropped_values_leave_nothing():
    case("dropout: infinities and NaN among the dropped and the kept")
    x = randn(gen(4), 64, 64)
    m = mask_of(64, 64, 0.5)
    bad = torch.where(m, x, torch.tensor([float("nan"), float("inf")], device=DEV).repeat(64, 32))
    assert torch.isfinite(train.dropout(bad, 0.5, SEED, offset=OFF)).all()
    y = train.dropout(torch.where(m, float("nan"), x), 0.5, SEED, offset=OFF)
    assert torch.equal(torch.isnan(y), m)


def test_dropout_writes_its_rows_alone():
    """What lies behind and between the rows stays: through the C entry, into the middle of a buffer."""
    case("dropout into the middle of a buffer")
    for D in (1, 9, 64, 1000):
        x = randn(gen(D), 37, D, dtype=BF)
        buf = torch.full((37 * D + 64,), 7.0, device=DEV, dtype=BF)
        d = _lib.Drop(SEED, None, OFF, 32768)
        _lib.check(_lib.lib().rwkv_dropout(x.data_ptr(), _lib.BF16, D, None, 0, buf[32:].data_ptr(), _lib.BF16, ctypes.byref(d),
                                           37, D, torch.cuda.current_stream().cuda_stream))
        assert (buf[:32] == 7).all() and (buf[32 + 37 * D:] == 7).all()
        assert torch.equal(buf[32:32 + 37 * D].reshape(37, D), train.dropout(x, 0.5, SEED, offset=OFF))


def test_dropout_of_more_than_2_32_bytes():
    """Rows whose chunks and addresses pass 2^31 and 2^32."""
    case("dropout 300001 x 16384 bf16")
    N, D = 300001, 16384   # 4.9e9 values
    x = torch.ones(1, D, device=DEV, dtype=BF).expand(N, D).contiguous()
    y = train.dropout(x, 0.5, SEED, offset=OFF)
    for row in (0, 131071, 131073, 262145, N - 1):
        m = torch.from_numpy(numbers(1, D, SEED, OFF, row) >= 32768).to(DEV)
        assert torch.equal(y[row:row + 1] != 0, m), row
    del x, y
    torch.cuda.empty_cache()


def test_dropout_of_rows_far_apart():
    """Rows 2^32 values apart and more: copied first."""
    case("dropout of rows 2^32 values apart")
    for step in ((1 << 32) - 8, (1 << 32) + 8):
        buf = torch.empty(step + 72, device=DEV, dtype=BF)
        v = buf.as_strided((2, 64), (step, 1), 8)
        v.copy_(randn(gen(1), 2, 64))
        run_dropout(v, 0.4, v.float())
        del buf, v
    torch.cuda.empty_cache()


def test_captured_backward_over_an_eager_graph_s_leaves():
    """The leaves' gradient nodes belong to the eager graph's stream: a captured
    backward pass that reaches them is refused, with a message, and the next
    capture, with leaves of its own, runs."""
    case("a captured backward pass while an eager graph of the same leaves lives")
    x, w = randn(gen(1), 6, 128, dtype=BF).requires_grad_(True), randn(gen(2), 16, 128, dtype=BF)
    one = torch.ones(128, device=DEV)
    calls = {"dropout": lambda a: train.dropout(a, 0.1, 1), "block_join": lambda a: train.block_join(a, a, one)[1],
             "wkv_tail": lambda a: train.wkv_tail(a, a, a, a, one, a, one, one), "gated_linear": lambda a: train.gated_linear(a, w)}
    for name, f in calls.items():
        eager = f(x)
        dy = torch.ones_like(eager)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                y = f(x)
                with pytest.raises(RuntimeError, match=f"{name}: its captured backward pass reaches a leaf"):
                    torch.autograd.grad(y, x, dy)
            own = x.detach().requires_grad_(True)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                dx, = torch.autograd.grad(f(own), own, dy)
        torch.cuda.current_stream().wait_stream(side)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            want, = torch.autograd.grad(f(x), x, dy)
            assert torch.equal(dx, want), name
        torch.autograd.grad(eager, x, dy)


def test_seed_tensor_in_a_graph():
    """Forward and backward captured once; each replay takes the seed that the tensor holds then."""
    case("dropout and block_join captured with their gradients, another seed each replay")
    x, o, w = randn(gen(5), 48, 320, dtype=BF), randn(gen(6), 48, 320, dtype=BF), torch.ones(320, device=DEV)
    dy = randn(gen(7), 48, 320, dtype=BF)
    seed = torch.zeros(1, dtype=torch.int64, device=DEV)

    def go(sd):
        a, b = x.detach().requires_grad_(True), o.detach().requires_grad_(True)
        y = train.dropout(a, 0.25, sd, offset=1)
        xs, h = train.block_join(y, b, w, p=0.25, seed=sd, offset=2)
        return (xs.detach(), h.detach(), *torch.autograd.grad((xs, h), (a, b), (dy, dy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(seed)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = go(seed)
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        seed.fill_(1000 + k)
        x.copy_(randn(gen(60 + k), 48, 320))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, go(1000 + k))), k


def test_seed_changed_before_the_backward_pass():
    case("dropout: a seed tensor changed in between is refused")
    x, seed = randn(gen(8), 4, 64).requires_grad_(True), torch.tensor(3, device=DEV)
    y = train.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x, torch.ones_like(y))


# ───────────────────────────── block join ─────────────────────────────

def ones(g, D, dt):
    return (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dt)


def join_inputs(N, D, sdt, dt, wdt, parts, seed=0):
    g = gen(seed + 131 * N + D)
    v = {"x": (2 * randn(g, N, D) + 0.5).to(sdt), "o": randn(g, N, D, dtype=dt), "weight": ones(g, D, wdt)}
    if "b" in parts:
        v["bias"] = randn(g, D, dtype=wdt, scale=0.3)
    if "p" in parts:
        v["post_weight"] = ones(g, D, wdt)
        if "b" in parts:
            v["post_bias"] = randn(g, D, dtype=wdt, scale=0.3)
    if "g" in parts:
        v["gate"] = randn(g, N, D, dtype=dt)
    if "s" in parts:
        v["scale"] = randn(g, D, dtype=wdt)
    return v, randn(g, N, D, dtype=sdt), randn(g, N, D, dtype=dt)


def join_ref(v, p, dx, dh, N, D, eps=1e-5, post_eps=1e-5):
    """x', h and the gradients with their bounds."""
    t = {n: E(a) for n, a in v.items()}
    row = 64 + 16   # a thread's 8 values, a wave's tree, 16 waves, a few more
    cols = max(1, N // 128) + 48   # a block's rows, the join of the blocks' partial rows
    m = mask_of(N, D, p) if round(65536 * p) else torch.ones(N, D, dtype=torch.bool, device=DEV)
    ms = E(scale_of(p), U)
    n = t["o"]
    if "post_weight" in t:
        oh, r1 = norm(t["o"], post_eps, row)
        n = oh * t["post_weight"]
        n = n + t["post_bias"] if "post_bias" in t else n
    u = n * t["gate"] if "gate" in t else n
    d = (u * ms).where(m)
    xs = t["x"] + (d * t["scale"] if "scale" in t else d)
    xh, r2 = norm(xs, eps, row)
    h = xh * t["weight"]
    h = h + t["bias"] if "bias" in t else h
    xk = xh
    G = E(dx) if dx is not None else E(torch.zeros(N, D, device=DEV))
    out = {}
    zero = E(torch.zeros(D, device=DEV))
    if dh is not None:
        G = G + norm_back(E(dh) * t["weight"], xk, r2, row)
        out["weight"], out["bias"] = (E(dh) * xk).sum(0, cols, False), E(dh).sum(0, cols, False)
    else:
        out["weight"] = out["bias"] = zero
    out["x"] = G
    gm = (G * ms).where(m)
    out["scale"] = (gm * u).sum(0, cols, False)
    du = gm * t["scale"] if "scale" in t else gm
    out["gate"] = du * n
    dn = du * t["gate"] if "gate" in t else du
    if "post_weight" in t:
        out["post_weight"], out["post_bias"] = (dn * oh).sum(0, cols, False), dn.sum(0, cols, False)
        out["o"] = norm_back(dn * t["post_weight"], oh, r1, row)
    else:
        out["o"] = dn
    return xs, h, {n: out[n] for n in v}


def call_join(v, p, **kw):
    return train.block_join(v["x"], v["o"], v["weight"], v.get("bias"), post_weight=v.get("post_weight"),
                            post_bias=v.get("post_bias"), gate=v.get("gate"), scale=v.get("scale"), p=p, seed=SEED, offset=OFF, **kw)


def run_join(N, D, sdt=F32, dt=F32, wdt=F32, parts="bpgs", p=0.2, seed=0):
    v, dx, dh = join_inputs(N, D, sdt, dt, wdt, parts, seed)
    leaves = {n: a.detach().clone().requires_grad_(True) for n, a in v.items()}
    xs, h = call_join(leaves, p)
    assert xs.dtype == sdt and h.dtype == dt
    grads = torch.autograd.grad((xs, h), list(leaves.values()), (dx, dh))
    with torch.no_grad():
        xs2, h2 = call_join(v, p)
        assert torch.equal(xs2, xs) and torch.equal(h2, h)
    rx, rh, rg = join_ref(v, p, dx, dh, N, D)
    check("x'", xs.detach(), rx)
    check("h", h.detach(), rh)
    for (n, w), got in zip(rg.items(), grads):
        assert got.dtype == v[n].dtype and got.shape == v[n].shape
        check("d" + n, got, w)
    return xs, h, grads


TYPES = [(F32, F32, F32), (F32, BF, F32), (F32, BF, BF), (BF, BF, F32), (BF, BF, BF), (F32, HF, F32), (F32, HF, HF), (HF, HF, F32),
         (HF, HF, HF)]


@pytest.mark.parametrize("sdt,dt,wdt", TYPES)
@pytest.mark.parametrize("N,D", [(1, 1024), (67, 1023), (9, 2056)])
def test_join_types(N, D, sdt, dt, wdt):
    case(f"join {N} x {D} stream {sdt}, {dt}, vectors {wdt}")
    run_join(N, D, sdt, dt, wdt)


@pytest.mark.parametrize("N,D", [(1, 1), (3, 2), (2, 31), (9, 512), (7, 513), (5, 1024), (6, 1025), (4, 2048), (3, 2049), (4, 4096),
                                 (3, 4097), (2, 8191), (2, 8192), (4097, 64), (5000, 33), (2200, 600)])
def test_join_widths(N, D):
    case(f"join width {N} x {D}")
    run_join(N, D, parts="bpgs" if D > 2 else "gs")   # a norm of one or two values says nothing


@pytest.mark.parametrize("sdt,dt", [(BF, BF), (HF, HF), (F32, HF)])
@pytest.mark.parametrize("N,D", [(4, 5), (2, 31), (70, 64), (9, 512), (7, 513), (6, 1025), (4, 2048), (3, 2049), (4, 4096), (3, 4097), (2, 8191),
                                 (2, 8192), (300, 256), (5000, 33), (1030, 1024)])
def test_join_widths_of_16_bit_types(N, D, sdt, dt):
    case(f"join width {N} x {D} stream {sdt}, {dt}")
    run_join(N, D, sdt, dt, dt)


@pytest.mark.parametrize("parts", ["", "b", "p", "pb", "g", "s", "pg", "ps", "gs", "pgs"])
@pytest.mark.parametrize("p", [0.0, 0.6])
def test_join_parts(parts, p):
    case(f"join with parts '{parts}', p {p}")
    run_join(37, 777, F32, BF, F32, parts, p)


@pytest.mark.parametrize("N,D,sdt,dt", [(3000, 2048, F32, BF), (700, 5000, BF, BF), (6001, 300, HF, HF)])
def test_join_many_rows_twice_the_same_bits(N, D, sdt, dt):
    case(f"join {N} x {D}, twice")
    a, b = run_join(N, D, sdt, dt), run_join(N, D, sdt, dt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(p, q) for p, q in zip(a[2], b[2]))


@pytest.mark.parametrize("which", ["x", "h"])
def test_join_one_result_used(which):
    case(f"join: a gradient of {which} alone")
    N, D = 40, 600
    v, dx, dh = join_inputs(N, D, F32, BF, F32, "bpgs")
    leaves = {n: a.detach().clone().requires_grad_(True) for n, a in v.items()}
    xs, h = call_join(leaves, 0.2)
    got = torch.autograd.grad(xs if which == "x" else h, list(leaves.values()), dx if which == "x" else dh)
    _, _, rg = join_ref(v, 0.2, dx if which == "x" else None, dh if which == "h" else None, N, D)
    for (n, w), g in zip(rg.items(), got):
        check("d" + n, g, w)


def test_join_each_gradient_alone():
    case("join: each input's gradient asked for alone, the same bits")
    v, dx, dh = join_inputs(50, 700, F32, BF, F32, "bpgs")
    leaves = {n: a.detach().clone().requires_grad_(True) for n, a in v.items()}
    xs, h = call_join(leaves, 0.2)
    both = torch.autograd.grad((xs, h), list(leaves.values()), (dx, dh), retain_graph=True)
    for (n, leaf), want in zip(leaves.items(), both):
        got, = torch.autograd.grad((xs, h), leaf, (dx, dh), retain_graph=True)
        assert torch.equal(got, want), n
        alone = {m: a.detach().requires_grad_(m == n) for m, a in v.items()}
        got, = torch.autograd.grad(call_join(alone, 0.2), alone[n], (dx, dh))
        assert torch.equal(got, want), n


def test_join_layouts():
    """Views, expanded and 3-D inputs: what contiguous copies give."""
    case("join of views")
    g = gen(9)
    big, wide = randn(g, 24, 400, dtype=BF), randn(g, 400, dtype=F32)
    w = wide[::2]
    for x, o in ((big[:, :200], big[:, 200:]), (big[:, 100:300], big.t()[:200].t()), (big[::2, 3:203], big[1::2, 1:201]),
                 (big.reshape(4, 6, 400)[..., :200], big.reshape(4, 6, 400)[..., 200:]),
                 (big.reshape(4, 6, 400).transpose(0, 1)[..., :200], big.reshape(4, 6, 400).transpose(0, 1)[..., 200:]),
                 (big[:1, :200].expand(7, 200), big[0, :200].expand(7, 200)), (big[3, :200], big[4, 200:])):
        v = {"x": x, "o": o, "weight": w, "gate": o.roll(1, -1), "scale": w.flip(0), "post_weight": w}
        a = {n: t.detach().requires_grad_(True) for n, t in v.items()}
        b = {n: t.detach().contiguous().clone().requires_grad_(True) for n, t in v.items()}
        ra, rb = call_join(a, 0.2), call_join(b, 0.2)
        assert all(torch.equal(p, q) for p, q in zip(ra, rb))
        dy = (randn(gen(1), *ra[0].shape, dtype=BF), randn(gen(2), 2, *ra[0].shape, dtype=BF)[1])
        ga = torch.autograd.grad(ra, list(a.values()), dy)
        gb = torch.autograd.grad(rb, list(b.values()), dy)
        assert all(torch.equal(p, q) for p, q in zip(ga, gb))
        ge = torch.autograd.grad(call_join(a, 0.2), a["x"], (dy[0][..., :1].expand_as(ra[0]), dy[1]))[0]
        gf = torch.autograd.grad(call_join(a, 0.2), a["x"], (dy[0][..., :1].expand_as(ra[0]).contiguous(), dy[1]))[0]
        assert torch.equal(ge, gf)


def test_join_empty_rows():
    case("join and tail of no rows")
    w = torch.ones(64, device=DEV, requires_grad=True)
    x, o = torch.zeros(0, 3, 64, device=DEV, requires_grad=True), torch.zeros(0, 3, 64, device=DEV, dtype=BF, requires_grad=True)
    xs, h = train.block_join(x, o, w, w, post_weight=w, scale=w, p=0.1)
    gx, go, gw = torch.autograd.grad((xs, h), (x, o, w), (torch.zeros_like(xs), torch.zeros_like(h)))
    assert xs.shape == h.shape == gx.shape == go.shape == (0, 3, 64) and not gw.any()
    y = train.wkv_tail(x, o, o, o, w, o, w, w)
    gw, gx = torch.autograd.grad(y, (w, x), torch.zeros_like(y))
    assert y.shape == (0, 3, 64) and not gw.any() and gx.shape == x.shape


def test_join_rows_of_one_value_and_bad_rows():
    case("join: constant rows, infinities, NaN stay in their rows")
    v, dx, dh = join_inputs(8, 96, F32, F32, F32, "bpgs")
    v["o"][1], v["x"][2] = 3.25, 0.0
    v["o"][2] = 0.0
    v["o"][4, 7], v["x"][5, 9], v["gate"][6, 3] = float("nan"), float("inf"), float("nan")
    leaves = {n: a.detach().requires_grad_(True) for n, a in v.items()}
    xs, h = call_join(leaves, 0.0)
    good = [0, 1, 2, 3, 7]
    assert torch.isfinite(xs[good]).all() and torch.isfinite(h[good]).all() and torch.isnan(h[[4, 5, 6]]).all()
    gx, go = torch.autograd.grad((xs, h), (leaves["x"], leaves["o"]), (dx, dh))
    assert torch.isfinite(gx[good]).all() and torch.isfinite(go[good]).all()


def test_join_changed_result_is_refused():
    case("join: x' changed in place before the backward pass")
    x, o, w = randn(gen(1), 4, 64).requires_grad_(True), randn(gen(2), 4, 64), torch.ones(64, device=DEV)
    xs, h = train.block_join(x, o, w)
    with torch.no_grad():
        xs.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(h, x, torch.ones_like(h))


def test_join_offset_rows_keep_their_precision():
    """Rows far from zero: the mean is taken out before the squares."""
    case("join: rows around 1000")
    N, D = 5, 1000
    v, dx, dh = join_inputs(N, D, F32, F32, F32, "p")
    v["x"] += 1000
    v["o"] -= 300
    xs, h = call_join(v, 0.0)
    rx, rh, _ = join_ref(v, 0.0, dx, dh, N, D)
    check("x'", xs, rx)
    check("h", h, rh)


def test_join_writes_its_rows_alone():
    case("join into the middle of buffers")
    L = _lib.lib()
    for D in (1, 9, 64, 1000, 3000, 5000):
        N = 5
        x, o, w = randn(gen(D), N, D), randn(gen(D + 1), N, D, dtype=BF), torch.ones(D, device=DEV)
        xs, h = torch.full((N * D + 64,), 7.0, device=DEV), torch.full((N * D + 64,), 7.0, device=DEV, dtype=BF)
        st = torch.full((N + 8, 4), 7.0, device=DEV)
        j = _lib.Join(x=x.data_ptr(), o=o.data_ptr(), ldx=D, ldo=D, x_dt=_lib.F32, dt=_lib.BF16, w_dt=_lib.F32,
                      weight=w.data_ptr(), eps=1e-5, N=N, D=D)
        s = torch.cuda.current_stream().cuda_stream
        _lib.check(L.rwkv_join_fwd(ctypes.byref(j), xs[32:].data_ptr(), h[32:].data_ptr(), st[4:].data_ptr(), s))
        for b in (xs, h):
            assert (b[:32] == 7).all() and (b[32 + N * D:] == 7).all()
        assert (st[:4] == 7).all() and (st[4 + N:] == 7).all()
        g = [torch.full((N * D + 64,), 7.0, device=DEV, dtype=d) for d in (F32, BF)] + [torch.full((D + 64,), 7.0, device=DEV)]
        ws = torch.empty(L.rwkv_join_bwd_workspace(N, D), dtype=torch.uint8, device=DEV)
        _lib.check(L.rwkv_join_bwd(ctypes.byref(j), xs[32:].data_ptr(), st[4:].data_ptr(), x.data_ptr(), o.data_ptr(),
                                   g[0][32:].data_ptr(), g[1][32:].data_ptr(), None, g[2][32:].data_ptr(), None, None, None, None,
                                   ws.data_ptr(), ws.numel(), s))
        for b, n in ((g[0], N * D), (g[1], N * D), (g[2], D)):
            assert (b[:32] == 7).all() and (b[32 + n:] == 7).all() and not (b[32:32 + n] == 7).any()


# ───────────────────────────── tail ─────────────────────────────

def run_tail(N, H, odt=F32, dt=F32, wdt=F32, seed=0, rk2=False):
    C = 64 * H
    g = gen(seed + 17 * N + H)
    v = {"o": randn(g, N, C, dtype=odt, scale=0.5), "r": randn(g, N, C, dtype=dt), "k": randn(g, N, C, dtype=dt),
         "v": randn(g, N, C, dtype=dt), "r_k": randn(g, C, dtype=wdt, scale=0.4), "gate": randn(g, N, C, dtype=dt),
         "weight": ones(g, C, wdt), "bias": randn(g, C, dtype=wdt, scale=0.3)}
    if rk2:
        v["r_k"] = v["r_k"].reshape(H, 64)
    dy = randn(g, N, C, dtype=dt)
    leaves = {n: a.detach().clone().requires_grad_(True) for n, a in v.items()}
    y = train.wkv_tail(**leaves)
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    with torch.no_grad():
        assert torch.equal(train.wkv_tail(**v), y)
    t = {n: E(a.reshape(-1, H, 64)) for n, a in v.items()}
    row, cols = 32, max(1, N // 16) + 64
    oh, inv = norm(t["o"], 64e-5, row)
    d = (t["r"] * t["k"] * t["r_k"]).sum(-1, row)
    q = oh * t["weight"] + t["bias"] + d * t["v"]
    check("y", y.detach(), (q * t["gate"]).view(N, C))
    Y = E(dy.reshape(-1, H, 64))
    dq = Y * t["gate"]
    e = (dq * t["v"]).sum(-1, row)
    want = {"o": norm_back(dq * t["weight"], oh, inv, row), "r": e * t["k"] * t["r_k"], "k": e * t["r"] * t["r_k"], "v": dq * d,
            "r_k": (e * t["r"] * t["k"]).sum(0, cols, False), "gate": Y * q, "weight": (dq * oh).sum(0, cols, False),
            "bias": dq.sum(0, cols, False)}
    for (n, a), got in zip(v.items(), grads):
        assert got.dtype == a.dtype and got.shape == a.shape
        check("d" + n, got, want[n].view(*a.shape))
    return y, grads


@pytest.mark.parametrize("odt,dt,wdt", TYPES)
@pytest.mark.parametrize("N,H", [(1, 12), (67, 5)])
def test_tail_types(N, H, odt, dt, wdt):
    case(f"tail {N} x {H} heads, o {odt}, {dt}, vectors {wdt}")
    run_tail(N, H, odt, dt, wdt)


@pytest.mark.parametrize("N,H", [(1, 1), (33, 1), (5, 2), (9, 3), (8, 4), (3, 7), (3, 8), (3, 9), (130, 16), (2, 32), (1, 64),
                                 (2, 65), (1, 1024), (20011, 1), (3000, 12)])
def test_tail_sizes(N, H):
    case(f"tail {N} x {H} heads")
    a = run_tail(N, H, rk2=True)
    b = run_tail(N, H, rk2=True)
    assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1], b[1]))


def test_tail_is_the_decode_step_s():
    case("tail against kernel.wkv_tail")
    g = gen(3)
    o, r, k, v, gate = (randn(g, 9, 256) for _ in range(5))
    rk, w, b = randn(g, 256), ones(g, 256, F32), randn(g, 256)
    want = kernel.wkv_tail(o, r, k, v, rk, w, b, gate, 4, 64, rows=9)
    got = train.wkv_tail(o, r, k, v, rk, gate, w, b)
    # both are within the bound of the 64-bit form, so within twice it of each other
    h = lambda a: E(a.reshape(-1, 4, 64))  # noqa: E731
    oh, _ = norm(h(o), 64e-5, 80)
    ref = ((oh * h(w) + h(b) + (h(r) * h(k) * h(rk)).sum(-1, 80) * h(v)) * h(gate)).view(9, 256)
    check("here", got, ref)
    check("decode", want, ref)


def test_tail_layouts_and_needs():
    case("tail of views; each gradient alone")
    g = gen(4)
    big = randn(g, 6, 5, 1000, dtype=HF)
    w = randn(g, 3, 128)
    args = dict(o=big[..., :128], r=big[..., 131:259], k=big[..., 300:428], v=big[..., 1::2][..., :128], r_k=w[0],
                gate=big.transpose(0, 1)[..., 500:628].transpose(0, 1), weight=w[1], bias=w[2])
    a = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    b = {n: t.detach().contiguous().clone().requires_grad_(True) for n, t in args.items()}
    ya, yb = train.wkv_tail(**a), train.wkv_tail(**b)
    dy = randn(g, 5, 6, 128, dtype=HF).transpose(0, 1)
    ga = torch.autograd.grad(ya, list(a.values()), dy, retain_graph=True)
    gb = torch.autograd.grad(yb, list(b.values()), dy.contiguous())
    assert torch.equal(ya, yb) and all(torch.equal(p, q) for p, q in zip(ga, gb))
    for (n, leaf), want in zip(a.items(), ga):
        one, = torch.autograd.grad(ya, leaf, dy, retain_graph=True)
        assert torch.equal(one, want), n


@pytest.mark.parametrize("N,H", [(1, 1), (5, 3), (37, 12), (3, 65)])
def test_tail_writes_its_rows_alone(N, H):
    case(f"tail {N} x {H} heads into the middle of buffers")
    L, s, C = _lib.lib(), torch.cuda.current_stream().cuda_stream, 64 * H
    o, r = randn(gen(1), N, C), randn(gen(2), N, C, dtype=BF)
    w = torch.ones(C, device=DEV)
    j = _lib.Tail(o=o.data_ptr(), r=r.data_ptr(), k=r.data_ptr(), v=r.data_ptr(), gate=r.data_ptr(), ldo=C, ldr=C, ldk=C, ldv=C, ldg=C,
                  o_dt=_lib.F32, dt=_lib.BF16, w_dt=_lib.F32, r_k=w.data_ptr(), weight=w.data_ptr(), bias=w.data_ptr(), eps=64e-5, N=N, H=H)
    put = lambda n, dt: torch.full((n + 64,), 7.0, device=DEV, dtype=dt)  # noqa: E731
    at = lambda t: t[32:].data_ptr()  # noqa: E731
    outs = [put(N * C, BF), put(N * C, F32), *(put(N * C, BF) for _ in range(4)), *(put(C, F32) for _ in range(3))]
    ws = torch.empty(L.rwkv_tail_bwd_workspace(N, H), dtype=torch.uint8, device=DEV)
    _lib.check(L.rwkv_tail_fwd(ctypes.byref(j), at(outs[0]), s))
    _lib.check(L.rwkv_tail_bwd(ctypes.byref(j), r.data_ptr(), C, *(at(t) for t in outs[1:]), ws.data_ptr(), ws.numel(), s))
    for t in outs:
        assert (t[:32] == 7).all() and (t[-32:] == 7).all() and not (t[32:-32] == 7).all()


# ───────────────────────────── many values ─────────────────────────────

def test_join_and_tail_past_2_31_values():
    """A row's results depend on no other row: the last rows of more than 2^31
    values are those of a call on them alone (bitwise; nothing dropped)."""
    N, D, n = 530000, 4096, 37   # 2.2e9 values
    case(f"join {N} x {D}")
    x = randn(gen(1), 1, D, dtype=BF).expand(N, D).contiguous()
    o, w = x.clone(), ones(gen(2), D, F32)
    x[-n:], o[-n:] = randn(gen(3), n, D), randn(gen(4), n, D)
    x[0] = 7.0
    def join(a, b):
        la, lb = a.requires_grad_(True), b.requires_grad_(True)
        xs, h = train.block_join(la, lb, w, post_weight=w, scale=w)
        return (xs.detach(), h.detach(), *torch.autograd.grad((xs, h), (la, lb), (b.detach(), a.detach())))
    big = join(x, o)
    small = join(x.detach()[-n:].clone(), o.detach()[-n:].clone())
    assert all(torch.equal(p[-n:], q) for p, q in zip(big, small))
    del big
    case(f"tail {N} x {D // 64} heads")
    def tail(a, b):
        la, lb = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = train.wkv_tail(la, lb, la, lb, w, la, w, w)
        return (y.detach(), *torch.autograd.grad(y, (la, lb), b.detach()))
    big = tail(x, o)
    small = tail(x[-n:].clone(), o[-n:].clone())
    assert all(torch.equal(p[-n:], q) for p, q in zip(big, small))
    del big, x, o
    torch.cuda.empty_cache()


# ───────────────────────────── graphs, streams, derivatives ─────────────────────────────

def test_tail_and_join_in_a_graph():
    case("tail and join with their gradients captured into one graph, replayed between eager work")
    g = gen(11)
    v = {n: randn(g, 96, 256, dtype=F32 if n == "o" else BF) for n in ("o", "r", "k", "v", "gate")}
    vec = {n: randn(g, 256) for n in ("r_k", "weight", "bias")}
    x, w, dy = randn(g, 96, 256), torch.ones(256, device=DEV), randn(g, 96, 256, dtype=BF)

    def go():
        lv = {n: t.detach().requires_grad_(True) for n, t in {**v, **vec}.items()}
        xs = x.detach().requires_grad_(True)
        y = train.wkv_tail(**lv)
        x1, h = train.block_join(xs, y, w, scale=vec["bias"])
        return (x1.detach(), h.detach(), *torch.autograd.grad((x1, h), [xs, *lv.values()], (x, dy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = go()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        v["o"].copy_(randn(gen(70 + k), 96, 256))
        vec["weight"].copy_(randn(gen(80 + k), 256))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, go())), k


def test_on_another_stream():
    case("the operators on a stream of their own")
    x, o, w = randn(gen(1), 300, 1024), randn(gen(2), 300, 1024, dtype=BF), torch.ones(1024, device=DEV)
    want = train.block_join(x, o, w, p=0.1, seed=5), train.dropout(x, 0.1, 5), train.wkv_tail(x, o, o, o, w, o, w, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = x.clone().requires_grad_(True)
        got = train.block_join(a, o, w, p=0.1, seed=5), train.dropout(a, 0.1, 5), train.wkv_tail(a, o, o, o, w, o, w, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1], want[0][1])
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    d1, = torch.autograd.grad(got[0][1].float().sum() + got[1].sum() + got[2].float().sum(), a)
    b = x.clone().requires_grad_(True)
    again = train.block_join(b, o, w, p=0.1, seed=5), train.dropout(b, 0.1, 5), train.wkv_tail(b, o, o, o, w, o, w, w)
    d2, = torch.autograd.grad(again[0][1].float().sum() + again[1].sum() + again[2].float().sum(), b)
    assert torch.equal(d1, d2)


def test_two_threads_on_two_streams():
    """Calls at the same time share nothing: each thread's results and gradients
    are those of the calls one after the other."""
    case("the operators from two threads, each on a stream of its own")
    import threading

    def inputs(k):
        g = gen(100 + k)
        D = (640, 1024)[k]
        return {n: randn(g, 200, D, dtype=F32 if n == "x" else BF) for n in ("x", "o", "gate", "dy")}, torch.ones(D, device=DEV)

    def go(v, w):
        t = {n: a.detach().requires_grad_(n != "dy") for n, a in v.items()}
        xs, h = train.block_join(t["x"], t["o"], w, post_weight=w, gate=t["gate"], scale=w, p=0.3, seed=11)
        y = train.wkv_tail(xs, h, t["o"], t["gate"], w, t["o"], w, w)
        z = train.dropout(y, 0.2, 12, residual=t["o"])
        return [z.detach(), *torch.autograd.grad(z, [t["x"], t["o"], t["gate"]], v["dy"])]

    data = [inputs(k) for k in range(2)]
    want = [go(*d) for d in data]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[k] = go(*data[k])
                    assert all(torch.equal(a, b) for a, b in zip(got[k], want[k])), k
            s.synchronize()
        except Exception as e:   # of the thread, told below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not failed and all(g is not None for g in got), failed


def test_second_and_forward_derivatives_are_refused():
    case("derivatives of derivatives, tangents of gradients")
    x, w = randn(gen(1), 4, 64).requires_grad_(True), torch.ones(64, device=DEV)
    calls = {"dropout": lambda: train.dropout(x, 0.1, 1), "block_join": lambda: train.block_join(x, x, w)[1],
             "wkv_tail": lambda: train.wkv_tail(x, x, x, x, w, x, w, w)}
    for name, f in calls.items():
        y = f()
        v = torch.ones_like(y).requires_grad_(True)
        dx, = torch.autograd.grad((v * y).sum(), x, create_graph=True)
        for to in (x, v):
            with pytest.raises(RuntimeError, match=f"{name}: gradients of its gradients"):
                torch.autograd.grad(dx.sum() + v.sum(), to, retain_graph=True)
        fa = torch.autograd.forward_ad
        y = f()
        with fa.dual_level():
            with pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
                torch.autograd.grad(y, x, fa.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_gradients_against_differences():
    """Central differences of the fp32 operators along one direction.  A sum of
    2^10 results, each off by up to 2^-18 of a magnitude around 4, over a step of
    2^-6: under 2^-18·4·2^5·2^7 = 2^-4 of error at worst, and a curvature term of
    the step's square; directional derivatives here are of the order of 100."""
    case("directional differences of join and tail")
    v, dx, dh = join_inputs(8, 128, F32, F32, F32, "bpgs")
    dirs = {n: randn(gen(i), *a.shape) for i, (n, a) in enumerate(v.items())}
    f = lambda s: sum((a.double() * b.double()).sum().item() for a, b in zip(  # noqa: E731
        call_join({n: a + s * dirs[n] for n, a in v.items()}, 0.2), (dx, dh)))
    leaves = {n: a.detach().requires_grad_(True) for n, a in v.items()}
    grads = torch.autograd.grad(call_join(leaves, 0.2), list(leaves.values()), (dx, dh))
    want = sum((g.double() * dirs[n].double()).sum().item() for n, g in zip(leaves, grads))
    h = 2.0 ** -7
    d1, d2 = (f(h) - f(-h)) / (2 * h), (f(h / 2) - f(-h / 2)) / h
    better = (4 * d2 - d1) / 3   # the step's square cancels
    print(f"  {want:.4f}, differences {d1:.4f} {d2:.4f}", flush=True)
    assert abs(better - want) <= 2.0 ** -4 + abs(d2 - d1) / 2 + 2.0 ** -10 * abs(want)


# ───────────────────────────── values that leave their range ─────────────────────────────

@pytest.mark.parametrize("parts", ["", "g", "s", "p", "bpgs"])
@pytest.mark.parametrize("sdt,dt", [(F32, F32), (F32, BF), (BF, BF)])
@pytest.mark.parametrize("N,D", [(6, 7), (9, 96), (5, 601), (3, 5000)])
def test_join_dropped_places_pass_no_gradient(N, D, sdt, dt, parts):
    """What the gradient of x' holds at dropped places, an infinity or a NaN too,
    reaches dx there and nothing else: the bits of a call with zeros there."""
    case(f"join {N} x {D} {sdt} {dt} '{parts}': bad gradients at dropped places")
    v, dx, dh = join_inputs(N, D, sdt, dt, F32, parts)
    m = mask_of(N, D, 0.4)
    assert not m.all()
    bad = torch.where(m, dx, torch.tensor([float("inf"), float("nan"), -float("inf")], device=DEV).repeat(D)[:D].to(sdt))
    leaves = {n: a.detach().clone().requires_grad_(True) for n, a in v.items()}
    xs, h = call_join(leaves, 0.4)
    want = torch.autograd.grad((xs, h), list(leaves.values()), (dx.masked_fill(~m, 0), dh), retain_graph=True)
    got = torch.autograd.grad((xs, h), list(leaves.values()), (bad, dh))
    for n, a, b in zip(leaves, got, want):
        if n == "x":
            assert not torch.isfinite(a[~m]).any() and torch.equal(a[m], b[m])
        else:
            assert torch.isfinite(b).all() and torch.equal(a, b), n


def test_join_dropped_places_of_a_bad_row():
    case("join: a NaN in dh and o, nothing of it at dropped places")
    for sdt in (F32, BF):
        v, dx, dh = join_inputs(4, 300, sdt, BF, F32, "gs")
        m = mask_of(4, 300, 0.4)
        dh[1, 5] = float("nan")
        v["gate"][2], v["o"][3] = v["gate"][2].masked_fill(~m[2], float("inf")), v["o"][3].masked_fill(~m[3], float("nan"))
        leaves = {n: a.detach().requires_grad_(True) for n, a in v.items()}
        xs, h = call_join(leaves, 0.4)
        assert torch.isfinite(xs).all() and torch.isfinite(h).all()
        g = dict(zip(leaves, torch.autograd.grad((xs, h), list(leaves.values()), (dx, dh))))
        assert torch.isnan(g["x"][1]).all() and torch.isfinite(g["x"][[0, 2, 3]]).all()
        for n in ("o", "gate"):
            assert not g[n][~m].any() and torch.isnan(g[n][1][m[1]]).all() and torch.isfinite(g[n][[0, 2, 3]]).all(), n


def test_rows_of_tiny_values():
    """eps = 0 and rows around 2^-66, whose variance is subnormal in fp32: what
    the layer norm makes of them.  The variance, 1024 squares around 2^-132 in
    steps of 2^-149 each off by up to half of one, is right to 2^-17 and its
    root's inverse to 2^-18; sums and products are far below that."""
    case("join and tail: rows around 2^-66 without eps")
    x = randn(gen(1), 5, 1024, scale=2.0 ** -66)
    w, b = ones(gen(2), 1024, F32), randn(gen(3), 1024)
    _, h = train.block_join(x, torch.zeros_like(x), w, b, eps=0.0)
    _, n = train.block_join(torch.zeros_like(x), x, w, b, post_weight=w, post_bias=b, post_eps=0.0)
    xs, _ = train.block_join(torch.zeros_like(x), x, w, b, post_weight=w, post_bias=b, post_eps=0.0)
    X, W, B = x.double(), w.double(), b.double()
    xh = (X - X.mean(-1, keepdim=True)) / X.var(-1, correction=0, keepdim=True).sqrt()
    ref = xh * W + B
    off = 2.0 ** -17 * (xh * W).abs() + 2.0 ** -22 * ref.abs()
    assert torch.isfinite(n).all()
    for t in (h, xs, train.layer_norm(x, w, b, 0.0)):
        assert ((t.double() - ref).abs() <= off).all()
    one, zero = torch.ones(1024, device=DEV), torch.zeros(1024, device=DEV)
    y = train.wkv_tail(x, zero.expand_as(x), zero.expand_as(x), zero.expand_as(x), zero, one.expand_as(x), w, b, eps=0.0)
    X = X.reshape(5, 16, 64)
    xh = ((X - X.mean(-1, keepdim=True)) / X.var(-1, correction=0, keepdim=True).sqrt()).reshape(5, 1024)
    # 64 squares of a head: right to 2^-15, were they all at the mean's size; a head's largest row of errors is half a step each
    assert ((y.double() - xh * W - B).abs() <= 2.0 ** -15 * (xh * W).abs() + 2.0 ** -22 * (xh * W + B).abs()).all()


@pytest.mark.parametrize("sdt,dt", [(F32, BF), (HF, HF)])
@pytest.mark.parametrize("N,D", [(5, 7), (700, 9), (1500, 1531), (2100, 1000), (1100, 2048), (600, 5001)])
def test_join_into_its_own_stream(N, D, sdt, dt):
    """Through the C entry, x' where x is: the same bits."""
    case(f"join {N} x {D} {sdt} {dt}, x' over x")
    L, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    of = {F32: _lib.F32, BF: _lib.BF16, HF: _lib.F16}
    x, o, w = randn(gen(1), N, D, dtype=sdt), randn(gen(2), N, D, dtype=dt), ones(gen(3), D, F32)
    buf, got = [], []
    for alias in (False, True):
        a = x.clone()
        xs, h, st = a if alias else torch.empty_like(x), torch.empty_like(o), torch.empty(N, 4, device=DEV)
        j = _lib.Join(x=a.data_ptr(), o=o.data_ptr(), ldx=D, ldo=D, x_dt=of[sdt], dt=of[dt], w_dt=_lib.F32, weight=w.data_ptr(),
                      post_weight=w.data_ptr(), scale=w.data_ptr(), eps=1e-5, post_eps=1e-5, drop=_lib.Drop(SEED, None, OFF, 6554), N=N, D=D)
        buf.append((a, j))
        _lib.check(L.rwkv_join_fwd(ctypes.byref(j), xs.data_ptr(), h.data_ptr(), st.data_ptr(), s))
        got.append((xs, h, st))
    assert all(torch.equal(p, q) for p, q in zip(*got)) and not torch.equal(got[0][0], x)
