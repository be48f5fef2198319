"""Training-side operators on the GPU where layout, value or use is out of the
ordinary.  Tolerances: half a step, finfo.eps / 2, per rounding to 16 bits;
2^-24 per fp32 operation; what a test adds to these it derives."""
import sys

import pytest
import torch

from swiftrwkv_amd import _lib, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def case(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


# ───────────────────────────── rows far apart ─────────────────────────────

def last_rows(t, step):
    """t's rows as the last rows of t.shape[0] blocks, `step` values apart."""
    rows, width = t.shape
    buf = torch.zeros(rows * step + 8, dtype=t.dtype, device=t.device)
    v = buf.as_strided((rows, width), (step, 1), 8)
    v.copy_(t)
    return v


LIMIT = 1 << 22   # values between rows up to which the products read them in place, 8 fewer


@pytest.mark.parametrize("step", [LIMIT - 8, LIMIT, LIMIT + 104])
@pytest.mark.parametrize("M,N,K", [(4, 8, 96), (20, 16, 104)])
def test_rows_far_apart(M, N, K, step):
    """x, W and dy with any distance between rows: what copies of them give."""
    case(f"linear {M} x {N} x {K}, rows {step} values apart")
    g = gen(M + N)
    x, w, dy = randn(g, M, K, dtype=BF), randn(g, N, K, dtype=BF, scale=0.1), randn(g, M, N, dtype=BF)
    for act, keep8 in (("none", False), ("tanh", False), ("none", True)):
        got = []
        for xv, wv, dv in ((x, w, dy), (last_rows(x, step), last_rows(w, step), last_rows(dy, step))):
            a, b = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
            y = train.linear(a, b, activation=act, keep8=keep8)
            got.append([y.detach(), *torch.autograd.grad(y, (a, b), dv)])
        assert all(torch.equal(p, q) for p, q in zip(*got)), (act, keep8)


def test_last_token_of_a_long_batch():
    case("linear and channel_mix on the last token's rows of a long batch")
    h = torch.zeros(4, 8200, 512, device=DEV, dtype=BF)
    h[:, -1] = randn(gen(1), 4, 512, dtype=BF)
    w = randn(gen(2), 64, 512, dtype=BF, scale=0.05)
    assert h[:, -1].stride(0) >= LIMIT
    assert torch.equal(train.linear(h[:, -1], w), train.linear(h[:, -1].contiguous(), w))
    one = torch.ones(512, device=DEV)
    with torch.no_grad():
        _, last = train.channel_mix(h, one, None, one, w, w.t().contiguous())
    assert torch.equal(train.linear(last, w), train.linear(last.contiguous(), w))


# ───────────────────────────── gradients of gradients ─────────────────────────────

def test_gradients_of_gradients_by_way_of_dy():
    """dx depends on dy: a second derivative that reaches dy's own inputs, and
    none of the operator's, raises instead of leaving its term out."""
    case("norm and linear: second derivatives through dy")
    g = gen(14)
    x, w, lw = randn(g, 6, 64, dtype=BF).requires_grad_(True), randn(g, 32, 64, dtype=BF), torch.ones(64, device=DEV)
    for f in (lambda: train.layer_norm(x, lw), lambda: train.linear(x, w), lambda: train.linear(x, w, activation="tanh"),
              lambda: train.linear(x, w, None, "none", torch.zeros(6, 32, device=DEV, dtype=BF))):
        y = f()
        v = torch.ones_like(y).requires_grad_(True)
        dx, = torch.autograd.grad((v * y).float().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="gradients of its gradients"):
            torch.autograd.grad(dx.float().sum() + v.float().sum(), v)
    # one that reads no gradient is as before
    y = train.linear(x, w)
    v = torch.ones_like(y).requires_grad_(True)
    dv, = torch.autograd.grad((v * y).float().sum(), v, create_graph=True)
    assert torch.equal(dv, y)


# ───────────────────────────── what is kept of an activation ─────────────────────────────

@pytest.mark.parametrize("dt,bias", [(BF, 2.0 ** -19), (HF, 2.0 ** -21)])
@pytest.mark.parametrize("res", [False, True])
def test_kept_relu_is_not_one_sided(dt, bias, res):
    """Errors of the kept relu(z) cancel over many values.  A remainder taken
    to the nearest step is off by up to 2^-16 (fp16 2^-18) either way; the mean
    of 2^19 such errors is their 700th part, and 2^-3 of a step is left here
    for the byte's clamp (one value in 512, one step) and for the rounding of
    the results, which differs from that of the exact slope for one value in
    2^8 by one step: a standard deviation of 2^-12 / 2^9.5.  Cut off instead of
    rounded, the errors' mean would be four times the bound and more."""
    case(f"mean error of the kept relu {dt} residual {res}")
    n = 1 << 20
    x, w = randn(gen(3), 1, 8, dtype=dt), randn(gen(4), n, 8, dtype=dt)
    b = torch.zeros(n, device=DEV, dtype=dt, requires_grad=True)
    y = train.linear(x, w, b, "relu2", torch.zeros(1, n, device=DEV) if res else None)
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    z = (x.double() @ w.double().t())[0]
    on = z > 0.01
    want = (2 * z).to(dt).double()
    mean = ((db.double() - want) / (2 * z))[on].mean().item()
    print(f"  mean {mean / bias:.3f} of the bound", flush=True)
    assert abs(mean) <= bias


# ───────────────────────────── rounding ─────────────────────────────

@pytest.mark.parametrize("M,N,K", [(5, 64, 8), (64, 96, 8), (33, 31, 9), (1, 40, 2048), (600, 640, 8), (4096, 4096, 8),
                                   (16, 128, 8192)])
def test_bf16_results_round_ties_to_even(M, N, K):
    """Rows with two values that are not zero: exact sums, rounded as torch
    rounds, ties to even, on each of the products' routes."""
    case(f"ties of bf16 results {M} x {N} x {K}")
    g = gen(M + N + K)
    pow2 = lambda *s: torch.exp2(torch.randint(-9, 1, s, generator=g, device=DEV).float())  # noqa: E731
    x, w, dy = (torch.zeros(s, device=DEV) for s in ((M, K), (N, K), (M, N)))
    x[:, 0], x[:, K - 1] = 1.0, pow2(M)
    w[:, 0], w[:, K - 1] = 1.0 + torch.randint(0, 128, (N,), generator=g, device=DEV) / 128, pow2(N)
    dy[:, 0], dy[:, N - 1] = 1.0, pow2(M)
    dy[0], dy[M - 1] = 1.0, pow2(N)
    r = (1.0 + torch.randint(0, 128, (M, N), generator=g, device=DEV) / 128).to(BF)
    x, w, dy = (v.to(BF).requires_grad_(True) for v in (x, w, dy))
    even = lambda v: v.float().to(BF)  # noqa: E731  (the sums are exact in fp32)
    X, W, DY = (v.detach().double() for v in (x, w, dy))
    y = train.linear(x, w)
    assert torch.equal(y, even(X @ W.t()))
    z = X @ W.t()
    yr = train.linear(x.detach(), w.detach(), None, "none", r)
    exact = z.float().double() == z
    assert exact.all() and torch.equal(yr, even(z + r.double()))
    h = train.linear(x.detach(), w.detach(), None, "relu2")
    sq = (z.float() * z.float())    # relu² is a product in fp32
    assert torch.equal(h, sq.to(BF))
    dx, dw = torch.autograd.grad(y, (x, w), dy.detach())
    # rows of two terms each
    assert torch.equal(dx[1:-1], even(DY @ W)[1:-1]) and torch.equal(dw[1:-1], even(DY.t() @ X)[1:-1])
    ties = (z + r.double()).float()
    low = ties.view(torch.int32) & 0xffff
    assert (low == 0x8000).any()   # there are ties among them


def slope64(act, z):
    if act == "tanh":
        return 1 / torch.cosh(z) ** 2
    return torch.sigmoid(z) * torch.sigmoid(-z) if act == "sigmoid" else 2 * z.clamp(min=0)


FUNC = 2.0 ** -20   # relative error of the fp32 e^z (a few units in the last place), for arguments about 1


def swept(dt, n, top):
    """z from −top to top as the product of x [1, 8] and w [n, 8] in two parts, exact in fp32 but for one sum."""
    z = torch.linspace(-top, top, n, device=DEV, dtype=torch.float64)
    w = torch.zeros(n, 8, device=DEV, dtype=dt)
    w[:, 0] = z.to(dt)
    w[:, 1] = ((z - w[:, 0].double()) * 64).to(dt)
    x = torch.zeros(1, 8, device=DEV, dtype=dt)
    x[0, 0], x[0, 1] = 1.0, 2.0 ** -6
    return x, w, (x.double() @ w.double().t())[0]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("act", ["tanh", "sigmoid"])
@pytest.mark.parametrize("how", ["alone", "residual", "keep8"])
def test_slope_where_the_activation_saturates(act, dt, how):
    """The slope keeps its relative precision as it goes to zero.  What is kept
    of z has 16 (bf16) or 18 (fp16) significant bits, to half a step, to one
    where the remainder's byte clamps: 2^-15 and 2^-17 of z, of which the slope
    takes at most 2|z| (tanh), |z| (sigmoid); from the 8-bit checkpoint z is
    what its codes stand for.  The sum z and e^z add 2^-24·2|z|, FUNC·(1 + |z|).
    One row: the bias gradient is dy·slope, rounded once (dy keeps fp16's off
    its subnormals)."""
    case(f"slope of {act} {dt} {how}, z to 16")
    x, w, z = swept(dt, 4096, 16.0)
    b = torch.zeros(4096, device=DEV, dtype=dt, requires_grad=True)
    res = torch.zeros(1, 4096, device=DEV, dtype=dt) if how == "residual" else None
    y = train.linear(x, w, b, act, res, keep8=how == "keep8")
    scale = 2.0 ** 14 if dt == HF else 1.0
    db, = torch.autograd.grad(y, b, torch.full_like(y, scale))
    kept = 2.0 ** -15 if dt == BF else 2.0 ** -17
    if how == "keep8":
        zf = z.float()   # the fp32 sum that the checkpoint is taken of
        z, kept = train.checkpoint8(zf).restore().double(), 0.0
    ref = slope64(act, z) * scale
    tiny = 2.0 ** -25 if dt == HF else 0.0
    rel = 2 * z.abs() * (kept + 2.0 ** -24) + FUNC * (1 + z.abs())
    u = torch.finfo(dt).eps / 2
    bound = ref * (rel + rel ** 2) * (1 + u) + u * ref + tiny
    worst = ((db.double() - ref).abs() / bound).max().item()
    print(f"  worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0


# ───────────────────────────── the padding columns of dz ─────────────────────────────

@pytest.mark.parametrize("N", [1, 3, 8, 16, 64, 505, 512, 513, 2048])
def test_padding_columns_of_dz_are_zeros(N):
    """rwkv_linear_dact writes zeros into every column from N to its pitch."""
    case(f"dact {N} columns, every pitch")
    L = _lib.lib()
    M = 37
    s = torch.cuda.current_stream().cuda_stream
    dy = randn(gen(N), M, N, dtype=BF)
    ws = torch.empty(L.rwkv_linear_dact_workspace(M, N), dtype=torch.uint8, device=DEV)
    for ldz in range(N, N + 8):
        for with_db in (False, True):
            dz = torch.full((M, ldz), float("nan"), device=DEV, dtype=BF)
            db = torch.full((N,), float("nan"), device=DEV, dtype=BF)
            _lib.check(L.rwkv_linear_dact(dy.data_ptr(), N, 1, None, None, 0, None, None, 0, dz.data_ptr(), ldz,
                                          db.data_ptr() if with_db else None, 1, M, N, ws.data_ptr(), ws.numel(), s))
            assert torch.equal(dz[:, :N], dy) and not dz[:, N:].any(), (ldz, with_db)
            if with_db:
                off = 2.0 ** -24 * 64 * dy.double().abs().sum(0) + 2.0 ** -8 * dy.double().sum(0).abs() + 2.0 ** -133
                assert ((db.double() - dy.double().sum(0)).abs() <= off).all()


# ───────────────────────────── forward mode ─────────────────────────────

def test_forward_mode_derivatives_are_refused():
    case("norm and linear: a tangent on the device")
    x, w, one = randn(gen(1), 4, 64, dtype=BF), randn(gen(2), 8, 64, dtype=BF), torch.ones(64, device=DEV)
    r = torch.zeros(4, 8, device=DEV)
    fa = torch.autograd.forward_ad
    with fa.dual_level():
        dual = lambda t: fa.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: train.layer_norm(dual(x), one), lambda: train.layer_norm(x, one, dual(one)),
                  lambda: train.linear(x, dual(w)), lambda: train.linear(x, w, None, "none", dual(r))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        assert train.linear(x, w).shape == (4, 8)   # no tangent among its inputs
        leaf = x.detach().requires_grad_(True)
        for y in (train.layer_norm(leaf, one), train.linear(leaf, w), train.linear(leaf, w, activation="tanh")):
            with pytest.raises(NotImplementedError, match="forward-mode"):   # and of a gradient
                torch.autograd.grad(y, leaf, dual(torch.ones_like(y)))


# ───────────────────────────── odd rows ─────────────────────────────

def test_few_rows_copy_no_weights():
    """A few rows through a W whose rows are not whole chunks: W is read as it
    lies, on every call, not copied into aligned rows first."""
    w = randn(gen(1), 8192, 8195, dtype=BF, scale=0.01)
    for M in (1, 16, 17, 40):
        case(f"memory of a product {M} x 8192 x 8195")
        x = randn(gen(M), M, 8195, dtype=BF)
        with torch.no_grad():
            train.linear(x, w)
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            y = train.linear(x, w)
            used = torch.cuda.max_memory_allocated() - before
        assert used < w.numel() * 2 / 2, (M, used)
        z = x.double() @ w.double().t()
        off = 2.0 ** -24 * (8195 + 32) * (x.double().abs() @ w.double().abs().t())
        assert ((y.double() - z).abs() <= 2.0 ** -8 * z.abs() + off * (1 + 2.0 ** -8)).all()
