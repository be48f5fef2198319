"""Training-side operators on the GPU against plain 64-bit forms.

Tolerances.  With u = finfo.eps / 2 of the output's type (half a step), a value
may be off by u·|value| for its own rounding, plus what its terms may be off by:
2^-24 per fp32 operation in the longest chain of sums (`chain`) times the sum
of the terms' magnitudes, plus u times the magnitude of each operand that the
operator rounds to 16 bits (dz, and the kept activation)."""
import sys

import pytest
import torch

from swiftrwkv_amd import _lib, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
E24 = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}   # half a step near 0
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def case(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def check(what, got, ref, off):
    """|got − ref| <= u·|ref| + off·(1 + u) elementwise, with equal NaNs and infinities."""
    u = torch.finfo(got.dtype).eps / 2
    got64, off = got.double(), torch.as_tensor(off, device=ref.device, dtype=torch.float64)
    assert got64.shape == ref.shape, (what, got64.shape, ref.shape)
    bound = u * ref.abs() + off * (1 + u) + TINY[got.dtype]
    worst = ((got64 - ref).abs() / bound).nan_to_num(nan=float("inf")).max().item() if ref.numel() else 0.0
    print(f"  {what}: worst error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0, (what, worst)


# ───────────────────────────── 8-bit checkpoints ─────────────────────────────

def kept(x):
    """(values, step) of the 8-bit checkpoint of rows x [N, D], by its definition, in 64 bits."""
    N, D = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -D % 32)).reshape(N, (D + 31) // 32, 32)
    top = v.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)
    e = torch.where(top > 0, e - 1, -200).clamp(min=-120)
    step = torch.exp2((e - 6).double())
    val = torch.round(v / step).clamp(-127, 127) * step
    val = torch.where(torch.isfinite(v).all(-1, keepdim=True), val, float("nan"))
    return val.flatten(1)[:, :D], step.expand_as(v).flatten(1)[:, :D]


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("N,D", [(1, 1), (1, 32), (3, 33), (5, 7), (64, 256), (129, 1000), (2, 4097), (4096, 96)])
def test_checkpoint_is_its_definition(N, D, dt):
    case(f"checkpoint8 {N} x {D} {dt}")
    x = randn(gen(N + D), N, D) * torch.exp2(torch.randint(-18, 12, (N, 1), generator=gen(1), device=DEV).float())
    x = x.to(dt)
    c = train.checkpoint8(x)
    assert c.codes.shape == (N, (D + 31) // 32 * 32) and c.nbytes == c.codes.numel() * 33 // 32
    assert torch.equal(c.codes[:, D:], torch.zeros_like(c.codes[:, D:]))
    ref, step = kept(x)
    got = c.restore()
    assert got.dtype == dt and got.shape == x.shape
    assert torch.equal(got, ref.to(dt))
    assert torch.equal(c.restore(F32).double(), ref) and torch.equal(c.restore(BF).double(), ref)
    # half a step, one at the clamped top; and a checkpoint of a restored row is itself
    assert ((ref - x.double()).abs() <= torch.where(x.double().abs() > 127.5 * step, step, step / 2)).all()
    again = train.checkpoint8(c.restore(F32))
    assert torch.equal(again.codes, c.codes) and torch.equal(again.scales, c.scales)


def test_checkpoint_edges():
    case("checkpoint8 edges: zeros, ties, extremes, infinities, NaN")
    x = torch.zeros(8, 64, device=DEV)
    x[1, :3] = torch.tensor([1.0, 2.5 / 64, 3.5 / 64])              # ties to even: codes 64, 2, 4
    x[2, 0] = 3.402823466e38                                         # the largest finite value clamps to 127
    x[3, 0], x[3, 1] = 1e-45, -1e-45                                 # subnormals: under the smallest step
    x[4, 5], x[5, 40], x[6, 0] = float("inf"), float("nan"), -float("inf")
    x[4, 32] = 1.0                                                   # the other group of a bad row
    x[7, 0] = 2.0 ** -120
    c = train.checkpoint8(x)
    got = c.restore()
    ref, _ = kept(x)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got.double().nan_to_num(), ref.nan_to_num())
    assert c.codes[1, :3].tolist() == [64, 2, 4] and c.codes[2, 0] == 127 and torch.isfinite(got[2]).all()
    assert torch.isnan(got[4, :32]).all() and got[4, 32] == 1.0 and c.scales[4, 0] == 255
    assert c.scales[0].tolist() == [7, 7] and got[7, 0] == 2.0 ** -120
    h = torch.full((1, 32), 65504.0, device=DEV, dtype=HF)
    assert torch.isfinite(train.checkpoint8(h).restore()).all()


def test_checkpoint_layouts():
    case("checkpoint8 of views, 3-D and empty")
    big = randn(gen(3), 10, 200, dtype=BF)
    for view in (big[:, 3:103], big[::2, :64], big.t(), big[:, 1::2], big[4], big.reshape(2, 5, 200), big[:1, 7:8],
                 big[:0], big[:1].expand(6, 200)):
        want, _ = kept(view.reshape(-1, view.shape[-1]))
        assert torch.equal(train.checkpoint8(view).restore(), want.reshape(view.shape).to(BF))


# ───────────────────────────── layer norm ─────────────────────────────

def norm64(x, w, b, eps, dy=None, x8=False):
    """y, (dx, dw, db) and their error terms' magnitudes, in 64 bits."""
    x, w = x.double(), w.double()
    D = x.shape[1]
    mean = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    y = (x - mean) * r * w + (0 if b is None else b.double())
    # what x̂ may be off by, per 2^-24: its own size, and the mean's error
    noise = (x - mean).abs() * r + x.abs().mean(-1, keepdim=True) * r
    ymag = noise * w.abs() + (0 if b is None else b.double().abs())
    if dy is None:
        return y, ymag
    dy = dy.double()
    xh = ((kept(x)[0] if x8 else x) - mean) * r
    noise = noise + xh.abs()
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = (g - m1 - xh * m2) * r
    dxmag = (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True) +
             noise * m2.abs() + xh.abs() * (g.abs() * noise).mean(-1, keepdim=True)) * r
    return y, ymag, dx, dxmag, (dy * xh).sum(0), (dy.abs() * noise).sum(0), dy.sum(0), dy.abs().sum(0)


def norm_chain(N, D):
    """fp32 operations in a row: a lane's share of a row (at most 64), the
    trees over lanes and waves, a handful of products; for the columns' sums a
    block's rows and the join of the blocks."""
    return 64 + 6 + 16 + 10, max(1, N // 512) + 4 + 32 + 16 + 10


def run_norm(N, D, xdt, odt, wdt, bias, x8, seed=0, x=None):
    g = gen(seed + N * 131 + D)
    x = (2 * randn(g, N, D) + 0.5).to(xdt) if x is None else x
    w, b = (1 + 0.3 * randn(g, D)).to(wdt), (0.2 * randn(g, D)).to(wdt) if bias else None
    dy = randn(g, N, D, dtype=odt)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = train.layer_norm(leaves[0], leaves[1], leaves[2] if bias else None, 1e-5, out_dtype=odt, keep8=x8)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(train.layer_norm(x, w, b, 1e-5, out_dtype=odt), y.detach())
    ref = norm64(x, w, b, 1e-5, dy, x8)
    row, colc = norm_chain(N, D)
    check("y", y.detach(), ref[0], E24 * row * ref[1])
    check("dx", grads[0], ref[2], E24 * 2 * row * ref[3])
    check("dw", grads[1], ref[4], E24 * (row + colc) * ref[5])
    if bias:
        check("db", grads[2], ref[6], E24 * colc * ref[7])
    return y, grads


@pytest.mark.parametrize("xdt,odt,wdt", [(F32, F32, F32), (F32, BF, F32), (F32, HF, F32), (BF, BF, F32), (BF, BF, BF),
                                         (HF, HF, HF), (HF, HF, F32)])
@pytest.mark.parametrize("N,D", [(1, 1024), (5, 768), (67, 1023), (300, 2049)])
def test_norm_types(N, D, xdt, odt, wdt):
    case(f"norm {N} x {D} {xdt} -> {odt}, weights {wdt}")
    run_norm(N, D, xdt, odt, wdt, True, False)


@pytest.mark.parametrize("x8", [False, True])
@pytest.mark.parametrize("N,D", [(1, 1), (3, 2), (2, 31), (9, 512), (7, 513), (4, 4096), (3, 4097), (2, 8193),
                                 (2, 16384), (2, 16385), (1, 65536), (4097, 64), (5000, 33)])
def test_norm_widths(N, D, x8):
    case(f"norm width {N} x {D} keep8 {x8}")
    run_norm(N, D, F32, F32, F32, D % 2 == 1, x8)


@pytest.mark.parametrize("N,D", [(2050, 2048), (1500, 4096), (700, 5000)])
def test_norm_many_rows_in_8_bits(N, D):
    case(f"norm {N} x {D} bf16 keep8, twice the same bits")
    _, a = run_norm(N, D, BF, BF, F32, True, True)
    _, b = run_norm(N, D, BF, BF, F32, True, True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_norm_rows_of_one_value_and_bad_rows():
    case("norm: constant rows, infinities, NaN")
    x = randn(gen(2), 6, 96)
    x[1] = 3.25
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    w, b = torch.ones(96, device=DEV), torch.zeros(96, device=DEV)
    xl = x.clone().requires_grad_(True)
    y = train.layer_norm(xl, w, b)
    assert torch.equal(y[1], torch.zeros_like(y[1]))
    assert torch.isnan(y[3:5]).all() and torch.isfinite(y[[0, 1, 2, 5]]).all()
    dx, = torch.autograd.grad(y, xl, torch.ones_like(y))
    assert torch.isfinite(dx[[0, 1, 2, 5]]).all() and torch.isnan(dx[3:5]).all()


def test_norm_layouts_and_needs():
    case("norm: views, 3-D, no rows, single gradients, an expanded dy")
    big = randn(gen(5), 40, 301)
    w = (1 + 0.1 * randn(gen(6), 200)).requires_grad_(True)
    for v in (big[:, 3:203], big[::3, 1:201], big[:, 1:201].reshape(4, 10, 200), big.t()[:200].t(),
              big[:1, :200].expand(5, 200), big[7, :200]):
        x = v.detach().requires_grad_(True)
        y = train.layer_norm(x, w)
        ref, mag = norm64(v.reshape(-1, 200), w.detach(), None, 1e-5)
        check("y", y.detach().reshape(-1, 200), ref, E24 * 96 * mag)
        only, = torch.autograd.grad(y.sum(), w, retain_graph=True)      # dy is an expanded scalar
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert torch.equal(only, dw) and dx.shape == v.shape
    e = torch.zeros(0, 200, device=DEV, requires_grad=True)
    y = train.layer_norm(e, w)
    dx, dw = torch.autograd.grad(y, (e, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 200) and torch.equal(dw, torch.zeros_like(w))
    b = torch.zeros(200, device=DEV, requires_grad=True)
    y = train.layer_norm(big[:, :200], w.detach(), b)
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    assert torch.equal(db, torch.full((200,), 40.0, device=DEV))


def directional(f, inputs, which, dy, seed):
    """(direction, central difference of Σ dy·f along it) in 64 bits."""
    d = torch.randn(inputs[which].shape, generator=gen(seed), device=DEV, dtype=torch.float64)
    h = 1e-6
    vals = []
    for sgn in (1, -1):
        a = [None if t is None else t.double() for t in inputs]
        a[which] = a[which] + sgn * h * d
        vals.append((f(*a) * dy.double()).sum())
    return d, (vals[0] - vals[1]) / (2 * h)


def test_norm_gradient_against_differences():
    case("norm: gradients against central differences")
    g = gen(8)
    x, w, b, dy = randn(g, 33, 257), 1 + 0.3 * randn(g, 257), randn(g, 257), randn(g, 33, 257)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(train.layer_norm(*leaves), leaves, dy)
    f = lambda x, w, b: norm64(x, w, b, 1e-5)[0]  # noqa: E731
    ref = norm64(x, w, b, 1e-5, dy)
    for i, mag in ((0, ref[3]), (1, ref[5]), (2, ref[7])):
        d, want = directional(f, (x, w, b), i, dy, 20 + i)
        got = (grads[i].double() * d).sum()
        # the gradient's own bound, and the difference's: h² of a curvature of
        # order one and 64-bit cancellation over h, both under 1e-7 of the sum's size
        off = (E24 * 300 * mag * d.abs()).sum() + 1e-7 * (grads[i].double() * d).abs().sum()
        assert abs(got - want) <= off, (i, got, want, off)


# ───────────────────────────── dense products ─────────────────────────────

ACT = {"none": lambda z: z, "relu2": lambda z: z.clamp(min=0) ** 2, "tanh": torch.tanh, "sigmoid": torch.sigmoid}
SLOPE = {"none": lambda z: torch.ones_like(z), "relu2": lambda z: 2 * z.clamp(min=0),
         "tanh": lambda z: 1 - torch.tanh(z) ** 2, "sigmoid": lambda z: torch.sigmoid(z) * torch.sigmoid(-z)}
FUNC = 2.0 ** -20   # relative error of the fp32 tanh and e^z (a few units in the last place)


def run_linear(M, N, K, dt, act="none", bias=False, res=None, x8=False, seed=0, scale=1.0):
    case(f"linear {M} x {N} x {K} {dt} {act} bias {bias} residual {res} keep8 {x8}")
    g = gen(seed + 7 * M + 3 * N + K)
    x, w = randn(g, M, K, dtype=dt), randn(g, N, K, dtype=dt, scale=scale / K ** 0.5)
    b = randn(g, N, dtype=dt, scale=0.3) if bias else None
    r = randn(g, M, N, dtype=res) if res else None
    leaves = {k: t.detach().clone().requires_grad_(True) for k, t in (("x", x), ("w", w), ("b", b), ("r", r))
              if t is not None}
    y = train.linear(leaves["x"], leaves["w"], leaves.get("b"), act, leaves.get("r"), keep8=x8)
    dy = randn(g, M, N, dtype=y.dtype)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        assert torch.equal(train.linear(x, w, b, act, r), y.detach())
    u = torch.finfo(dt).eps / 2
    X, W, DY = x.double(), w.double(), dy.double()
    z = X @ W.t() + (0 if b is None else b.double())
    bz = E24 * (K + 32) * (X.abs() @ W.abs().t() + (0 if b is None else b.double().abs()))   # what z may be off by
    a = ACT[act](z)
    ea = {"none": bz, "relu2": 2 * z.clamp(min=0) * bz + bz ** 2, "tanh": bz, "sigmoid": bz}[act] + FUNC * a.abs()
    yr = a + (0 if r is None else r.double())
    check("y", y.detach(), yr, ea + E24 * yr.abs())
    # the slope, from what is kept: the activation in 16 bits, or z in 8
    s = SLOPE[act](z)
    tiny = TINY[dt]
    if act == "none":
        es = torch.zeros_like(z)
    elif x8:
        step = kept(z)[1] * 2 + bz    # one step; the next larger where the group's top rounds over a power of two
        es = {"relu2": 2.0, "tanh": 1.0, "sigmoid": 0.25}[act] * step
    else:
        es = {"relu2": 2 * (u * z.clamp(min=0) + bz + tiny), "tanh": 2 * a.abs() * (u * a.abs() + bz + tiny),
              "sigmoid": u * a + bz + tiny}[act] + 4 * E24
    dz = DY * s
    ez = DY.abs() * es
    check_z = ez + u * (dz.abs() + ez) + tiny      # dz is rounded for the products
    Xk = kept(x)[0] if x8 else X
    check("dx", grads["x"], dz @ W, check_z @ W.abs() + E24 * (N + 32) * (dz.abs() @ W.abs()))
    check("dw", grads["w"], dz.t() @ Xk, check_z.t() @ Xk.abs() + E24 * (M + 32) * (dz.abs().t() @ Xk.abs()))
    if b is not None:
        check("db", grads["b"], dz.sum(0), ez.sum(0) + E24 * (M // 16 + 64) * dz.abs().sum(0))
    if r is not None:
        assert torch.equal(grads["r"], dy)
    return y, grads


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("act", ["none", "relu2", "tanh", "sigmoid"])
@pytest.mark.parametrize("bias,res,x8", [(False, None, False), (True, "own", False), (True, "f32", True),
                                         (False, None, True)])
def test_linear_epilogues(dt, act, bias, res, x8):
    run_linear(150, 200, 136, dt, act, bias, {None: None, "own": dt, "f32": F32}[res], x8)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 512, 768), (16, 96, 256), (17, 33, 65),
                                   (64, 64, 64), (65, 127, 129), (128, 256, 320), (257, 511, 264), (1000, 24, 40),
                                   (3, 2048, 1000), (2048, 3, 1000), (300, 300, 2050), (513, 1025, 72)])
def test_linear_sizes(M, N, K):
    run_linear(M, N, K, BF if (M + N + K) % 2 else HF, "relu2", True, None, False)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (4, 1024, 4096), (40, 4096, 2048), (4096, 96, 2048),
                                   (4096, 2048, 96), (2304, 2560, 520), (4096, 4096, 256), (600, 4104, 1032)])
def test_linear_large(M, N, K):
    run_linear(M, N, K, BF, "relu2", False, F32, False)
    run_linear(M, N, K, HF, "tanh", True, None, True, seed=1)


@pytest.mark.parametrize("M,N,K", [
    (16, 512, 1024), (16, 33, 1023), (9, 8192, 1100), (16, 8200, 2056), (17, 512, 1024),   # few rows, and one more
    (2048, 4096, 640), (1024, 8192, 320),                                                  # 256 x 128 tiles
    (4096, 4096, 328), (4864, 4096, 1032), (5120, 4096, 4096),                             # 256 x 256, whole rounds and a rest
    (512, 384, 8192), (130, 250, 6000),                                                    # ranges of K
    (300, 200, 1021), (2050, 1030, 515), (1100, 1030, 1001), (20, 14000, 4099)])           # odd rows, the last three padded
def test_linear_routes(M, N, K):
    run_linear(M, N, K, BF, "tanh", True, None, False)
    run_linear(M, N, K, HF, "relu2", False, F32, (M + K) % 3 == 0, seed=2)
    run_linear(M, N, K, BF, "none", False, None, False, seed=3)


def test_linear_misaligned_rows_and_gradients():
    """x, W and dy as views that start between 16-byte chunks, of one width."""
    case("linear: misaligned views of x, W and dy")
    g = gen(21)
    for M, N, K in ((40, 96, 128), (10, 96, 128), (70, 64, 200)):
        x, w = randn(g, M, K + 8, dtype=BF)[:, 1:K + 1], randn(g, N, K + 8, dtype=BF, scale=0.1)[:, 3:K + 3]
        dy = randn(g, M, N + 8, dtype=BF)[:, 5:N + 5]
        xa, wa = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = train.linear(xa, wa)
        dx, dw = torch.autograd.grad(y, (xa, wa), dy)
        X, W, DY = x.double(), w.double(), dy.double()
        check("y", y.detach(), X @ W.t(), E24 * (K + 32) * (X.abs() @ W.abs().t()))
        check("dx", dx, DY @ W, E24 * (N + 32) * (DY.abs() @ W.abs()))
        check("dw", dw, DY.t() @ X, E24 * (M + 32) * (DY.abs().t() @ X.abs()))


def test_kept_activation_has_eight_more_bits():
    """tanh's and relu²'s gradients through an fp32 residual, whose dy of 1
    shows the slope before its rounding to dz: db sums it in fp32.  One row:
    db = slope, off by its own rounding, the kept value's 2^-16 (bf16) or
    2^-18 (fp16) of the activation and the fp32 function."""
    for dt, bits in ((BF, 2.0 ** -16), (HF, 2.0 ** -18)):
        for act, res in (("tanh", False), ("tanh", True), ("sigmoid", False), ("relu2", False), ("relu2", True)):
            case(f"kept {act} {dt} residual {res}")
            g = gen(5)
            x, w = randn(g, 1, 64, dtype=dt), randn(g, 640, 64, dtype=dt, scale=0.2)
            b = torch.zeros(640, device=DEV, dtype=dt, requires_grad=True)
            r = torch.zeros(1, 640, device=DEV) if res else None
            y = train.linear(x, w, b, act, r)
            db, = torch.autograd.grad(y, b, torch.ones_like(y))
            z = (x.double() @ w.double().t())[0]
            bz = E24 * 96 * (x.double().abs() @ w.double().abs().t())[0]
            a = ACT[act](z)
            kept_off = {"tanh": 2 * a.abs() * a.abs(), "sigmoid": a, "relu2": 2 * z.clamp(min=0)}[act] * bits
            check("slope", db, SLOPE[act](z), kept_off + 2 * bz + FUNC * (1 + a.abs()) + TINY[dt] * 2)


def test_linear_layouts_and_needs():
    case("linear: views, 3-D, no rows, single gradients")
    g = gen(11)
    big, wbig = randn(g, 60, 400, dtype=BF), randn(g, 90, 400, dtype=BF, scale=0.05)
    plain = train.linear(big[:, 8:136].contiguous(), wbig[:, 8:136].contiguous())
    assert torch.equal(train.linear(big[:, 8:136], wbig[:, 8:136]), plain)                     # pitched, aligned
    odd = train.linear(big[:, 3:131], wbig[:, 3:131])                                          # pitched, misaligned
    ref = big[:, 3:131].double() @ wbig[:, 3:131].double().t()
    mag = big[:, 3:131].double().abs() @ wbig[:, 3:131].double().abs().t()
    check("misaligned", odd, ref, E24 * 160 * mag)
    x3 = big[:, :128].reshape(3, 20, 128)
    assert torch.equal(train.linear(x3, wbig[:, :128]), train.linear(x3.reshape(60, 128), wbig[:, :128]).reshape(3, 20, 90))
    assert train.linear(x3[0, 0], wbig[:, :128]).shape == (90,)
    xt = big[:60, :60].t()
    check("transposed", train.linear(xt, wbig[:, :60]), xt.double() @ wbig[:, :60].double().t(),
          E24 * 92 * (xt.double().abs() @ wbig[:, :60].double().abs().t()))
    w = wbig[:, :128].contiguous().requires_grad_(True)
    b = torch.zeros(90, device=DEV, dtype=BF, requires_grad=True)
    e = torch.zeros(0, 128, device=DEV, dtype=BF, requires_grad=True)
    for act in ("none", "relu2"):
        y = train.linear(e, w, b, act)
        de, dw, db = torch.autograd.grad(y, (e, w, b), torch.zeros_like(y))
        assert y.shape == (0, 90) and de.shape == (0, 128) and not dw.any() and not db.any()
        x = big[:, :128].contiguous().requires_grad_(True)
        y = train.linear(x, w, b, act)
        dy = randn(g, 60, 90, dtype=BF)
        both = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
        for i, t in enumerate((x, w, b)):
            one, = torch.autograd.grad(y, t, dy, retain_graph=True)
            assert torch.equal(one, both[i])
        # a dy that is a slice of wider rows, whose other columns are no zeros
        wide = torch.full((60, 104), float("nan"), device=DEV, dtype=BF)
        wide[:, :90] = dy
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, w, b), wide[:, :90]), both))


def test_linear_bad_values_stay_in_their_rows():
    case("linear: NaN and infinity in one row reach that row alone")
    for K, N in ((128, 96), (131, 77)):
        x, w = randn(gen(1), 70, K, dtype=HF), randn(gen(2), N, K, dtype=HF, scale=0.1)
        x[5, K - 1], x[69, 0] = float("nan"), float("inf")
        for act in ("none", "relu2", "tanh", "sigmoid"):
            y = train.linear(x, w, activation=act)
            keep = [i for i in range(70) if i not in (5, 69)]
            assert torch.isnan(y[5]).all() and torch.isfinite(y[keep]).all()
        w2 = w.clone()
        w2[3, K - 1] = float("nan")
        y = train.linear(x[:5], w2)
        assert torch.isnan(y[:, 3]).all() and torch.isfinite(y[:, [c for c in range(N) if c != 3]]).all()


def test_linear_gradient_against_differences():
    g = gen(9)
    for act in ("relu2", "tanh", "sigmoid"):
        case(f"linear {act}: gradients against central differences")
        x, w = randn(g, 40, 56, dtype=HF), randn(g, 48, 56, dtype=HF, scale=0.13)
        b, dy = randn(g, 48, dtype=HF), randn(g, 40, 48, dtype=HF)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(train.linear(*leaves, act), leaves, dy)
        f = lambda x, w, b: ACT[act](x @ w.t() + b)  # noqa: E731
        dz = (dy.double() * SLOPE[act](x.double() @ w.double().t() + b.double())).abs()
        mags = (dz @ w.double().abs(), dz.t() @ x.double().abs(), dz.sum(0))
        for i in range(3):
            d, want = directional(f, (x, w, b), i, dy, 30 + i)
            got = (grads[i].double() * d).sum()
            # u for the result, dz and the kept activation (whose slope may be twice as far off)
            off = 2.0 ** -11 * ((4 * mags[i] + dy.double().abs().sum() / 100 + grads[i].double().abs()) * d.abs()).sum()
            assert abs(got - want) <= off, (act, i, got, want, off)


def test_streams_and_repeats():
    case("norm and linear on another stream, and twice the same bits")
    g = gen(12)
    x, w = randn(g, 500, 640, dtype=BF), randn(g, 384, 640, dtype=BF, scale=0.04)
    lw = torch.ones(640, device=DEV)

    def go():
        a, b, c = (t.detach().clone().requires_grad_(True) for t in (x, w, lw))
        y = train.linear(train.layer_norm(a, c, keep8=True), b, activation="relu2", keep8=True)
        return [y.detach(), *torch.autograd.grad(y, (a, b, c), torch.ones_like(y))]

    here = go()
    assert all(torch.equal(p, q) for p, q in zip(here, go()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = go()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(here, there))


def test_what_autograd_refuses():
    case("norm and linear: gradients of gradients, a kept tensor changed in place, a second backward pass")
    g = gen(14)
    x = randn(g, 6, 64, dtype=BF).requires_grad_(True)
    w, lw = randn(g, 32, 64, dtype=BF).requires_grad_(True), torch.ones(64, device=DEV)
    for f in (lambda: train.layer_norm(x, lw), lambda: train.linear(x, w, activation="tanh")):
        y = f()
        dx, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
        with pytest.raises(RuntimeError, match="gradients of its gradients"):
            torch.autograd.grad(dx.float().sum(), x)
        y = f()
        y.backward(torch.ones_like(y))
        with pytest.raises(RuntimeError, match="second time"):
            y.backward(torch.ones_like(y))
    y = train.linear(x, w, activation="tanh")
    with torch.no_grad():
        y.mul_(2)                            # tanh's gradient reads y
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x, torch.ones_like(y))
    assert x.grad.shape == x.shape and w.grad.shape == w.shape


def test_forward_in_a_graph():
    case("norm, linear and checkpoint captured into a graph, replayed between eager work")
    g = gen(13)
    x, w = randn(g, 24, 1024, dtype=BF), randn(g, 256, 1024, dtype=BF, scale=0.03)
    lw = torch.ones(1024, device=DEV)

    def go():
        h = train.layer_norm(x, lw)
        return train.linear(h, w, activation="relu2"), train.checkpoint8(h).restore()

    with torch.no_grad():
        want = go()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = go()
        torch.cuda.current_stream().wait_stream(side)
        for k in range(4):
            x.copy_(randn(gen(50 + k), 24, 1024, dtype=BF))
            graph.replay()
            torch.cuda.synchronize()
            want = go()
            assert all(torch.equal(p, q) for p, q in zip(out, want)), k


# ───────────────────────────── together ─────────────────────────────

@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("B,T,D,F,dt", [(2, 33, 128, 512, BF), (1, 1, 256, 640, HF), (3, 50, 192, 200, HF)])
def test_channel_mix(B, T, D, F, dt, keep8):
    """The whole half block against 64-bit autograd of its formulas: relative
    2-norms, 16 half steps of the 16-bit type for its eight rounded values in
    a row (8-bit checkpoints: their step, 2^-6 of a group's top, for the two
    activations and the norm's row, an average over a row of 32)."""
    case(f"channel_mix {B} x {T} x {D} x {F} {dt} keep8 {keep8}")
    g = gen(B * T + D)
    x = randn(g, B, T, D)
    lw, lb, xk = 1 + 0.1 * randn(g, D), 0.1 * randn(g, D), torch.rand(D, generator=g, device=DEV)
    key, val = randn(g, F, D, dtype=dt, scale=D ** -0.5), randn(g, D, F, dtype=dt, scale=F ** -0.5)
    shift = randn(g, B, D, dtype=dt)
    dy = randn(g, B, T, D)
    leaves = [t.clone().requires_grad_(True) for t in (x, lw, lb, xk, key, val, shift)]
    y, last = train.channel_mix(*leaves, keep8=keep8)
    grads = torch.autograd.grad(y, leaves, dy)
    big = [t.detach().double().requires_grad_(True) for t in (x, lw, lb, xk, key, val, shift)]
    X, LW, LB, XK, KY, VL, SH = big
    m = X.mean(-1, keepdim=True)
    xl = (X - m) / torch.sqrt((X - m).square().mean(-1, keepdim=True) + 1e-5) * LW + LB
    prev = torch.cat([SH.unsqueeze(1), xl[:, :-1]], 1)
    xkk = xl + (prev - xl) * XK
    ref = X + (torch.relu(xkk @ KY.t()) ** 2) @ VL.t()
    want = torch.autograd.grad(ref, big, dy.double())
    u = torch.finfo(dt).eps / 2
    tol = 16 * u + (2.0 ** -5 if keep8 else 0)
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    assert y.dtype == F32 and rel(y.detach(), ref.detach()) <= 16 * u and rel(last.detach(), xl[:, -1].detach()) <= 2 * u
    for name, a, b in zip(("x", "ln_weight", "ln_bias", "x_k", "key", "value", "shift"), grads, want):
        print(f"  d{name}: {rel(a, b):.2e}", flush=True)
        assert a.shape == b.shape and rel(a, b) <= tol, name
