"""Gated products on the GPU against plain 64-bit forms.

Tolerances.  A pre-activation z is an fp32 sum of K products: 2^-24·(K + 32) of
their magnitudes' sum.  act and its slope carry that on by the largest slope and
curvature there is, and add FUNC·(1 + |z|) of their size for the fp32 σ (as the
dense products' tests take it).  The backward pass has z in 16 (bf16) or 18
(fp16) bits, to one step where the remainder's byte clamps, and rounds dz to 16
bits: half a step of its type."""
import sys

import pytest
import torch

from swiftrwkv_amd import _lib, train

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
E24, FUNC = 2.0 ** -24, 2.0 ** -20
TINY = {BF: 2.0 ** -133, HF: 2.0 ** -25}
KEPT = {BF: 2.0 ** -15, HF: 2.0 ** -17}
GATES = train.GATES


def case(msg):
    print(f"[case] {msg}", flush=True)
    sys.stdout.flush()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def act64(name, z):
    """act, act' and act'' (its largest magnitude) in 64 bits."""
    s = torch.sigmoid(z)
    if name == "relu2":
        return z.clamp(min=0) ** 2, 2 * z.clamp(min=0), 2.0
    if name == "sigmoid":
        return s, s * torch.sigmoid(-z), 0.1
    if name == "silu":
        return z * s, s + z * s * torch.sigmoid(-z), 0.5
    a = 2 * (2 / torch.pi) ** 0.5
    u, du = a * (z + 0.044715 * z ** 3), a * (1 + 3 * 0.044715 * z ** 2)
    s = torch.sigmoid(u)
    return z * s, s + z * s * torch.sigmoid(-u) * du, 0.81


def act_off(name, z, ez):
    """What act(z) in fp32 may be off by for a z off by ez."""
    v, d, c = act64(name, z)
    return (d.abs() + c * ez) * ez + FUNC * (1 + z.abs()) * v.abs() + (E24 * v.abs())


def slope_off(name, z, ez):
    v, d, c = act64(name, z)
    if name == "relu2":
        return 2 * ez + E24 * d
    size = {"sigmoid": d, "silu": d.abs() + v.abs(), "gelu_tanh": d.abs() + v.abs() * (1 + z * z)}[name]
    return c * ez + 2 * FUNC * (1 + z.abs()) * size + E24 * size


def check(what, got, ref, off):
    u = torch.finfo(got.dtype).eps / 2
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bound = u * (ref.abs() + off) + off + TINY[got.dtype]
    w = ((got.double() - ref).abs() / bound).nan_to_num(nan=float("inf")).max().item() if got.numel() else 0.0
    print(f"  {what}: worst error {w:.3f} of its bound", flush=True)
    assert w <= 1.0, (what, w)


def run(M, F, K, dt, act, x=None, w=None, dy=None):
    g = gen(M + 3 * F + 7 * K)
    x = randn(g, M, K, dtype=dt) if x is None else x
    w = randn(g, 2 * F, K, dtype=dt, scale=1.5 * K ** -0.5) if w is None else w
    dy = randn(g, M, F, dtype=dt) if dy is None else dy
    a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y = train.gated_linear(a, b, act)
    dx, dw = torch.autograd.grad(y, (a, b), dy)
    with torch.no_grad():
        assert torch.equal(train.gated_linear(x, w, act), y)
    X, W, DY = x.double(), w.double(), dy.double()
    z, ez = X @ W.t(), E24 * (K + 32) * (X.abs() @ W.abs().t())
    (zg, zu), (eg, eu) = z.chunk(2, 1), ez.chunk(2, 1)
    v, d, _ = act64(act, zg)
    ev = act_off(act, zg, eg)
    check("y", y.detach(), v * zu, ev * (zu.abs() + eu) + v.abs() * eu + E24 * (v * zu).abs())
    u = torch.finfo(dt).eps / 2
    eg, eu = eg + KEPT[dt] * zg.abs() + TINY[dt], eu + KEPT[dt] * zu.abs() + TINY[dt]
    ev, ed = act_off(act, zg, eg), slope_off(act, zg, eg)
    dz = torch.cat([DY * zu * d, DY * v], 1)
    off = torch.cat([DY.abs() * (ed * (zu.abs() + eu) + d.abs() * eu), DY.abs() * ev], 1)
    off = off + (u + 4 * E24) * (dz.abs() + off) + TINY[dt]
    check("dx", dx, dz @ W, off @ W.abs() + E24 * (2 * F + 64) * ((dz.abs() + off) @ W.abs()))
    check("dw", dw, dz.t() @ X, off.t() @ X.abs() + E24 * (M + 64) * ((dz.abs() + off).t() @ X.abs()))
    return y, dx, dw


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("act", GATES)
@pytest.mark.parametrize("M,F,K", [(1, 40, 64), (20, 72, 96), (150, 200, 333)])
def test_gates(M, F, K, act, dt):
    case(f"gated {M} x {F} x {K} {act} {dt}")
    run(M, F, K, dt, act)


@pytest.mark.parametrize("M,F,K", [(1, 1, 1), (1, 5, 8), (2, 8, 7), (3, 17, 33), (16, 40, 64), (16, 4099, 2056), (9, 4096, 1031), (17, 64, 64),
                                   (17, 100, 1000), (40, 3, 4096), (64, 512, 512), (100, 96, 4096), (129, 257, 515), (300, 1000, 600),
                                   (1000, 1001, 1000), (1024, 1024, 1024), (2048, 2048, 512), (4096, 4096, 256), (4096, 1037, 520),
                                   (130, 2050, 4099), (700, 3001, 2001), (256, 64, 16384), (2500, 6000, 1024),
                                   (16, 2100, 4096), (16, 2100, 4104), (13, 2200, 5000), (9, 2100, 7280), (5, 2100, 13100), (1, 2064, 32768),
                                   (1, 2050, 65530), (2, 64, 16384), (7, 4100, 513), (16, 4200, 512), (3, 9000, 40), (12, 8200, 1027),
                                   (4, 6000, 2040), (200, 300, 8192), (1000, 1200, 8192), (700, 6000, 4096), (700, 3000, 8192), (1500, 6000, 4096),
                                   (100, 1200, 4097), (1500, 3000, 1003)])
def test_gated_routes(M, F, K):
    case(f"gated {M} x {F} x {K}")
    a = run(M, F, K, BF, "silu")
    b = run(M, F, K, BF, "silu")
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("M,F,K", [(20, 48, 64), (140, 520, 256), (600, 640, 512), (4096, 2048, 512), (200, 300, 8192), (1000, 1200, 8192),
                                   (700, 6000, 4096), (700, 3000, 8192), (1500, 6000, 4096), (100, 1200, 4097), (1500, 3000, 1003)])
def test_gated_is_two_products(M, F, K):
    """Both halves of W where they belong, whatever the tile: W's rows one at a
    time are zero but for one column, so each z is one value of x."""
    case(f"gated columns {M} x {F} x {K}")
    x = torch.randint(-8, 9, (M, K), generator=gen(1), device=DEV).to(HF)
    at = torch.randint(0, K, (2 * F,), generator=gen(2), device=DEV)
    w = torch.zeros(2 * F, K, device=DEV, dtype=HF)
    w[torch.arange(2 * F, device=DEV), at] = 1.0
    y = train.gated_linear(x, w, "relu2")
    assert torch.equal(y, (x[:, at[:F]].float().clamp(min=0) ** 2 * x[:, at[F:]].float()).to(HF))


def test_gated_past_2_31_values():
    """More than 2^31 pre-activations: small integers and W's rows of a single
    one, so that every value of the last rows is exact."""
    M, F, K, n = 76000, 14336, 64, 40
    case(f"gated {M} x {F} x {K}")
    x = torch.randint(-8, 9, (M, K), generator=gen(1), device=DEV).to(HF)
    at = torch.randint(0, K, (2 * F,), generator=gen(2), device=DEV)
    w = torch.zeros(2 * F, K, device=DEV, dtype=HF)
    w[torch.arange(2 * F, device=DEV), at] = 1.0
    a = x.detach().requires_grad_(True)
    y = train.gated_linear(a, w, "relu2")
    dy = torch.zeros(M, F, device=DEV, dtype=HF)
    dy[-n:, 0], dy[-n:, F - 1], dy[-n:, F // 2 + 1] = 1.0, -2.0, 1.0
    dx, = torch.autograd.grad(y, a, dy)
    zg, zu = x[-n:, at[:F]].float(), x[-n:, at[F:]].float()
    r = zg.clamp(min=0)
    assert torch.equal(y[-n:], (r * r * zu).to(HF))
    d = dy[-n:].float()
    dz = torch.cat([d * zu * 2 * r, d * r * r], 1)
    want = torch.zeros(n, K, device=DEV).index_add_(1, at, dz)
    assert torch.equal(dx[-n:], want.to(HF)) and not dx[:-n].any()
    del x, y, dy, dx, a
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M,F,K", [(1, 1, 1), (3, 5, 8), (16, 33, 40), (16, 4099, 64), (40, 100, 64), (130, 70, 72), (300, 1001, 600), (1030, 2055, 136),
                                   (50, 60, 4096), (700, 1500, 2048)])
def test_gated_writes_its_rows_alone(M, F, K):
    """The result, both kept pre-activations and dz, into the middle of buffers."""
    case(f"gated {M} x {F} x {K} into the middle of buffers")
    L, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    x, w, dy = randn(gen(1), M, K, dtype=BF), randn(gen(2), 2 * F, K, dtype=BF, scale=K ** -0.5), randn(gen(3), M, F, dtype=BF)
    ldz = (2 * F + 7) // 8 * 8
    put = lambda n, dt: torch.full((n + 128,), 7, device=DEV, dtype=dt)  # noqa: E731
    h, aux, rem, dz = put(M * F, BF), put(2 * M * F, BF), put(2 * M * F, torch.uint8), put(M * ldz, BF)
    ws = torch.empty(max(L.rwkv_gated_fwd_workspace(M, F, K), 16), dtype=torch.uint8, device=DEV)
    at = lambda t: t[64:].data_ptr()  # noqa: E731
    _lib.check(L.rwkv_gated_fwd(x.data_ptr(), K, w.data_ptr(), K, at(h), at(aux), at(rem), 2, _lib.BF16, M, F, K, ws.data_ptr(), ws.numel(), s))
    _lib.check(L.rwkv_gated_dact(dy.data_ptr(), F, at(aux), at(rem), 2, at(dz), ldz, _lib.BF16, M, F, s))
    for t in (h, aux, rem, dz):
        assert (t[:64] == 7).all() and (t[-64:] == 7).all()
    assert torch.equal(h[64:-64].reshape(M, F), train.gated_linear(x, w))


def test_gated_layouts():
    case("gated: views, one row, several axes, far rows, expanded dy")
    g = gen(5)
    big, wide = randn(g, 30, 500, dtype=BF), randn(g, 64, 700, dtype=BF, scale=0.1)
    for x, w in ((big[:, 3:103], wide[:, :100]), (big[::3, :96], wide[:, 100:196]), (big.t()[:96], wide[::2, :30]),
                 (big[:, ::5], wide[:, ::7]), (big.reshape(5, 6, 500)[..., :64], wide[:50, 1:65]), (big[4, :64], wide[:, :64]),
                 (big[:1, :64].expand(9, 64), wide.t()[:64, :].t()[:, :64]), (big[:0, :64], wide[:, :64])):
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        c, d = x.detach().contiguous().requires_grad_(True), w.detach().contiguous().requires_grad_(True)
        ya, yc = train.gated_linear(a, b), train.gated_linear(c, d)
        F = w.shape[0] // 2
        assert ya.shape == (*x.shape[:-1], F) and torch.equal(ya, yc)
        dy = randn(gen(2), *ya.shape[:-1], 2 * F, dtype=BF)
        ga = torch.autograd.grad(ya, (a, b), dy[..., F:])
        gc = torch.autograd.grad(yc, (c, d), dy[..., F:].contiguous())
        assert all(torch.equal(p, q) for p, q in zip(ga, gc))
        y1, y2 = train.gated_linear(a, b), train.gated_linear(c, d)
        e1, = torch.autograd.grad(y1.float().sum(), a)
        e2, = torch.autograd.grad(y2, c, torch.ones_like(y2))
        assert torch.equal(e1, e2)
    step = (1 << 22) + 104   # rows further apart than the products reach
    buf = torch.zeros(20 * step + 8, device=DEV, dtype=BF)
    x = buf.as_strided((20, 64), (step, 1), 8)
    x.copy_(big[:20, :64])
    assert torch.equal(train.gated_linear(x, wide[:, :64]), train.gated_linear(big[:20, :64], wide[:, :64]))


def test_gated_values():
    """Infinities and NaN stay in their rows and columns; where σ saturates z passes or nothing does."""
    case("gated: extremes")
    K, F = 8, 12
    for act in GATES:
        w = torch.zeros(2 * F, K, device=DEV, dtype=BF)
        w[:, 0] = 1.0
        z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 100.0, -100.0, 1e4, -1e4, 1e18, -1e18, float("nan")], device=DEV)
        x = torch.zeros(z.numel(), K, device=DEV, dtype=BF)
        x[:, 0] = z.to(BF)
        w[F:, 0] = 0.0
        w[F:, 1] = 1.0
        x[:, 1] = 1.0
        a, b = x.requires_grad_(True), w.requires_grad_(True)
        y = train.gated_linear(a, b, act)
        dx, dw = torch.autograd.grad(y, (a, b), torch.ones_like(y))
        zz = x.detach()[:, 0].double()
        v, d, _ = act64(act, zz.clamp(-1e15, 1e15))
        v = torch.where(zz.abs() > 1e15, (zz ** 2 if act == "relu2" else zz if act != "sigmoid" else 1.0) * (zz > 0), v)
        fin = slice(0, 12)
        assert torch.isnan(y[12]).all() and torch.isfinite(dx[fin]).all() and torch.isnan(dx[12, 0])
        off = FUNC * 64 * v.abs()[fin, None] + 1e-37
        check(act, y.detach()[fin], v[fin, None].expand(-1, F), off.expand(-1, F))
        d = torch.where(zz.abs() > 1e15, (2 * zz if act == "relu2" else 1.0 if act != "sigmoid" else 0.0) * (zz > 0), d)
        # twelve equal columns; dz is rounded
        check(act + " dz", dx[fin, 0], 12 * d[fin], 12 * ((2.0 ** -8 + FUNC * 64) * d.abs() + 2.0 ** -13 * (d.abs() > 0))[fin])


@pytest.mark.parametrize("dt,bits", [(BF, (0x7fc0, 0x7fff, -1, -64, 0x7f81)), (HF, (0x7e00, 0x7fff, -1, -512, 0x7c01))])
def test_gated_nan_of_any_pattern(dt, bits):
    """A NaN in x reaches the result and both gradients, whatever its bits and
    sign, on the kernels for few rows and for tiles; other rows stay clean."""
    case(f"gated: NaN patterns {dt}")
    for M in (8, 200):
        for act in GATES:
            x, w = randn(gen(1), M, 64, dtype=dt), randn(gen(2), 48, 64, dtype=dt, scale=0.1)
            for i, b in enumerate(bits):
                x[i].view(torch.int16)[3 + i] = b
            n = len(bits)
            assert torch.isnan(x[:n]).any(1).all() and not torch.isnan(x[n:]).any()
            a, c = x.requires_grad_(True), w.requires_grad_(True)
            y = train.gated_linear(a, c, act)
            dx, = torch.autograd.grad(y, a, torch.ones_like(y))
            assert torch.isnan(y[:n]).all() and torch.isfinite(y[n:]).all()
            assert torch.isnan(dx[:n]).all() and torch.isfinite(dx[n:]).all()


@pytest.mark.parametrize("M,F,K", [(4, 512, 8), (300, 512, 8)])
def test_kept_pre_activations_are_not_one_sided(M, F, K):
    """bf16: the mean error of the kept 24 bits.  Values' errors are up to 2^-17
    of their size either way (half a step of 2^-16), their mean over 2^11 values
    and more under 2^-17/2^4; cut off they would all lie one way, 2^-17 in the
    mean.  Seen through dzu = dy·act(zg) with relu², act = z²: twice that."""
    case(f"kept bits of {M} x {F}")
    L = _lib.lib()
    x, w = randn(gen(1), M, K, dtype=BF), randn(gen(2), 2 * F, K, dtype=BF)
    h, aux = torch.empty(M, F, device=DEV, dtype=BF), torch.empty(M, 2 * F, device=DEV, dtype=BF)
    rem = torch.empty(M, 2 * F, device=DEV, dtype=torch.int8)
    n = L.rwkv_gated_fwd_workspace(M, F, K)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
    _lib.check(L.rwkv_gated_fwd(x.data_ptr(), K, w.data_ptr(), K, h.data_ptr(), aux.data_ptr(), rem.data_ptr(), 0, _lib.BF16, M, F, K,
                                ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    z = x.double() @ w.double().t()
    bits = aux.float().view(torch.int32) + rem.int() * 256
    kept = bits.view(torch.float32).double()
    on = z.abs() > 0.5   # where the fp32 sum's own error, 2^-24·8 of its terms, says nothing
    rel = ((kept - z) / z)[on]
    off = 2.0 ** -17 + 2.0 ** -21 * 8 / 0.5
    print(f"  mean {rel.mean().item() * 2 ** 17:.3f}, most {rel.abs().max().item() * 2 ** 17:.3f} of 2^-17", flush=True)
    assert rel.abs().max() <= 2 * off and abs(rel.mean().item()) <= 2.0 ** -21


def test_gated_in_a_graph():
    case("gated products with their gradients captured, replayed between eager work")
    x, w, dy = randn(gen(1), 40, 512, dtype=BF), randn(gen(2), 256, 512, dtype=BF, scale=0.05), randn(gen(3), 40, 128, dtype=BF)

    def go():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = train.gated_linear(a, b)
        return (y.detach(), *torch.autograd.grad(y, (a, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = go()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        x.copy_(randn(gen(90 + k), 40, 512))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, go())), k


def test_gated_refuses_second_and_forward_derivatives():
    case("gated: derivatives of derivatives, tangents")
    x, w = randn(gen(1), 4, 64, dtype=BF).requires_grad_(True), randn(gen(2), 16, 64, dtype=BF)
    y = train.gated_linear(x, w)
    v = torch.ones_like(y).requires_grad_(True)
    dx, = torch.autograd.grad((v * y).float().sum(), x, create_graph=True)
    for to in (x, v):
        with pytest.raises(RuntimeError, match="gated_linear: gradients of its gradients"):
            torch.autograd.grad(dx.float().sum() + v.float().sum(), to, retain_graph=True)
    fa = torch.autograd.forward_ad
    y = train.gated_linear(x, w)
    with fa.dual_level():
        with pytest.raises(NotImplementedError, match="gated_linear: forward-mode"):
            torch.autograd.grad(y, x, fa.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("F", [1, 3, 4, 8, 37, 505, 512])
def test_padding_columns_of_gated_dz_are_zeros(F):
    """rwkv_gated_dact writes every column from 2F to its pitch, and nothing behind the last row."""
    case(f"gated dact {F} columns, every pitch")
    M = 37
    dy, kept = randn(gen(F), M, F, dtype=BF), randn(gen(F + 1), M, 2 * F, dtype=BF)
    rem = torch.zeros(M, 2 * F, device=DEV, dtype=torch.uint8)
    want = torch.cat([2 * kept[:, :F].clamp(min=0) * kept[:, F:].float() * dy.float(), kept[:, :F].float().clamp(min=0) ** 2 * dy], 1)
    for ldz in range(2 * F, 2 * F + 8):
        dz = torch.full((M + 1, ldz), float("nan"), device=DEV, dtype=BF)
        _lib.check(_lib.lib().rwkv_gated_dact(dy.data_ptr(), F, kept.data_ptr(), rem.data_ptr(), 0, dz.data_ptr(), ldz, _lib.BF16, M, F,
                                              torch.cuda.current_stream().cuda_stream))
        assert not dz[:M, 2 * F:].any() and torch.isnan(dz[M]).all(), ldz
        assert ((dz[:M, :2 * F].double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs()).all(), ldz


@pytest.mark.parametrize("M", [1, 16, 200])
@pytest.mark.parametrize("act", GATES)
def test_pre_activations_past_the_type(act, M):
    """fp16: pre-activations of 98304 (the type ends at 65504) under a gate that
    leaves the result and both gradients inside it; the other rows are zeros.
    Every z has a few bits, so what is kept of it is exact; from |zg| = 100 on
    act and its slope are 0, 1 or powers of z.  dz is rounded once."""
    case(f"gated: large pre-activations {act}, {M} rows")
    K, F, big = 8, 12, 98304.0
    x, w = torch.zeros(M, K, device=DEV, dtype=HF), torch.zeros(2 * F, K, device=DEV, dtype=HF)
    w[:F, 0], w[F:, 1] = 2.0, 2.0
    dy = torch.zeros(M, F, device=DEV, dtype=HF)
    dy[0] = 2.0 ** -6
    seen = 0
    for g, u in ((-2.0, big), (-20.0, big), (-20.0, -big), (0.0, big), (0.0, -big), (-big, 2.0), (-big, big), (-big, -big), (big, 2.0 ** -7), (big, 0.0)):
        x[0, 0], x[0, 1] = g / 2, u / 2
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = train.gated_linear(a, b, act)
        dx, dw = torch.autograd.grad(y, (a, b), dy)
        z = torch.tensor(g, dtype=torch.float64)
        v, d, _ = act64(act, z)
        far = abs(g) > 100
        ev, ed = (E24 * v.abs(), E24 * d.abs()) if far else (act_off(act, z, 0.0), slope_off(act, z, 0.0))
        half = 2.0 ** -11
        dz = [t.item() for t in (2.0 ** -6 * u * d, 2.0 ** -6 * v)]
        off = [t.item() for t in (2.0 ** -6 * abs(u) * ed, 2.0 ** -6 * ev)]
        off = [half * (abs(t) + o) + o + TINY[HF] for t, o in zip(dz, off)]
        row = lambda t: torch.tensor(t, dtype=torch.float64, device=DEV)  # noqa: E731
        if abs(u * v) < 6e4:
            check(f"{g} {u} y", y.detach()[0, :1], row([u * v.item()]), row([abs(u) * ev.item()]))
        for k in range(2):
            # An infinity by right: of dx, or of the other factor's dz, which is rounded to
            # fp16 too (relu², zg = 98304: dzu = 2^-6·98304² = 1.5e8) and meets W's zeros in dx.
            if abs(24 * dz[k]) >= 6e4 or abs(dz[1 - k]) >= 6e4:
                continue
            seen += 1
            check(f"{g} {u} dx{k}", dx[0, k:k + 1], row([24 * dz[k]]), row([24 * off[k]]))
            rows, other = dw[k * F:(k + 1) * F], 1 - k
            for c, at in ((k, (g, u)[k] / 2), (other, (g, u)[other] / 2)):
                if abs(dz[k] * at) < 6e4:
                    check(f"{g} {u} dw{k}{c}", rows[:, c], row([dz[k] * at] * F), row([off[k] * abs(at)] * F))
            assert not rows[:, 2:].any() and not dx[1:].any()
    assert seen >= 14


def test_what_is_kept_of_fp16_pre_activations():
    """The upper 24 bits of the fp32 value, rounded to nearest: within 2^-16 of
    it (half a step of 2^-15), past fp16's range as inside it; both kernels."""
    case("kept bits of fp16")
    L, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for M, F, K in ((4, 512, 8), (300, 512, 8), (200, 300, 8192)):
        x, w = randn(gen(1), M, K, dtype=HF, scale=400.0), randn(gen(2), 2 * F, K, dtype=HF, scale=400.0 * K ** -0.5)
        h, aux = torch.empty(M, F, device=DEV, dtype=HF), torch.empty(M, 2 * F, device=DEV, dtype=torch.int16)
        rem = torch.empty(M, 2 * F, device=DEV, dtype=torch.int8)
        ws = torch.empty(max(L.rwkv_gated_fwd_workspace(M, F, K), 16), dtype=torch.uint8, device=DEV)
        _lib.check(L.rwkv_gated_fwd(x.data_ptr(), K, w.data_ptr(), K, h.data_ptr(), aux.data_ptr(), rem.data_ptr(), 1, _lib.F16, M, F, K,
                                    ws.data_ptr(), ws.numel(), s))
        kept = (aux.int() * 65536 + rem.int() * 256).view(torch.float32).double()
        z, ez = x.double() @ w.double().t(), E24 * (K + 32) * (x.double().abs() @ w.double().abs().t())
        assert (z.abs() > 65520).float().mean() > 0.2
        w_ = ((kept - z).abs() / (2.0 ** -16 * (z.abs() + ez) + ez)).nan_to_num(nan=float("inf")).max().item()
        print(f"  {M} x {F} x {K}: worst error {w_:.3f} of its bound", flush=True)
        assert w_ <= 1.0


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gates_far_below_zero_pass_nothing(act):
    """act(z) = z·σ(..) of a z far below zero is under 2^-100 however large z is:
    dzu = dy·act(zg) and with it dx are zeros."""
    case(f"gated: {act} far below zero")
    for z in (-101.0, -2.0 ** 60, -2.0 ** 126):
        x, w = torch.zeros(2, 8, device=DEV, dtype=BF), torch.zeros(2, 8, device=DEV, dtype=BF)
        x[:, 0], w[0, 0], x[:, 1], w[1, 1] = z, 1.0, 1.0, 1.0
        a = x.requires_grad_(True)
        y = train.gated_linear(a, w, act)
        dx, = torch.autograd.grad(y, a, torch.ones_like(y))
        assert (y.double().abs() <= 2.0 ** -100).all() and (dx.double().abs() <= 2.0 ** -100).all(), (z, y, dx)


FEW = [(1, 2050, 65530), (1, 2064, 32768), (2, 2050, 32760), (16, 45, 40), (16, 517, 513), (7, 99, 1027), (1, 33, 2056), (16, 2101, 4096),
       (10, 2053, 5000), (7, 2059, 7280), (5, 2099, 13099), (16, 300, 8), (3, 5, 7), (1, 4096, 1024), (13, 8200, 1031), (2, 4100, 2055)]


def gate_of_whole_numbers(zg, zu, dt):
    r = zg.clamp(min=0)
    return ((r * r) * zu).to(dt)   # two fp32 products, as the kernel takes them, and the rounding


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,F,K", FEW)
def test_few_rows_are_two_products(M, F, K, dt):
    """The kernel of up to sixteen rows, exactly.  First, each z is one value of
    x: rows of W are zero but for one column, among them the last one, those of
    the last chunk of 8, of the last 64 and of the last 512."""
    case(f"gated columns, few rows: {M} x {F} x {K} {dt}")
    x = torch.randint(-8, 9, (M, K), generator=gen(1), device=DEV).to(dt)
    at = torch.randint(0, K, (2 * F,), generator=gen(2), device=DEV)
    for part, size in enumerate((1, 8, 64, 512)):
        lo = max(0, (K - 1) // size * size)
        some = torch.arange(part, 2 * F, 8, device=DEV)
        at[some] = lo + torch.arange(some.numel(), device=DEV) % (K - lo)
    w = torch.zeros(2 * F, K, device=DEV, dtype=dt)
    w[torch.arange(2 * F, device=DEV), at] = 1.0
    y = train.gated_linear(x, w, "relu2")
    assert torch.equal(y, gate_of_whole_numbers(x[:, at[:F]].float(), x[:, at[F:]].float(), dt))


@pytest.mark.parametrize("M,F,K", FEW + [(17, 300, 4096), (40, 100, 16384), (100, 96, 8200), (200, 300, 8192), (700, 3000, 8192), (129, 70, 4099)])
def test_every_value_of_k_counts(M, F, K):
    """Whole numbers, whose sums fp32 holds exactly (under 2^24: K·8): a range of K
    that is left out or taken twice changes them.  bf16, whose range the products
    stay in; every row and column depends on every k, as nothing is zero."""
    case(f"gated whole numbers: {M} x {F} x {K}")
    assert 8 * K < 2 ** 24
    sign = lambda *s, seed: torch.randint(0, 2, s, generator=gen(seed), device=DEV) * 2 - 1  # noqa: E731
    x = (torch.randint(1, 9, (M, K), generator=gen(1), device=DEV) * sign(M, K, seed=2)).to(BF)
    w = sign(2 * F, K, seed=3).to(BF)
    z = (x.double() @ w.double().t()).float()
    assert z.abs().max() < 2 ** 24
    for f in (lambda: train.gated_linear(x, w, "relu2"), lambda: train.gated_linear(x, w.detach().requires_grad_(True), "relu2").detach()):
        assert torch.equal(f(), gate_of_whole_numbers(z[:, :F], z[:, F:], BF))


@pytest.mark.parametrize("dt", [BF, HF])
def test_saved_tensor_hooks(dt):
    """Hooks that keep floating point tensors in another type leave the kept bits
    of the pre-activations alone, which are no numbers of x's type: with lossless
    hooks (float64) nothing changes, with x and W kept in 8 bits behind the point
    (bfloat16) dx, which reads W, is off by half a step of it, 2^-8, a term."""
    case(f"gated: saved tensor hooks {dt}")
    x, w, dy = randn(gen(1), 40, 96, dtype=dt), randn(gen(2), 128, 96, dtype=dt, scale=0.1), randn(gen(3), 40, 64, dtype=dt)

    def grads(to):
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        pack = lambda t: (t.to(to), t.dtype) if to and t.is_floating_point() else (t, t.dtype)  # noqa: E731
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda p: p[0].to(p[1])):
            y = train.gated_linear(a, b)
        return torch.autograd.grad(y, (a, b), dy)

    want, same, low = grads(None), grads(torch.float64), grads(torch.bfloat16)
    assert all(torch.equal(p, q) for p, q in zip(want, same))
    X, W, DY = x.double(), w.double(), dy.double()
    zg, zu = (X @ W.t()).chunk(2, 1)
    v, d, _ = act64("silu", zg)
    dz = torch.cat([DY * zu * d, DY * v], 1).abs()
    for p, q, terms in ((want[0], low[0], dz @ W.abs()), (want[1], low[1], dz.t() @ X.abs())):
        # each side rounds its result too; 2^-7 of the terms holds the operand's half step and theirs
        assert ((p.double() - q.double()).abs() <= 2.0 ** -7 * terms + 2.0 ** -24).all()
