"""The training forms on the GPU against their formulas in 64 bits.

Tolerances: a rounding to a type moves a value by at most u = finfo(type).eps / 2 of it
(bf16 2^-8).  Where a result is a sum of products of rounded values, the roundings are
independent, each uniform within its bound b, and the sum of n of them stays within
8 / sqrt(3) * sqrt(sum b^2) (eight standard deviations of the widest such sum); the
result's own rounding adds u of it.  fp32 sums of n terms add (n + 8) 2^-24 of the sum of
magnitudes at most; the kernels' chains are far shorter than n, so sqrt-like constants
are written where they are used."""
import math

import pytest
import torch

from hybridagent_amd import _lib, training

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
S8 = 8.0 / math.sqrt(3.0)
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def U(dt):
    return torch.finfo(dt).eps / 2


def R(dt, v):
    """A rounding of v: u of it; below the smallest normal number values are spaced eps times that
    number, so half a step is u of it (fp16: spacing 2^-24 below 2^-14, half a step 2^-25)."""
    return U(dt) * v.abs().clamp_min(torch.finfo(dt).tiny)


@pytest.fixture(scope="module")
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _normal(g, *shape, std=1.0, mean=0.0, dt=BF):
    return (torch.randn(*shape, generator=g, device=g.device) * std + mean).to(dt)


def _within(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    worst = float((d / tol.clamp_min(1e-300)).max()) if d.numel() else 0.0
    print(f"{what}: worst {worst:.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the tolerance, worst {worst:.2f}"


# ---------------------------------------------------------------- layer norm


def _ln64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    rstd = ((x - mean[..., None]).square().mean(-1) + eps).rsqrt()
    xh = (x - mean[..., None]) * rstd[..., None]
    return xh * w.double() + (0 if b is None else b.double()), mean, rstd, xh


def _ln_back64(dy, xh, w, rstd):
    dy = dy.double()
    g = dy * w.double()
    dx = rstd[..., None] * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).flatten(0, -2).sum(0), dy.flatten(0, -2).sum(0)


# (rows, width): one row and one element, odd widths, either side of each kernel form's width and
# row count, the widest
LN_SHAPES = [(1, 1), (1, 2816), (3, 7), (5, 64), (513, 1001), (511, 2816), (1031, 2816), (640, 3080), (17, 4096),
             (2, 8191), (600, 8192), (515, 40), (2100, 136), (530, 2049)]


@pytest.mark.parametrize("dt", [BF, HF, SF], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,H", LN_SHAPES)
def test_layer_norm(dev, M, H, dt):
    g = _gen(dev, 100 + M + H)
    x = _normal(g, M, H, std=1.5, mean=0.3, dt=dt)
    x[:, ::97] *= 6
    w, b = _normal(g, H, std=0.1, mean=1.0, dt=dt), _normal(g, H, std=0.1, dt=dt)
    dy = _normal(g, M, H, dt=dt)
    eps = 1e-5
    y, mean, rstd = _lib.layer_norm(x, w, b, eps, return_stats=True)
    want, m64, r64, xh = _ln64(x, w, b, eps)
    # statistics: chains of at most 48 adds in a thread and ten across them
    scale = x.double().abs().mean(-1) + m64.abs()
    _within(mean, m64, 60 * E32 * scale + 1e-30, f"mean {M}x{H}")
    dm = 60 * E32 * scale[:, None] + 4 * E32 * x.double().abs()     # of x - mean
    dxh = dm * r64[:, None] + 64 * E32 * xh.abs()
    # the mean of squares: 60 adds, and the deviations' errors, half of it after the root
    dr = r64 * (34 * E32 + (r64 ** 2) * ((x.double() - m64[:, None]).abs() * dm).mean(-1))
    _within(rstd, r64, dr, f"rstd {M}x{H}")
    dxh = dxh + xh.abs() * (dr / r64)[:, None]
    _within(y, want, R(dt, want) + dxh * w.double().abs() + 4 * E32 * (want.abs() + b.double().abs()),
            f"y {M}x{H}")
    assert torch.equal(_lib.layer_norm(x, w, b, eps), y)
    nb = _lib.layer_norm(x, w, None, eps)
    wantn = xh * w.double()
    _within(nb, wantn, R(dt, wantn) + dxh * w.double().abs() + 4 * E32 * wantn.abs(), f"no bias {M}x{H}")

    # backward, on the exact statistics in fp32 (each off by 2^-24 of itself)
    mean, rstd = m64.float(), r64.float()
    dx, dw, db = _lib.layer_norm_backward(dy, x, w, mean, rstd)
    wx, ww, wb = _ln_back64(dy, xh, w, r64)
    d64, g64 = dy.double(), dy.double() * w.double()
    exh = 4 * E32 * (r64[:, None] * (x.double().abs() + m64.abs()[:, None]) + xh.abs())
    s0, s1 = g64.abs().mean(-1, keepdim=True), (g64 * xh).abs().mean(-1, keepdim=True)
    e1 = 66 * E32 * s1 + (g64.abs() * exh).mean(-1, keepdim=True)
    t = r64[:, None] * (4 * E32 * g64.abs() + 66 * E32 * s0 + xh.abs() * e1 + exh * s1) + 8 * E32 * wx.abs() \
        + 8 * E32 * r64[:, None] * (g64.abs() + s0 + xh.abs() * s1)
    _within(dx, wx, R(dt, wx) + t, f"dx {M}x{H}")
    # column sums: a thread's rows, eight wavefronts, 32 partial sums and eight of those
    n = M / 256 + 64
    _within(dw, ww, R(dt, ww) + n * E32 * (d64 * xh).abs().sum(0) + (d64.abs() * exh).sum(0), f"dw {M}x{H}")
    _within(db, wb, R(dt, wb) + n * E32 * d64.abs().sum(0), f"db {M}x{H}")
    again = _lib.layer_norm_backward(dy, x, w, mean, rstd, bias=False)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw) and again[2] is None


def test_layer_norm_rows_do_not_meet(dev):
    """Non-finite rows change their own results alone; constant rows give the bias."""
    g = _gen(dev, 5)
    x, w, b = _normal(g, 700, 2816), _normal(g, 2816, mean=1.0, std=0.1), _normal(g, 2816)
    y = _lib.layer_norm(x, w, b)
    z = x.clone()
    z[3, 5], z[9, 0], z[699, 2815] = float("inf"), float("nan"), float("-inf")
    z[20] = 0.5
    yz = _lib.layer_norm(z, w, b)
    for r in (3, 9, 699):
        assert torch.isnan(yz[r]).all()
    assert torch.equal(yz[20], b)
    keep = torch.ones(700, dtype=torch.bool)
    keep[[3, 9, 20, 699]] = False
    assert torch.equal(yz[keep], y[keep])


@pytest.mark.parametrize("dt", [BF, HF, SF], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,H", [(600, 1544), (600, 1999), (5, 3001)])
def test_layer_norm_other_row_lengths(dev, M, H, dt):
    """Rows that the shapes above leave out: other numbers of elements per thread."""
    test_layer_norm(dev, M, H, dt)


@pytest.mark.parametrize("H,dt", [(2816, BF), (1000, SF), (24, HF)])
def test_layer_norm_layouts(dev, H, dt):
    """Leading shapes, strided rows, rows at any alignment of their type: the same bits."""
    g = _gen(dev, 6)
    big = _normal(g, 3, 5, 2 * H, dt=dt)
    x = big[..., ::2]
    w, b = _normal(g, H, mean=1.0, std=0.1, dt=dt), _normal(g, H, dt=dt)
    y, mean, rstd = _lib.layer_norm(x, w, b, return_stats=True)
    assert y.shape == x.shape and mean.shape == (3, 5)
    assert torch.equal(y, _lib.layer_norm(x.contiguous().reshape(15, H), w, b).reshape(3, 5, H))
    flat = torch.empty(15 * H + 1, dtype=dt, device=dev)
    off = flat[1:].view(15, H).copy_(x.reshape(15, H))     # not 16-byte aligned
    _within(_lib.layer_norm(off, w, b), y.reshape(15, H).double(),
            U(dt) * 2 * y.reshape(15, H).double().abs() + 1e-5, "unaligned rows")
    dy = _normal(g, H, dt=dt).expand(3, 5, H)
    got = _lib.layer_norm_backward(dy, x, w, mean, rstd)
    want = _lib.layer_norm_backward(dy.contiguous(), x.contiguous(), w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_no_rows(dev):
    w = torch.ones(64, dtype=BF, device=dev)
    x = torch.empty(0, 64, dtype=BF, device=dev)
    s = torch.empty(0, device=dev)
    assert _lib.layer_norm(x, w, w).shape == (0, 64)
    dx, dw, db = _lib.layer_norm_backward(x, x, w, s, s)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    gw, dn = torch.ones(96, 64, dtype=BF, device=dev), torch.ones(64, 96, dtype=BF, device=dev)
    y, saved = _lib.gated_mlp(x, gw, gw, dn, return_saved=True)
    assert y.shape == (0, 64)
    dx, *grads = _lib.gated_mlp_backward(x, x, gw, gw, dn, saved)
    assert dx.shape == (0, 64) and not any(t.any() for t in grads)
    p = [w, w, gw[:64], w, gw[:64], w, w, w]
    out, saved = _lib.hybridlink_train(x, *p)
    dh, *grads = _lib.hybridlink_backward(x, x, *p, saved)
    assert out.shape == dh.shape == (0, 64) and not any(t.any() for t in grads)


# ---------------------------------------------------------------- gated MLP

C0, C1 = math.sqrt(2.0 / math.pi), 0.044715


def _gelu64(a):
    """gelu_tanh, its slope and the size of a times its second derivative."""
    t = torch.tanh(C0 * (a + C1 * a ** 3))
    du = C0 * (1 + 3 * C1 * a * a)
    slope = 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * du
    second = (1 - t * t) * du + 0.5 * a * ((1 - t * t) * C0 * 6 * C1 * a - 2 * t * (1 - t * t) * du * du)
    return 0.5 * a * (1 + t), slope, (a * second).abs()


def _mm(a, b):
    return a @ b


def _mlp64(x, wg, wu, wd, dy=None):
    """Results and tolerances of the block and its gradients."""
    u = U(BF)
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    a, b = x @ wg.t(), x @ wu.t()
    act, slope, curve = _gelu64(a)
    h = act * b
    # fp32: the products' sums, and the activation's exponential and division (2^-20 of |a|)
    f = lambda p, q: 64 * E32 * (p.abs() @ q.abs())
    ea, eb = f(x, wg.t()), f(x, wu.t())
    eh = slope.abs() * b.abs() * ea + act.abs() * eb + 2.0 ** -20 * a.abs() * b.abs()
    y = h @ wd.t()
    ty = u * y.abs() + S8 * (((u * h.abs()) ** 2) @ (wd.t() ** 2)).sqrt() + f(h, wd.t()) + eh @ wd.t().abs()
    out = {"y": (y, ty)}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ wd
    edh = f(dy, wd)
    da, db = dh * b * slope, dh * act
    ra = dh.abs() * (u * (b * slope).abs() + u * curve * b.abs()) + u * da.abs()      # roundings
    rb = dh.abs() * u * (a * slope).abs() + u * db.abs()
    fa = edh * (b * slope).abs() + dh.abs() * 2.0 ** -20 * (1 + a.abs()) * b.abs()    # fp32
    fb = edh * act.abs() + dh.abs() * 2.0 ** -20 * a.abs()
    dx = da @ wg + db @ wu
    tx = u * dx.abs() + S8 * ((ra ** 2) @ (wg ** 2) + (rb ** 2) @ (wu ** 2) + 2 * (ra * rb) @ (wg * wu).abs()).sqrt() \
        + f(da, wg) + f(db, wu) + fa @ wg.abs() + fb @ wu.abs()
    out["dx"] = (dx, tx)
    for name, p, r, e in (("dgate", da, ra, fa), ("dup", db, rb, fb)):
        g = p.t() @ x
        out[name] = (g, u * g.abs() + S8 * ((r.t() ** 2) @ (x ** 2)).sqrt() + f(p.t(), x) + e.t() @ x.abs())
    g = dy.t() @ h
    out["ddown"] = (g, u * g.abs() + S8 * ((dy.t() ** 2) @ ((u * h) ** 2)).sqrt() + f(dy.t(), h) + dy.t().abs() @ eh)
    return out


def _mlp_inputs(dev, T, H, I, seed):
    g = _gen(dev, seed)
    return (_normal(g, T, H), _normal(g, I, H, std=H ** -0.5), _normal(g, I, H, std=H ** -0.5),
            _normal(g, H, I, std=I ** -0.5), _normal(g, T, H, std=0.1))


# (rows, H, I): one token to some thousands, the smallest widths, widths and rows that leave a rest in
# every tile, and the model's shape
MLP_SHAPES = [(1, 32, 32), (1, 2816, 2112), (2, 64, 32), (7, 2816, 2112), (16, 512, 192), (17, 96, 160), (31, 2816, 704),
              (33, 160, 2816), (64, 1024, 480), (65, 288, 736), (100, 2816, 2112), (129, 2048, 512), (193, 2816, 2112),
              (257, 544, 1312), (517, 2816, 2112), (1031, 1056, 1088), (2049, 2816, 704), (4097, 320, 96)]


@pytest.mark.parametrize("T,H,I", MLP_SHAPES)
def test_gated_mlp(dev, T, H, I):
    x, wg, wu, wd, dy = _mlp_inputs(dev, T, H, I, 200 + T + H + I)
    want = _mlp64(x, wg, wu, wd, dy)
    y = _lib.gated_mlp(x, wg, wu, wd)
    _within(y, *want["y"], f"y {T}x{H}x{I}")
    y2, saved = _lib.gated_mlp(x, wg, wu, wd, return_saved=True)
    assert torch.equal(y2, y)
    grads = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved)
    for name, got in zip(("dx", "dgate", "dup", "ddown"), grads):
        _within(got, *want[name], f"{name} {T}x{H}x{I}")
    again = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_gated_mlp_large_values(dev):
    """Gates far from zero, where the activation is 0 or the identity, and a gate of zero."""
    T, H, I = 40, 64, 64
    x, wg, wu, wd, dy = _mlp_inputs(dev, T, H, I, 9)
    for s in (0.0, 1e-3, 30.0, 1e4):
        w = (wg.float() * s).to(BF)
        want = _mlp64(x, w, wu, wd, dy)
        y, saved = _lib.gated_mlp(x, w, wu, wd, return_saved=True)
        got = (y, *_lib.gated_mlp_backward(dy, x, w, wu, wd, saved))
        for (name, (v, t)), q in zip(want.items(), got):
            _within(q, v, t + 1e-30, f"{name} gate x {s}")


def test_gated_mlp_rows_do_not_meet(dev):
    """A non-finite row leaves the other rows' results as they were."""
    for T in (5, 300):
        x, wg, wu, wd, dy = _mlp_inputs(dev, T, 320, 224, 10 + T)
        y, saved = _lib.gated_mlp(x, wg, wu, wd, return_saved=True)
        dx = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved)[0]
        z = x.clone()
        z[2, 7], z[T - 1] = float("nan"), float("inf")
        yz, sz = _lib.gated_mlp(z, wg, wu, wd, return_saved=True)
        dz, *grads = _lib.gated_mlp_backward(dy, z, wg, wu, wd, sz)
        keep = torch.ones(T, dtype=torch.bool)
        keep[[2, T - 1]] = False
        assert torch.equal(yz[keep], y[keep]) and torch.equal(dz[keep], dx[keep])
        assert torch.isnan(yz[2]).all() and torch.isnan(dz[2]).all()
        assert torch.isnan(grads[0][:, 7]).all()


@pytest.mark.parametrize("T", [3, 260])
def test_gated_mlp_some_gradients(dev, T):
    x, wg, wu, wd, dy = _mlp_inputs(dev, T, 256, 160, 11)
    _, saved = _lib.gated_mlp(x, wg, wu, wd, return_saved=True)
    full = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved)
    for needs in ((True, False, False, False), (False, True, False, False), (False, False, True, True),
                  (False, False, False, True), (False,) * 4):
        got = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved, needs=needs)
        for n, p, q in zip(needs, got, full):
            assert (p is None) != n
            if n:  # (a product may be split otherwise when fewer run together)
                _within(p, q.double(), 2 * U(BF) * q.double().abs() + 1e-6 * q.double().abs().max(), f"needs {needs}")


def test_gradients_against_differences(dev):
    """The gradients along a direction against differences of the formulas in 64 bits."""
    T, H, I = 24, 64, 96
    x, wg, wu, wd, dy = _mlp_inputs(dev, T, H, I, 12)
    _, saved = _lib.gated_mlp(x, wg, wu, wd, return_saved=True)
    grads = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved)
    args = [t.double() for t in (x, wg, wu, wd)]
    f = lambda *a: ((_gelu64(a[0] @ a[1].t())[0] * (a[0] @ a[2].t())) @ a[3].t() * dy.double()).sum()
    tols = _mlp64(x, wg, wu, wd, dy)
    for i, (got, name) in enumerate(zip(grads, ("dx", "dgate", "dup", "ddown"))):
        v = torch.randn(args[i].shape, generator=_gen(dev, 13 + i), device=dev, dtype=torch.float64)
        step = 1e-5
        at = lambda s: f(*[t + s * v if j == i else t for j, t in enumerate(args)])
        diff = (at(step) - at(-step)) / (2 * step)
        tol = S8 / 8 * 8 * (tols[name][1] * v).square().sum().sqrt() + 1e-6 * diff.abs()
        _within((got.double() * v).sum()[None], diff[None], tol[None], f"difference {name}")


# ---------------------------------------------------------------- HybridLink


def _link_inputs(dev, T, H, seed):
    g = _gen(dev, seed)
    std = H ** -0.5
    return (_normal(g, T, H, std=1.2, mean=0.1),
            [_normal(g, H, std=0.05, mean=1.0), _normal(g, H, std=0.02), _normal(g, H, H, std=std),
             _normal(g, H, std=0.02), _normal(g, H, H, std=std), _normal(g, H, std=0.02),
             _normal(g, H, std=0.05, mean=1.0), _normal(g, H, std=0.02)], _normal(g, T, H, std=0.1))


def _link64(h, params, dout, eps=1e-5):
    F = torch.nn.functional
    h, *p = [t.double().requires_grad_() for t in (h, *params)]
    n = (h.shape[-1],)
    r = h + F.linear(F.gelu(F.linear(F.layer_norm(h, n, p[0], p[1], eps), p[2], p[3])), p[4], p[5])
    y = F.layer_norm(r, n, p[6], p[7], eps)
    return y.detach(), torch.autograd.grad(y, (h, *p), dout.double())


@pytest.mark.parametrize("T,H", [(1, 32), (1, 2816), (5, 64), (32, 2816), (33, 96), (65, 800), (300, 2816), (1025, 544),
                                 (2049, 1056)])
def test_hybridlink_training(dev, T, H):
    """In the Frobenius norm: each rounded tensor on a result's way (a, z's gradient slope, g, r, dr, dz,
    da and the result: eight at most) carries at most u of its size, and each map on the way has
    about unit gain on such noise, so a result is off by at most 8 u; a chain of fewer by as many."""
    u = U(BF)
    h, params, dout = _link_inputs(dev, T, H, 300 + T + H)
    want, grads = _link64(h, params, dout)
    out, saved = _lib.hybridlink_train(h, *params)
    got = _lib.hybridlink_backward(dout, h, *params, saved)
    rel = lambda p, q: float((p.double() - q).norm() / q.norm().clamp_min(1e-300))
    e = rel(out, want)
    print(f"out {T}x{H}: {e / u:.2f} u", flush=True)
    assert e <= 4 * u
    for i, (p, q) in enumerate(zip(got, grads)):
        e = rel(p, q)
        print(f"gradient {i} {T}x{H}: {e / u:.2f} u", flush=True)
        assert torch.isfinite(p).all() and e <= 8 * u, i
    out2, saved2 = _lib.hybridlink_train(h, *params)
    assert torch.equal(out2, out)
    assert all(torch.equal(p, q) for p, q in zip(got, _lib.hybridlink_backward(dout, h, *params, saved2)))
    # the inference map rounds a few intermediates more
    assert rel(_lib.hybridlink(h, *params), want) <= 6 * u


@pytest.mark.parametrize("T,H,I", [(3, 4160, 96), (20, 64, 4320), (50, 4160, 96), (50, 64, 4320), (130, 96, 64),
                                   (512, 544, 96), (513, 64, 288)])
def test_gated_mlp_few_rows_of_wide_or_narrow_outputs(dev, T, H, I):
    """More columns than one round of the few-rows workgroups has, and more rows of few columns."""
    test_gated_mlp(dev, T, H, I)


@pytest.mark.parametrize("T,H", [(20, 4160), (50, 4160), (200, 96), (512, 32)])
def test_hybridlink_few_rows_of_wide_or_narrow_outputs(dev, T, H):
    test_hybridlink_training(dev, T, H)


# with the shapes above: every tile of every product and epilogue, and every split's join, on 256 CUs
@pytest.mark.parametrize("T,H,I", [
    (265, 32, 5472), (1574, 5024, 32), (1990, 64, 3616), (2053, 64, 5472), (2160, 5920, 480), (2883, 992, 4320),
    (9592, 1184, 64), (12212, 672, 32), (12840, 768, 864), (13445, 32, 544), (16898, 544, 416), (18069, 96, 768),
    (18484, 352, 192), (19030, 544, 128), (20342, 640, 256)])
def test_gated_mlp_every_tile(dev, T, H, I):
    test_gated_mlp(dev, T, H, I)


@pytest.mark.parametrize("T,H", [
    (1, 4128), (65, 2784), (66, 5408), (66, 5664), (5398, 352), (13124, 960), (16349, 704), (16382, 320), (16402, 480),
    (19737, 288), (19995, 608), (21795, 352), (21846, 416), (21902, 192)])
def test_hybridlink_every_tile(dev, T, H):
    test_hybridlink_training(dev, T, H)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("T", [5, 40, 64, 300, 700])
def test_a_row_that_is_not_finite_stays_alone(dev, T, bad):
    """Widths that end inside a stage: what lies behind a row's end is the next row."""
    H, I, r = 96, 160, 3
    x, wg, wu, wd, dy = _mlp_inputs(dev, T, H, I, 400 + T)
    others = torch.arange(T, device=dev) != r
    x2, dy2 = x.clone(), dy.clone()
    x2[r] = bad
    dy2[r] = bad
    y, saved = _lib.gated_mlp(x, wg, wu, wd, return_saved=True)
    assert torch.equal(_lib.gated_mlp(x2, wg, wu, wd)[others], y[others])
    dx = _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved)[0]
    assert torch.equal(_lib.gated_mlp_backward(dy2, x, wg, wu, wd, saved)[0][others], dx[others])
    wd2 = wd.clone()
    wd2[r] = bad
    y2 = _lib.gated_mlp(x, wg, wu, wd2)
    columns = torch.arange(H, device=dev) != r
    assert torch.equal(y2[:, columns], y[:, columns]) and not torch.isfinite(y2[:, r]).any()


# ---------------------------------------------------------------- as they are used


def test_module_trains_like_the_formula(dev):
    """HybridLink and the gated MLP in a row under autograd: the gradients that reach every leaf,
    against the formula's in 64 bits; a leaf used twice gets both."""
    H, I, T = 96, 160, 50
    torch.manual_seed(3)
    link = training.HybridLink(H, device=dev)
    x, wg, wu, wd, dy = _mlp_inputs(dev, T, H, I, 14)
    nw = _normal(_gen(dev, 15), H, mean=1.0, std=0.05)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd, nw)]
    norm = training.layer_norm(x, nw)
    y = link(x + training.gated_mlp(norm, wg, wu, wd)) + norm
    y.backward(dy)
    p64 = [p.detach().double().requires_grad_() for p in link.parameters()]
    l64 = [t.detach().double().requires_grad_() for t in leaves]
    F = torch.nn.functional
    n64 = F.layer_norm(l64[0], (H,), l64[4], None, 1e-5)
    v = l64[0] + F.linear(F.gelu(F.linear(n64, l64[1]), approximate="tanh") * F.linear(n64, l64[2]), l64[3])
    r = v + F.linear(F.gelu(F.linear(F.layer_norm(v, (H,), p64[0], p64[1], 1e-5), p64[2], p64[3])), p64[4], p64[5])
    y64 = F.layer_norm(r, (H,), p64[6], p64[7], 1e-5) + n64
    y64.backward(dy.double())
    u = U(BF)
    # at most eight roundings in each of the three maps on a gradient's way, and torch's two sums
    for i, (p, q) in enumerate(zip([*leaves, *link.parameters()], [*l64, *p64])):
        e = float((p.grad.double() - q.grad).norm() / q.grad.norm())
        print(f"leaf {i}: {e / u:.2f} u", flush=True)
        assert e <= 18 * u, i
    with torch.no_grad():
        assert torch.equal(link(x), _lib.hybridlink(x, *link.parameters()))


def test_frozen_weights_and_second_derivative(dev):
    x, wg, wu, wd, dy = _mlp_inputs(dev, 9, 64, 96, 16)
    x.requires_grad_()
    y = training.gated_mlp(x, wg, wu, wd)
    (g,) = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    w = torch.ones(64, dtype=BF, device=dev)
    assert not training.layer_norm(x.detach(), w).requires_grad
    wd.requires_grad_()
    training.gated_mlp(x.detach(), wg, wu, wd).backward(dy)
    assert wd.grad is not None and wg.grad is None


def test_refusals(dev):
    x, wg, wu, wd, dy = _mlp_inputs(dev, 9, 64, 96, 17)
    w = torch.ones(64, dtype=BF, device=dev)
    y, saved = _lib.gated_mlp(x, wg, wu, wd, return_saved=True)
    _, mean, rstd = _lib.layer_norm(x, w, return_stats=True)
    bad = [lambda: _lib.layer_norm(x.double(), w), lambda: _lib.layer_norm(x, w.float()),
           lambda: _lib.layer_norm(x, w[:63]), lambda: _lib.layer_norm(x, w, w[:63]),
           lambda: _lib.layer_norm(torch.ones(2, 8200, dtype=BF, device=dev), torch.ones(8200, dtype=BF, device=dev)),
           lambda: _lib.layer_norm_backward(dy[:8], x, w, mean, rstd),
           lambda: _lib.layer_norm_backward(dy.float(), x, w, mean, rstd),
           lambda: _lib.layer_norm_backward(dy, x, w, mean[:8], rstd),
           lambda: _lib.layer_norm_backward(dy, x, w, mean, rstd.double()),
           lambda: _lib.gated_mlp(x.float(), wg, wu, wd), lambda: _lib.gated_mlp(x, wg, wu[:64], wd),
           lambda: _lib.gated_mlp(x, wg, wu, wd.t()), lambda: _lib.gated_mlp(x[:, :48], wg[:, :48], wu[:, :48], wd[:48]),
           lambda: _lib.gated_mlp(x, wg[:80], wu[:80], wd[:, :80]),
           lambda: _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved[:-1]),
           lambda: _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved.view(torch.int16)),
           lambda: _lib.gated_mlp_backward(dy[:, :32], x, wg, wu, wd, saved),
           lambda: _lib.gated_mlp_backward(dy, x, wg, wu, wd, saved, needs=(True,)),
           lambda: _lib.hybridlink_train(x, w, w, wg, w, wg, w, w, w)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    with pytest.raises(RuntimeError, match="GPU only"):
        _lib.gated_mlp_backward(dy.cpu(), x, wg, wu, wd, saved)


def _train_step(x, wg, wu, wd, dy, link, nw):
    n, mean, rstd = _lib.layer_norm(x, nw, return_stats=True)
    y, saved = _lib.gated_mlp(n, wg, wu, wd, return_saved=True)
    out, ls = _lib.hybridlink_train(y, *link)
    dh, *gl = _lib.hybridlink_backward(dy, y, *link, ls)
    dn, *gm = _lib.gated_mlp_backward(dh, n, wg, wu, wd, saved)
    return (out, *gl, *gm, *_lib.layer_norm_backward(dn, x, nw, mean, rstd, bias=False)[:2])


@pytest.mark.parametrize("T", [4, 333])
def test_streams_and_graphs(dev, T):
    """The step on another stream, two at once, and captured: replays on new inputs, with eager
    work between them, give the eager bits."""
    H, I = 288, 160
    link = _link_inputs(dev, 1, H, 20)[1]
    nw = _normal(_gen(dev, 21), H, mean=1.0, std=0.05)
    a, b = _mlp_inputs(dev, T, H, I, 22), _mlp_inputs(dev, T, H, I, 23)
    step = lambda v: _train_step(*v, link, nw)
    same = lambda p, q: all(torch.equal(s, t) for s, t in zip(p, q))
    ra, rb = step(a), step(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            pa = step(a)
        with torch.cuda.stream(s2):
            pb = step(b)
        torch.cuda.synchronize()
        assert same(pa, ra) and same(pb, rb)
    buf = [t.clone() for t in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(buf)
    for v, r in ((b, rb), (a, ra), (b, rb)):
        for p, q in zip(buf, v):
            p.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert same(outs, r)
        assert same(step(a), ra)
        torch.cuda.synchronize()


def test_no_backward_pass_is_recorded_under_capture(dev):
    x, wg, wu, wd, _ = _mlp_inputs(dev, 4, 64, 96, 24)
    wg.requires_grad_()
    ref = _lib.gated_mlp(x, wg, wu, wd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            training.gated_mlp(x, wg, wu, wd)
        with torch.no_grad():
            y = training.gated_mlp(x, wg, wu, wd)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)


def test_offsets_past_32_bits(dev):
    """Rows whose bytes pass 2^32: the last ones against the same rows alone."""
    H, M = 2816, 800_000
    w = torch.ones(H, dtype=BF, device=dev)
    x = torch.zeros(M, H, dtype=BF, device=dev)
    tail = _normal(_gen(dev, 25), 700, H)
    x[-700:] = tail
    y, mean, rstd = _lib.layer_norm(x, w, w, return_stats=True)
    y2, m2, r2 = _lib.layer_norm(tail, w, w, return_stats=True)
    assert torch.equal(y[-700:], y2) and torch.equal(mean[-700:], m2) and torch.equal(rstd[-700:], r2)
    del y
    wg, wd = _normal(_gen(dev, 26), 32, H, std=0.02), _normal(_gen(dev, 27), H, 32, std=0.2)
    y, saved = _lib.gated_mlp(x, wg, wg, wd, return_saved=True)
    want = _mlp64(tail, wg, wg, wd, tail)
    _within(y[-700:], *want["y"], "y of the last rows")
    dx, dg, du, dd = _lib.gated_mlp_backward(x, x, wg, wg, wd, saved)
    _within(dx[-700:], *want["dx"], "dx of the last rows")
    for got, name in ((dg, "dgate"), (du, "dup"), (dd, "ddown")):
        _within(got, *want[name], name)
