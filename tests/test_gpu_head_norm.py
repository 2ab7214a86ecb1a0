"""The heads' norm with the position rotation, its gradients and the form that appends to a paged
cache, against 64 bits (autograd in 64 bits for the gradients)."""
import math

import pytest
import torch

import attention_reference as ref
from hybridagent_amd import _lib

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


def _inputs(T, Hq, Hk, D, R, dtype, P=500, weights=True, v=True):
    q, k = ref.normal(1, T, Hq, D, dtype=dtype, std=2.0), ref.normal(2, T, Hk, D, dtype=dtype, std=0.5)
    v = ref.normal(3, T, Hk, D, dtype=dtype) if v else None
    cos, sin = ref.rope_tables(P, R) if R else (None, None)
    pos = (torch.arange(T, device="cuda") * 37 % P).int()
    w = [ref.normal(4 + i, D, dtype=dtype, std=0.2, mean=1.0) if weights else None for i in range(2)]
    return q, k, v, cos, sin, pos, *w


def _exact(x, w, cos, sin, pos, norm=True):
    """(y, its magnitude before cancellation) of rows x in 64 bits."""
    u = x
    if norm:
        u = u * (u.square().mean(-1, keepdim=True) + EPS).rsqrt()
    if w is not None:
        u = u * w
    if cos is None:
        return u, u.detach().abs()
    c, s = (t.double()[pos.long()][:, None] for t in (cos, sin))
    h = c.shape[-1]
    a, b, rest = u[..., :h], u[..., h:2 * h], u[..., 2 * h:]
    mag = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()], -1).detach()
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1), mag


def _check(q, k, v, cos, sin, pos, qw, kw):
    """fp32: the mean of D squares, its root, three products and a sum: 16 units of the magnitude at
    most beside the roundings; gradients as many of the magnitudes that cancel in them."""
    dt, D = q.dtype, q.shape[2]
    u = ref.half_step(dt)
    e = (16 + D / 8) * ref.F32
    got = _lib.head_norm_rope(q, k, v, cos, sin, pos, qw, kw, EPS)
    dys = [None if t is None else ref.normal(20 + i, *t.shape, dtype=dt, std=0.1) for i, t in enumerate((q, k, v))]
    grads = _lib.head_norm_rope_backward(*dys, q, k, v, cos, sin, pos, qw, kw, EPS)
    for name, x, w, y, dy, dx, dw in zip("qkv", (q, k, v), (qw, kw, None), got, dys, grads, (*grads[3:], None)):
        if x is None:
            assert y is None and dx is None
            continue
        X = x.double().requires_grad_()
        W = None if w is None else w.double().requires_grad_()
        turned = (cos, sin) if name != "v" else (None, None)
        norm = name == "v" or w is not None
        Y, mag = _exact(X, W, *turned, pos, norm)
        ref.check(y, (Y.detach(), u * Y.detach().abs() + e * mag + ref.least(dt)), name)
        gx, *gw = torch.autograd.grad(Y, (X,) if W is None else (X, W), dy.double())
        r = (X.detach().square().mean(-1, keepdim=True) + EPS).rsqrt() if norm else torch.ones(1, device="cuda")
        # |g|: the turned gradient's magnitude; t = g w; dx = r (t - xh mean(t xh))
        g = _exact(dy.double(), None, turned[0], None if turned[1] is None else -turned[1], pos, norm=False)[1]
        t = g if w is None else g * w.double().abs()
        xh = (X.detach() * r).abs()
        mag = r * (t + xh * (t * xh).mean(-1, keepdim=True)) if norm else g
        ref.check(dx, (gx, u * gx.abs() + 4 * e * mag + ref.least(dt)), "d" + name)
        if w is not None:
            many = (g * xh).sum((0, 1))
            # in rows per lane, then lanes, wavefronts and workgroups
            ref.check(dw, (gw[0], u * gw[0].abs() + (4 * e + 64 * ref.F32) * many + ref.least(dt)), f"d{name} weight")
    again = _lib.head_norm_rope_backward(*dys, q, k, v, cos, sin, pos, qw, kw, EPS)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("D,R", [(64, 64), (64, 16), (80, 40), (96, 24), (128, 128), (256, 256), (512, 128), (512, 0),
                                 (8, 8), (504, 504)])
@pytest.mark.parametrize("T", [1, 37])
def test_head_norm_rope(T, D, R, dtype):
    _check(*_inputs(T, 5, 3, D, R, dtype))


@pytest.mark.parametrize("dtype", [BF, FF])
def test_many_tokens(dtype):
    _check(*_inputs(3000, 4, 2, 64, 32, dtype))
    _check(*_inputs(700, 16, 8, 256, 256, dtype))


@pytest.mark.parametrize("weights,v", [(False, True), (True, False), (False, False)])
def test_without_weights_or_values(weights, v):
    _check(*_inputs(19, 4, 2, 128, 64, BF, weights=weights, v=v))


def test_no_tokens():
    args = _inputs(0, 4, 2, 128, 64, BF)
    q, k, v = _lib.head_norm_rope(*args)
    assert q.shape == (0, 4, 128) and k.shape == v.shape == (0, 2, 128)
    grads = _lib.head_norm_rope_backward(q, k, v, *args)
    assert grads[0].shape == (0, 4, 128) and not grads[3].any() and not grads[4].any()


def test_far_positions():
    """Angles of far positions, from tables of 64 bits."""
    q, k, v, _, _, _, qw, kw = _inputs(9, 2, 1, 64, 64, FF)
    P = 131072
    cos, sin = ref.rope_tables(P, 64)
    _check(q, k, v, cos, sin, torch.arange(P - 9, P, device="cuda", dtype=torch.int32), qw, kw)


def test_positions_outside_the_tables():
    q, k, v, cos, sin, pos, qw, kw = _inputs(6, 4, 2, 128, 64, BF)
    want = _lib.head_norm_rope(q, k, v, cos, sin, pos, qw, kw)
    bad = pos.clone()
    bad[1], bad[4] = -1, 500
    got = _lib.head_norm_rope(q, k, v, cos, sin, bad, qw, kw)
    fine = [0, 2, 3, 5]
    for a, b in zip(got, want):
        assert torch.equal(a[fine], b[fine])
    assert bool(got[0][[1, 4]].isnan().all()) and bool(got[1][[1, 4]].isnan().all()) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,R,page", [(64, 64, 16), (96, 24, 32), (256, 256, 64), (512, 128, 1024)])
@pytest.mark.parametrize("v_norm", [False, True])
def test_append(D, R, page, dtype, v_norm):
    """The same rows as head_norm_rope's, at their slots; nothing else of the cache is touched."""
    T, Hq, Hk = 53, 6, 3
    q, k, v, cos, sin, pos, qw, kw = _inputs(T, Hq, Hk, D, R, dtype)
    pages = -(-3 * T // page) + 1
    slots = torch.randperm(pages * page, device="cuda")[:T].int()
    slots[7], slots[20], slots[21] = -1, pages * page, 2 ** 31 - 1
    caches = [ref.normal(30 + i, pages, Hk, page, D, dtype=dtype) for i in range(2)]
    want = [t.transpose(1, 2).flatten(0, 1).clone() for t in caches]
    yq, yk, yv = _lib.head_norm_rope(q, k, v, cos, sin, pos, qw, kw, EPS)
    got = _lib.append_kv(q, k, v, cos, sin, pos, slots, *caches, qw, kw, EPS, v_norm=v_norm)
    kept = [i for i in range(T) if i not in (7, 20, 21)]
    at = slots.long()[kept]
    want[0][at] = yk[kept]
    want[1][at] = yv[kept] if v_norm else v[kept]
    assert torch.equal(got, yq)
    for t, w in zip(caches, want):
        assert torch.equal(t.transpose(1, 2).flatten(0, 1), w)


def test_strides():
    """Heads of one projection [T, all columns], tokens apart, heads before tokens, an odd address."""
    T, Hq, Hk, D = 21, 4, 2, 64
    q, k, v, cos, sin, pos, qw, kw = _inputs(T, Hq, Hk, D, 32, BF)
    want = _lib.head_norm_rope(q, k, v, cos, sin, pos, qw, kw)
    both = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    wide = torch.zeros(2 * T, Hq, D, device="cuda", dtype=BF)
    wide[::2] = q
    odd = torch.zeros(T * Hk * D + 1, device="cuda", dtype=BF)[1:].view(T, Hk, D)
    odd.copy_(k)
    parts = [t.unflatten(1, (-1, D)) for t in both.split([Hq * D, Hk * D, Hk * D], 1)]
    for args in (parts, (wide[::2], k.transpose(0, 1).contiguous().transpose(0, 1), v), (q, odd, v)):
        got = _lib.head_norm_rope(*args, cos, sin, pos, qw, kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert math.isfinite(float(want[0].float().sum()))


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,R", [(64, 16), (96, 24), (512, 128), (512, 0), (8, 0)])
def test_columns_behind_the_turned_ones(D, R, bad, dtype):
    """A column that is not finite reaches its norm and its turned partner, no column beside it."""
    q, k, v, cos, sin, pos, _, _ = _inputs(7, 3, 2, D, R, dtype, weights=False)
    want = _lib.head_norm_rope(q, k, v, cos, sin, pos)
    dys = [ref.normal(20 + i, *t.shape, dtype=dtype) for i, t in enumerate((q, k, v))]
    back = _lib.head_norm_rope_backward(*dys, q, k, v, cos, sin, pos)
    for at in sorted({R, R + 3, R + 4, D - 1}):
        x, d = [t.clone() for t in (q, k)], [t.clone() for t in dys]
        for t in (*x, *d[:2]):
            t[2, 1, at] = bad
        got = _lib.head_norm_rope(*x, v, cos, sin, pos)
        grads = _lib.head_norm_rope_backward(*d, q, k, v, cos, sin, pos)
        for a, b in (*zip(got[:2], want), *zip(grads[:2], back)):
            b = b.clone()
            b[2, 1, at] = bad
            assert torch.equal(a.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0)), at


@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_normed_columns_behind_the_turned_ones(dtype, bad):
    """With weights: infinity over itself is not a number, a finite column over infinity zero; of the weights'
    gradients the column alone."""
    D, R, at = 64, 16, 33
    q, k, v, cos, sin, pos, qw, kw = _inputs(7, 3, 2, D, R, dtype)
    dys = [ref.normal(20 + i, *t.shape, dtype=dtype) for i, t in enumerate((q, k, v))]
    *_, wq, wk = _lib.head_norm_rope_backward(*dys, q, k, v, cos, sin, pos, qw, kw)
    d = [t.clone() for t in dys]
    d[0][2, 1, at] = d[1][2, 1, at] = bad
    *_, gq, gk = _lib.head_norm_rope_backward(*d, q, k, v, cos, sin, pos, qw, kw)
    other = torch.arange(D, device="cuda") != at
    for g, w in ((gq, wq), (gk, wk)):
        assert not g[at].isfinite() and torch.equal(g[other], w[other])
    x = q.clone()
    x[2, 1, at] = bad
    y = _lib.head_norm_rope(x, k, v, cos, sin, pos, qw, kw)[0][2, 1]
    assert bool(y[at].isnan()) and bool((y[other].isnan() if bad != bad else y[other] == 0).all())
