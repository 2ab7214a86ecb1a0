"""Attention at the ends of its numbers' ranges: scores far below zero, infinite keys and values, and
fp16 where weights and slopes lie below its normal numbers; against 64 bits, as test_gpu_attention.py."""
import math
import time

import pytest
import torch

import attention_reference as ref
from hybridagent_amd import _lib
from test_gpu_attention import _cache, _check, _inputs, _split

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def dev():
    assert _lib.available(), "libw4a16moe.so must be built"
    return torch.device("cuda:0")


@pytest.fixture(autouse=True)
def underflow(monkeypatch):
    """The bounds know no end of fp32, and 64 bits keep a weight of e^-200.  fp32's normal numbers end at
    2^-126 and what is below may be zero: a weight is off by 2^-126, and a slope, weight x (dout v - delta)
    with magnitudes below 2^16 here, by 2^-110.  bf16 ends there too."""
    fp16 = ref.least(HF)
    monkeypatch.setattr(ref, "least", lambda dtype: fp16 if dtype == HF else 2.0 ** -110)


# ---------------------------------------------------------------- scores far below zero

# the score of key j beside a few units of noise: all low; the first steps low; falling; low blocks
SHAPES = {
    "all": lambda j, low: torch.full_like(j, low),
    "first": lambda j, low: torch.where(j < 70, low, 4.0),
    "falling": lambda j, low: low / 16 * j.clamp(max=64),
    "blocks": lambda j, low: torch.where(j // 96 % 2 == 0, low, 2.0),
}


def _scored(lens_q, lens_k, Hq, Hk, D, dtype, shape, low):
    """Inputs whose scores, at a scale of one, go by the key's place in its sequence."""
    q, k, v, cu_q, cu_k, dout = _inputs(lens_q, lens_k, Hq, Hk, D, dtype, std=0.1)
    j = torch.cat([torch.arange(n, device="cuda", dtype=torch.float64) for n in lens_k])
    q[..., 0] = 1.0
    k[..., 0] = SHAPES[shape](j, low).to(dtype)[:, None]
    return q, k, v, cu_q, cu_k, dout


@pytest.mark.parametrize("low", [-90.0, -200.0, -1000.0])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_low_scores(D, shape, low):
    lens = [1, 300, 33]
    _check(*_scored(lens, lens, 4, 2, D, BF, shape, low), scale=1.0)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_low_scores_fp16(D):
    lens = [1, 300, 33]
    _check(*_scored(lens, lens, 4, 2, D, HF, "first", -200.0), scale=1.0)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_low_scores_of_many_heads(D, shape):
    """The larger tiles, which many heads take."""
    lens = [300, 33]
    _check(*_scored(lens, lens, 128, 2, D, BF, shape, -200.0), scale=1.0)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_low_scores_of_shared_sums(D, shape):
    """Every part of a tile begins with a maximum of its own."""
    lens = [1500, 3, 900]
    assert _split(lens, lens, 4, 1, D) == (True, True)
    _check(*_scored(lens, lens, 4, 1, D, BF, shape, -200.0), scale=1.0)


@pytest.mark.parametrize("window", [1, 16, 90])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [64, 256, 512])
def test_low_scores_in_windows(D, shape, window):
    lens = [300, 33]
    _check(*_scored(lens, lens, 4, 2, D, BF, shape, -200.0), scale=1.0, window=window)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_low_scores_all_keys_seen(D):
    _check(*_scored([5, 100], [205, 37], 4, 2, D, BF, "first", -200.0), scale=1.0, causal=False)


def _decode_scored(lens, D, dtype, low_of, window=0, width=None, Hq=4, Hk=2, page=16):
    """Decoding with keys whose scores, at a scale of one, are low_of(place, length)."""
    kc, vc, table, lengths, keys, values = _cache(lens, Hk, D, page, dtype, width=width)
    q = ref.normal(1, len(lens), Hq, D, dtype=dtype, std=0.1)
    q[..., 0] = 1.0
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        keys[b][..., 0] = low_of(j.double(), n).to(dtype)[:, None]
        kc[table[b].long()[j // page], :, j % page] = keys[b]
    out = _lib.decode_attention(q, kc, vc, table, lengths, scale=1.0, window=window)
    for b, n in enumerate(lens):
        want = ref.attend(q[b:b + 1], keys[b], values[b], 1.0, True, window, dtype)
        ref.check(out[b:b + 1], want["out"], f"sequence {b} of {n}")


@pytest.mark.parametrize("low", [-90.0, -200.0, -1000.0])
@pytest.mark.parametrize("shape", [*SHAPES, "last"])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_decode_low_scores(D, window, shape, low):
    """Tables on both sides of the width up to which a workgroup has all of a sequence's keys; "last":
    the last key alone is low, in a wavefront of its own where the length is one more than 32."""
    of = (lambda j, n: torch.where(j == n - 1, low, 10.0)) if shape == "last" else lambda j, n: SHAPES[shape](j, low)
    limit = 128 * min(8, 1024 // D)
    for width in (limit // 16, limit // 16 + 1):
        _decode_scored([1, 33, 129, 181, 0, 32], D, BF, of, window=window, width=width)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [64, 512])
def test_decode_low_scores_long(D, shape):
    _decode_scored([9000, 3, 2500], D, HF, lambda j, n: SHAPES[shape](j, -200.0), Hq=8, Hk=1, page=64)


# ---------------------------------------------------------------- scores that are minus infinity


def _without_first(q, k, v, lens, scale, window):
    """Each sequence's queries but the first over its keys but the first, in 64 bits: (rows, bounds)."""
    cu = ref.offsets([n - 1 for n in lens])
    kept = torch.cat([torch.arange(n - 1, device="cuda") + 1 + at for n, at in zip(lens, ref.offsets(lens).tolist())])
    return kept, ref.packed(q[kept], k[kept], v[kept], cu, cu, scale, True, window)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,window", [(4, 0), (4, 1), (4, 40), (128, 0)])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_infinite_key(D, Hq, window, dtype):
    """The first key of a sequence is infinite and every query's score of it minus infinity: the query
    that sees nothing else has no softmax, the others give it no weight."""
    lens = [150, 1, 90]
    q, k, v, cu, _, dout = _inputs(lens, lens, Hq, 2, D, dtype)
    first = cu[:-1].long()
    q[..., 0], k[first, :, 0] = -1.0, math.inf
    out, lse = _lib.attention(q, k, v, cu, window=window, return_lse=True)
    assert bool(out[first].isnan().all()) and bool((lse[:, first] == -math.inf).all())
    kept, want = _without_first(q, k, v, lens, D ** -0.5, window)
    ref.check(out[kept], want["out"], "out")
    ref.check(lse[:, kept], want["lse"], "lse")
    dq, dk, dv = _lib.attention_backward(dout, q, k, v, out, lse, cu, window=window)
    for name, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        assert bool(t[first].isnan().all()), name


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_infinite_keys_of_shared_sums(D, causal):
    """A sequence without one finite score, in parts; the others, and queries without keys, are as they were."""
    lens_q, lens_k = [1500, 30, 900], [1500, 20, 900]
    assert _split(lens_q, lens_k, 4, 1, D) == (True, True)
    q, k, v, cu_q, cu_k, dout = _inputs(lens_q, lens_k, 4, 1, D, BF)
    q[..., 0] = -1.0
    want = ref.packed(q, k, v, cu_q, cu_k, D ** -0.5, causal, 0, dout)
    k[:1500, :, 0] = math.inf
    out, lse = _lib.attention(q, k, v, cu_q, cu_k, causal=causal, return_lse=True)
    assert bool(out[:1500].isnan().all()) and bool((lse[:, :1500] == -math.inf).all())
    grads = _lib.attention_backward(dout, q, k, v, out, lse, cu_q, cu_k, causal=causal)
    for name, t, at in (("out", out, 1500), *zip(("dq", "dk", "dv"), grads, (1500, 1500, 1500))):
        assert bool(t[:at].isnan().all()), name
        ref.check(t[at:], tuple(x[at:] for x in want[name]), name)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_decode_infinite_keys(D, window, dtype):
    """Keys whose scores are minus infinity have no weight: some of a wavefront's, all of one's, all of a
    piece's; a token that sees no others has no softmax.  The finite scores are low: e^-200."""
    lens, spoilt = [1, 33, 181, 300, 0, 9000, 2500], [1, 32, 181, 7, 0, 5000, 2500]
    limit = 128 * min(8, 1024 // D)
    for few, width in ((5, limit // 16), (5, limit // 16 + 1), (7, None)):
        kc, vc, table, lengths, keys, values = _cache(lens[:few], 2, D, 16, dtype, width=width)
        q = ref.normal(1, few, 4, D, dtype=dtype, std=0.1)
        q[..., 0] = -1.0
        for b, n in enumerate(lens[:few]):
            j = torch.arange(n, device="cuda")
            keys[b][..., 0] = torch.where(j < spoilt[b], math.inf, 200.0).to(dtype)[:, None]
            kc[table[b].long()[j // 16], :, j % 16] = keys[b]
        out = _lib.decode_attention(q, kc, vc, table, lengths, scale=1.0, window=window)
        for b, n in enumerate(lens[:few]):
            if n and spoilt[b] == n:
                assert bool(out[b].isnan().all()), n
                continue
            rest = [t[b][spoilt[b]:] for t in (keys, values)]
            want = ref.attend(q[b:b + 1], *rest, 1.0, True, window, dtype)
            ref.check(out[b:b + 1], want["out"], f"sequence {b} of {n}")


# ---------------------------------------------------------------- fp16 below its normal numbers

# fp16's normal numbers end at 2^-14 and all at 2^-24.  The bounds of these tests have every weight and slope
# rounded by half a step of itself (``least`` zero), and the results' last rounding by 2^-25 besides.


@pytest.fixture
def relative(monkeypatch):
    monkeypatch.setattr(ref, "least", lambda dtype: 0.0)


@pytest.mark.parametrize("size", [3e-5, 1e-4, 1e-3, 1.0])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_small_gradients_fp16(relative, D, size):
    """dout of any size: the slopes' smallest are a weight of 1 / 1500 of it."""
    lens = [1500, 40]
    q, k, v, cu, _, dout = _inputs(lens, lens, 2, 1, D, HF)
    dout = (dout.float() * size).half()
    out, lse = _lib.attention(q, k, v, cu, return_lse=True)
    want = ref.packed(q, k, v, cu, cu, D ** -0.5, True, 0, dout)
    for name, t in zip(("dq", "dk", "dv"), _lib.attention_backward(dout, q, k, v, out, lse, cu)):
        ref.check(t, want[name], name, slack=2.0 ** -25)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_large_gradients_fp16(relative, D):
    """Slopes beyond fp16's 65504 whose sums it holds."""
    lens = [70, 9]
    q, k, v, cu, _, dout = _inputs(lens, lens, 4, 2, D, HF, std=0.2)
    k, v, dout = k * 0.2, v * 8.0, dout * 2500.0
    want = ref.packed(q, k, v, cu, cu, D ** -0.5, True, 0, dout)
    assert max(float(want[n][0].abs().max()) for n in ("dq", "dk", "dv")) < 50000
    out, lse = _lib.attention(q, k, v, cu, return_lse=True)
    for name, t in zip(("dq", "dk", "dv"), _lib.attention_backward(dout, q, k, v, out, lse, cu)):
        ref.check(t, want[name], name, slack=2.0 ** -25)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_gradients_of_unequal_rows_fp16(relative, D):
    """Each query's gradient a size of its own, growing and falling along the sequence."""
    lens = [700, 300]
    q, k, v, cu, _, dout = _inputs(lens, lens, 4, 2, D, HF)
    e = torch.cat([torch.linspace(-12, 6, 700, device="cuda"), torch.linspace(6, -12, 300, device="cuda")])
    dout = (dout.float() * 2.0 ** e[:, None, None]).half()
    out, lse = _lib.attention(q, k, v, cu, return_lse=True)
    want = ref.packed(q, k, v, cu, cu, D ** -0.5, True, 0, dout)
    for name, t in zip(("dq", "dk", "dv"), _lib.attention_backward(dout, q, k, v, out, lse, cu)):
        ref.check(t, want[name], name, slack=2.0 ** -25)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_gradient_of_values_of_many_keys_fp16(D):
    """n equal weights: 1 / n is 20.5 of fp16's least steps.  dv is the gradients' sum over n, off by the roundings
    of p and of itself; lse and the exponential add 2^-17 at most (log n is 13.6 and rounded to 2^-20)."""
    n, m = 818400, 33
    q = torch.zeros(m, 1, D, device="cuda", dtype=HF)
    k, v = ref.normal(2, n, 1, D, dtype=HF), ref.normal(3, n, 1, D, dtype=HF)
    dout = ref.normal(4, m, 1, D, dtype=HF, std=5.0, mean=60.0)
    cu_q, cu_k = ref.offsets([m]), ref.offsets([n])
    out, lse = _lib.attention(q, k, v, cu_q, cu_k, causal=False, return_lse=True)
    _, _, dv = _lib.attention_backward(dout, q, k, v, out, lse, cu_q, cu_k, causal=False, needs=(False, False, True))
    want = (dout.double().sum(0) / n)[None]
    off = float(((dv.double() - want) / want).abs().max())
    assert off <= 2 * ref.half_step(HF) + 2.0 ** -17, off


def _faint(n, D):
    """One key with a score of 0 and n with one whose weight is 2^-25: as much as 1/128 together where n is
    2^18.  (key, value, the result's first column): the one key's value is zero, the others' one."""
    k = torch.zeros(n + 1, 1, D, device="cuda", dtype=HF)
    k[1:, 0, 0] = 1.0
    v = torch.ones(n + 1, 1, D, device="cuda", dtype=HF)
    v[0] = 0.0
    return k, v, n * 2.0 ** -25 / (1 + n * 2.0 ** -25)


# the scale: 25 ln 2 is off by 2^-21 in fp32 at most, as are the products with log2 e, and so each weight by
# 2^-19 of itself; their sum of n terms by n 2^-24 in the worst order, in tiles by far less: 2^-10 is allowed
# for all and half a step of the result
FAINT = 2.0 ** -10 + 2.0 ** -11


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_faint_weights_fp16(D):
    n = 1 << 18
    k, v, want = _faint(n, D)
    q = torch.zeros(1, 1, D, device="cuda", dtype=HF)
    q[..., 0] = -1.0
    out = _lib.attention(q, k, v, ref.offsets([1]), ref.offsets([n + 1]), scale=25 * math.log(2.0))
    off = float((out.double() / want - 1).abs().max())
    assert off <= FAINT, off


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_decode_faint_weights_fp16(D):
    """256 sequences of the same pages: a workgroup has all of one, and a wavefront of it the first key."""
    n, page, B = (1 << 16) - 1, 1024, 256
    k, v, want = _faint(n, D)
    kc, vc = (t.view(-1, page, 1, D).transpose(1, 2).contiguous() for t in (k, v))
    q = torch.zeros(B, 1, D, device="cuda", dtype=HF)
    q[..., 0] = -1.0
    table = torch.arange(kc.shape[0], device="cuda", dtype=torch.int32).expand(B, -1)
    out = _lib.decode_attention(q, kc, vc, table, torch.full((B,), n + 1, device="cuda", dtype=torch.int32),
                                scale=25 * math.log(2.0))
    off = float((out.double() / want - 1).abs().max())
    assert off <= FAINT, off


# ---------------------------------------------------------------- values that are not finite, in number


def _sprinkled(v, share, seed=9):
    """v with a share of its elements not finite: the clean v, the spoilt one, where."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    bad = torch.rand(v.shape, generator=g, device="cuda") < share
    kind = torch.randint(0, 3, v.shape, generator=g, device="cuda")
    values = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=v.dtype)[kind]
    return v.masked_fill(bad, 0.0), torch.where(bad, values, v), bad


def _hit(bad, lens_q, lens_k, g, window):
    """Where a query sees such a value: [Tq, Hq, D]."""
    res, k0 = [], 0
    for n, m in zip(lens_q, lens_k):
        seen = ref.seen_keys(n, m, True, window, "cuda").double()
        res.append((seen @ bad[k0:k0 + m].double().flatten(1)).view(n, *bad.shape[1:]) > 0)
        k0 += m
    return torch.cat(res).repeat_interleave(g, 1)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("share", [0.0003, 0.05])
@pytest.mark.parametrize("Hq,window", [(4, 0), (4, 1), (4, 40), (4, 130), (128, 0), (128, 40)])
@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_many_values_that_are_not_finite(D, Hq, window, share, dtype):
    lens_q, lens_k = [400, 33], [350, 90]
    q, k, v, cu_q, cu_k, _ = _inputs(lens_q, lens_k, Hq, 2, D, dtype)
    clean, v, bad = _sprinkled(v, share)
    hit = _hit(bad, lens_q, lens_k, Hq // 2, window)
    want, bound = ref.packed(q, k, clean, cu_q, cu_k, D ** -0.5, True, window)["out"]
    out = _lib.attention(q, k, v, cu_q, cu_k, window=window)
    assert not out[hit].isfinite().any()
    ref.check(out.double().masked_fill(hit, 0.0), (want.masked_fill(hit, 0.0), bound), "out")


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_many_values_that_are_not_finite_in_shared_sums(D):
    lens = [1500, 900]
    assert _split(lens, lens, 4, 2, D)[0]
    q, k, v, cu, _, _ = _inputs(lens, lens, 4, 2, D, BF)
    clean, v, bad = _sprinkled(v, 0.0005)
    hit = _hit(bad, lens, lens, 2, 0)
    want, bound = ref.packed(q, k, clean, cu, cu, D ** -0.5, True, 0)["out"]
    out = _lib.attention(q, k, v, cu)
    assert not out[hit].isfinite().any()
    ref.check(out.double().masked_fill(hit, 0.0), (want.masked_fill(hit, 0.0), bound), "out")


@pytest.mark.parametrize("what", ["first", "all", "last", "one", "sparse"])
@pytest.mark.parametrize("D", [64, 512])
def test_values_that_are_not_finite_take_no_square_time(D, what):
    """One key after the other for every query took 75 to 115 times as long: 30 times is allowed here."""
    n = 8192
    q, k, v, cu, _, _ = _inputs([n], [n], 2, 1, D, HF)
    bad = v.clone()
    at = {"first": slice(0, 1), "all": slice(None), "last": slice(-1, None), "one": slice(5000, 5001),
          "sparse": slice(150, None, 301)}[what]
    bad[at, 0, 7] = math.inf

    def took(v):
        best = math.inf
        for _ in range(3):
            torch.cuda.synchronize()
            start = time.perf_counter()
            _lib.attention(q, k, v, cu)
            torch.cuda.synchronize()
            best = min(best, time.perf_counter() - start)
        return best

    took(v)
    fine, spoilt = took(v), took(bad)
    print(f"{1e6 * fine:.0f} us, {1e6 * spoilt:.0f} us", flush=True)
    assert spoilt < 30 * fine


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_gradients_of_huge_scores_fp16(D):
    """Scores of 10^7, where fp32 leaves a weight of one a factor of 2^2: log2 e times them has a last place
    of 2, and three such roundings of half a place lie between the forward pass' maximum and p.  dv, p dout
    of one key, is that much and no infinity."""
    q = torch.zeros(1, 1, D, device="cuda", dtype=HF)
    q[..., 0] = 3600.0
    for k0 in (2600.0, 2801.0, 3003.0, 3301.0, 3333.0):
        k, v, dout = q * (k0 / 3600.0), torch.ones_like(q), torch.full_like(q, 100.0)
        cu = ref.offsets([1])
        out, lse = _lib.attention(q, k, v, cu, scale=1.0, return_lse=True)
        dv = _lib.attention_backward(dout, q, k, v, out, lse, cu, scale=1.0)[2]
        assert bool((out == 1).all()) and bool(((dv >= 12.5) & (dv <= 800.0)).all()), (k0, dv)
