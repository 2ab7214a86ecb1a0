"""What the attention half of a decoder layer refuses, on the CPU: the C ABI on the host before any
launch, the Python functions before the C ABI, the differentiable forms and the paged cache."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from hybridagent_amd import _lib, attention, training

NULL, FAKE, ODD = None, ctypes.c_void_p(4096), ctypes.c_void_p(4104)  # never dereferenced
OK, ERR_NULL, SHAPE, ALIGN, WORKSPACE = 0, 1, 2, 4, 5
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libw4a16moe.so not built")
    return _lib.load()


def _norm(lib, **kw):
    a = dict(q=FAKE, qt=256, qh=64, k=FAKE, kt=128, kh=64, v=FAKE, vt=128, vh=64, cos=FAKE, sin=FAKE, pos=FAKE,
             qw=FAKE, kw=FAKE, yq=FAKE, yk=FAKE, yv=FAKE, dtype=0, T=5, Hq=4, Hk=2, D=64, P=100, R=32, eps=1e-6)
    assert set(kw) <= set(a)
    return lib.w4a16_head_norm_rope(*{**a, **kw}.values(), NULL)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), SHAPE), (dict(dtype=-1), SHAPE), (dict(T=-1), SHAPE), (dict(T=1 << 24), SHAPE),
    (dict(Hq=0), SHAPE), (dict(Hk=0), SHAPE), (dict(Hq=1025), SHAPE), (dict(D=60), SHAPE), (dict(D=520), SHAPE),
    (dict(D=0), SHAPE), (dict(R=4), SHAPE), (dict(R=72), SHAPE), (dict(R=-8), SHAPE), (dict(P=0), SHAPE),
    (dict(P=1 << 31), SHAPE), (dict(eps=-1.0), SHAPE), (dict(eps=float("nan")), SHAPE), (dict(qt=-64), SHAPE),
    (dict(kh=BIG), SHAPE), (dict(q=NULL), ERR_NULL), (dict(k=NULL), ERR_NULL), (dict(pos=NULL), ERR_NULL),
    (dict(cos=NULL), ERR_NULL), (dict(kw=NULL), ERR_NULL), (dict(yq=NULL), ERR_NULL), (dict(yv=NULL), ERR_NULL),
    (dict(q=ODD), ALIGN), (dict(qt=260), ALIGN), (dict(vh=68), ALIGN), (dict(cos=ODD), ALIGN), (dict(kw=ODD), ALIGN),
    (dict(yk=ODD), ALIGN), (dict(T=0, q=NULL, k=NULL, v=NULL, pos=NULL, yq=NULL), OK)])
def test_head_norm_rope_host_validation(lib, kw, status):
    assert _norm(lib, **kw) == status


def test_head_norm_rope_backward_host_validation(lib):
    def call(**kw):
        a = dict(dq=FAKE, dk=FAKE, dv=FAKE, q=FAKE, qt=256, qh=64, k=FAKE, kt=128, kh=64, v=FAKE, vt=128, vh=64,
                 cos=FAKE, sin=FAKE, pos=FAKE, qw=FAKE, kw=FAKE, xq=FAKE, xk=FAKE, xv=FAKE, wq=FAKE, wk=FAKE, dtype=0,
                 T=5, Hq=4, Hk=2, D=64, P=100, R=32, eps=1e-6, ws=FAKE, bytes=1 << 30)
        return lib.w4a16_head_norm_rope_backward(*{**a, **kw}.values(), NULL)

    need = lib.w4a16_head_norm_rope_backward_workspace_bytes(5, 4, 2, 64)
    assert need > 0 and need % 16 == 0 and lib.w4a16_head_norm_rope_backward_workspace_bytes(0, 4, 2, 64) == 0
    assert call(bytes=need - 1) == call(ws=NULL) == WORKSPACE
    for name in ("dq", "dv", "xk", "xv", "wq", "wk", "qw", "q"):
        assert call(**{name: NULL}) == ERR_NULL, name
    for name in ("dq", "dk", "xv", "ws", "q"):
        assert call(**{name: ODD}) == ALIGN, name
    assert call(dtype=7) == call(D=520) == call(Hk=0) == SHAPE


def test_append_host_validation(lib):
    def call(**kw):
        a = dict(q=FAKE, qt=256, qh=64, k=FAKE, kt=128, kh=64, v=FAKE, vt=128, vh=64, cos=FAKE, sin=FAKE, pos=FAKE,
                 slots=FAKE, qw=FAKE, kw=FAKE, yq=FAKE, yk=NULL, yv=NULL, kc=FAKE, kp=2 * 16 * 64, vc=FAKE,
                 vp=2 * 16 * 64, dtype=0, norm=1, T=5, Hq=4, Hk=2, D=64, P=100, R=32, pages=9, page=16, eps=1e-6)
        return lib.w4a16_append_kv(*{**a, **kw}.values(), NULL)

    for kw in (dict(dtype=2), dict(page=8), dict(page=24), dict(page=2048), dict(pages=0), dict(pages=1 << 28),
               dict(kp=2 * 16 * 64 - 8), dict(vp=0), dict(D=12), dict(vt=BIG)):
        assert call(**kw) == SHAPE, kw
    for kw in (dict(v=NULL), dict(slots=NULL), dict(yq=NULL), dict(kc=NULL), dict(vc=NULL), dict(yk=FAKE),
               dict(yv=FAKE)):
        assert call(**kw) == ERR_NULL, kw
    for kw in (dict(kc=ODD), dict(vp=2 * 16 * 64 + 4), dict(yk=ODD, yv=FAKE), dict(yq=ODD)):
        assert call(**kw) == ALIGN, kw
    assert call(T=0) == OK


def _attn(lib, back=False, **kw):
    heads = dict(q=FAKE, qt=256, qh=64, k=FAKE, kt=128, kh=64, v=FAKE, vt=128, vh=64)
    sizes = dict(dtype=0, B=2, Tq=50, Tk=60, Hq=4, Hk=2, D=64, scale=0.125, causal=1, window=0)
    if back:
        a = {"dout": FAKE, **heads, "out": FAKE, "lse": FAKE, "cu_q": FAKE, "cu_k": FAKE, "dq": FAKE, "dk": FAKE,
             "dv": FAKE, **sizes, "ws": FAKE, "bytes": 1 << 30}
    else:
        a = {**heads, "cu_q": FAKE, "cu_k": FAKE, "out": FAKE, "lse": FAKE, **sizes, "ws": FAKE, "bytes": 1 << 30}
    assert set(kw) <= set(a)
    return (lib.w4a16_attention_backward if back else lib.w4a16_attention)(*{**a, **kw}.values(), NULL)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), SHAPE), (dict(B=-1), SHAPE), (dict(B=(1 << 14) + 1), SHAPE), (dict(Tq=1 << 24), SHAPE),
    (dict(Tk=-1), SHAPE), (dict(Hq=3), SHAPE), (dict(Hk=0), SHAPE), (dict(Hq=2048), SHAPE), (dict(D=96), SHAPE),
    (dict(D=1024), SHAPE), (dict(scale=0.0), SHAPE), (dict(scale=-1.0), SHAPE), (dict(scale=float("inf")), SHAPE),
    (dict(scale=float("nan")), SHAPE), (dict(window=-1), SHAPE), (dict(window=5, causal=0), SHAPE),
    (dict(kt=BIG), SHAPE), (dict(Tq=(1 << 24) - 1, Hq=1024), SHAPE), (dict(Tq=(1 << 24) - 1, Hq=32, D=256), SHAPE), (dict(q=NULL), ERR_NULL), (dict(v=NULL), ERR_NULL),
    (dict(cu_q=NULL), ERR_NULL), (dict(cu_k=NULL), ERR_NULL), (dict(out=NULL), ERR_NULL), (dict(k=ODD), ALIGN),
    (dict(vt=132), ALIGN), (dict(out=ODD), ALIGN)])
def test_attention_host_validation(lib, kw, status, back):
    assert _attn(lib, back, **kw) == status


def test_attention_backward_host_validation(lib):
    need = lib.w4a16_attention_backward_workspace_bytes(2, 50, 60, 4, 2, 64, 0)
    assert need >= 4 * 4 * 50
    for B, Tq, Tk in ((0, 50, 60), (0, 50, 0), (5, 50, 0), (65, 50, 60), (1 << 20, 1, 1)):
        assert lib.w4a16_attention_backward_workspace_bytes(B, Tq, Tk, 4, 2, 128, 0) == 4 * 4 * Tq
        assert lib.w4a16_attention_workspace_bytes(B, Tq, Tk, 4, 2, 128, 0) == 0
    for kw in (dict(dk=NULL), dict(dv=NULL), dict(dout=NULL), dict(lse=NULL)):
        assert _attn(lib, True, **kw) == ERR_NULL, kw
    for kw in (dict(dq=ODD), dict(dv=ODD), dict(ws=ODD), dict(dout=ODD)):
        assert _attn(lib, True, **kw) == ALIGN, kw
    assert _attn(lib, True, bytes=need - 1) == _attn(lib, True, ws=NULL) == WORKSPACE
    # one long sequence of few heads: its workgroups share the sums
    need, sizes = lib.w4a16_attention_workspace_bytes(1, 5000, 5000, 4, 2, 64, 0), dict(B=1, Tq=5000, Tk=5000)
    assert need > 0 and lib.w4a16_attention_workspace_bytes(1, 50000, 50000, 64, 2, 64, 0) == 0
    assert _attn(lib, False, bytes=need - 1, **sizes) == _attn(lib, False, ws=NULL, **sizes) == WORKSPACE
    assert _attn(lib, False, ws=ODD, **sizes) == ALIGN
    assert _attn(lib, False, Tq=0, q=NULL, out=NULL) == OK


def test_decode_host_validation(lib):
    need = lib.w4a16_decode_attention_workspace_bytes(3, 4, 2, 64, 2048)
    assert need > 0 and lib.w4a16_decode_attention_workspace_bytes(3, 4, 2, 64, 128) == 0

    def call(**kw):
        a = dict(q=FAKE, qt=256, qh=64, kc=FAKE, kp=2 * 16 * 64, vc=FAKE, vp=2 * 16 * 64, table=FAKE, lengths=FAKE,
                 out=FAKE, dtype=0, B=3, Hq=4, Hk=2, D=64, pages=9, page=16, width=128, scale=0.125, window=0, ws=FAKE,
                 bytes=need)
        return lib.w4a16_decode_attention(*{**a, **kw}.values(), NULL)

    for kw in (dict(dtype=2), dict(B=-1), dict(B=(1 << 14) + 1), dict(B=BIG), dict(Hq=5), dict(D=80), dict(page=8), dict(page=48),
               dict(pages=0), dict(pages=1 << 28), dict(width=0), dict(width=1 << 28), dict(scale=0.0), dict(window=-1),
               dict(kp=0), dict(vp=2 * 16 * 64 - 8), dict(qt=-8), dict(B=1 << 14, Hq=1024, Hk=1024, width=1 << 20, kp=1024 * 16 * 64, vp=1024 * 16 * 64)):
        assert call(**kw) == SHAPE, kw
    for name in ("q", "kc", "vc", "table", "lengths", "out"):
        assert call(**{name: NULL}) == ERR_NULL, name
    for kw in (dict(q=ODD), dict(kc=ODD), dict(kp=2 * 16 * 64 + 4), dict(out=ODD), dict(ws=ODD), dict(qh=68)):
        assert call(**kw) == ALIGN, kw
    assert call(bytes=need - 1) == call(ws=NULL) == WORKSPACE
    assert call(B=0) == OK
    assert lib.w4a16_decode_attention_workspace_bytes(0, 4, 2, 64, 2048) == 0


# ---------------------------------------------------------------- the Python functions


@pytest.fixture
def no_gpu(monkeypatch):
    """The functions on CPU tensors, up to the launch: it must not be reached."""
    monkeypatch.setattr(_lib, "_gpu_of", lambda *t: 0)

    def launch(what, *args):
        raise AssertionError(f"{what} was launched")
    monkeypatch.setattr(_lib, "_launch", launch)


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _rope(T=5, Hq=4, Hk=2, D=64, dtype=BF):
    i = torch.zeros(T, dtype=torch.int32)
    return dict(q=_z(T, Hq, D, dtype=dtype), k=_z(T, Hk, D, dtype=dtype), v=_z(T, Hk, D, dtype=dtype),
                cos=torch.zeros(9, 16), sin=torch.zeros(9, 16), positions=i, q_weight=_z(D, dtype=dtype),
                k_weight=_z(D, dtype=dtype))


ROPE_WRONG = [dict(q=_z(5, 4, 64, dtype=torch.float64)), dict(q=_z(5, 256)), dict(k=_z(4, 2, 64)), dict(k=_z(5, 2, 32)),
              dict(k=_z(5, 2, 64, dtype=HF)), dict(v=_z(5, 3, 64)), dict(v=_z(5, 2, 64, dtype=F32)), dict(cos=None),
              dict(sin=torch.zeros(9, 8)), dict(cos=_z(9, 16)), dict(positions=torch.zeros(5)),
              dict(positions=torch.zeros(5, dtype=torch.int64)), dict(positions=torch.zeros(4, dtype=torch.int32)),
              dict(q_weight=None), dict(k_weight=_z(32)), dict(q_weight=torch.zeros(64))]


@pytest.mark.parametrize("i", range(len(ROPE_WRONG)))
def test_head_norm_rope_arguments(no_gpu, i):
    a = {**_rope(), **ROPE_WRONG[i]}
    with pytest.raises(ValueError):
        _lib.head_norm_rope(**a)
    with pytest.raises(ValueError):
        _lib.append_kv(**a, slots=a["positions"], k_cache=_z(3, 2, 16, 64), v_cache=_z(3, 2, 16, 64))
    with pytest.raises(ValueError):
        _lib.head_norm_rope_backward(_z(5, 4, 64), _z(5, 2, 64), _z(5, 2, 64), **a)


def test_head_norm_rope_backward_arguments(no_gpu):
    a, d = _rope(), (_z(5, 4, 64), _z(5, 2, 64), _z(5, 2, 64))
    for wrong in ((d[1], d[1], d[2]), (d[0], d[0], d[2]), (d[0], d[1], None), (d[0].half(), d[1], d[2])):
        with pytest.raises(ValueError):
            _lib.head_norm_rope_backward(*wrong, **a)
    with pytest.raises(ValueError):
        _lib.head_norm_rope_backward(*d, **{**a, "v": None})


def test_append_arguments(no_gpu):
    a, kc = _rope(), _z(3, 2, 16, 64)
    slots = torch.zeros(5, dtype=torch.int32)
    for wrong in (dict(v=None), dict(slots=slots[:4]), dict(slots=slots.long()), dict(k_cache=_z(3, 4, 16, 64)),
                  dict(k_cache=_z(3, 2, 16, 32)), dict(k_cache=_z(3, 2, 16, 64, dtype=HF)), dict(v_cache=_z(4, 2, 16, 64)),
                  dict(k_cache=_z(3, 16, 2, 64).transpose(1, 2)), dict(k_cache=_z(2, 16, 64)),
                  dict(k_cache=_z(3, 1, 16, 64), v_cache=_z(3, 1, 16, 64))):
        with pytest.raises(ValueError):
            _lib.append_kv(**{**a, "slots": slots, "k_cache": kc, "v_cache": kc.clone(), **wrong})
    with pytest.raises(ValueError):  # there is no cache of fp32
        b = _rope(dtype=F32)
        _lib.append_kv(**b, slots=slots, k_cache=_z(3, 2, 16, 64, dtype=F32), v_cache=_z(3, 2, 16, 64, dtype=F32))


def test_attention_arguments(no_gpu):
    cu = torch.tensor([0, 5], dtype=torch.int32)
    a = dict(q=_z(5, 4, 64), k=_z(5, 2, 64), v=_z(5, 2, 64), cu_q=cu)
    lse = torch.zeros(4, 5)
    for wrong in (dict(q=_z(5, 4, 64, dtype=F32)), dict(q=_z(5, 256)), dict(k=_z(5, 2, 32)), dict(v=_z(5, 2, 64, dtype=HF)),
                  dict(v=_z(5, 1, 64)), dict(k=_z(5, 3, 64), v=_z(5, 3, 64)), dict(k=_z(5, 0, 64), v=_z(5, 0, 64)),
                  dict(q=_z(5, 4, 96), k=_z(5, 2, 96), v=_z(5, 2, 96)), dict(k=_z(6, 2, 64), v=_z(6, 2, 64)),
                  dict(cu_q=cu.long()), dict(cu_q=cu[:0]), dict(cu_q=cu[None]), dict(cu_k=cu[:1]), dict(window=3, causal=False)):
        with pytest.raises(ValueError):
            _lib.attention(**{**a, **wrong})
        with pytest.raises(ValueError):
            _lib.attention_backward(_z(5, 4, 64), out=_z(5, 4, 64), lse=lse, **{**a, **wrong})
    for wrong in (dict(dout=_z(5, 2, 64)), dict(out=_z(5, 4, 64, dtype=HF)), dict(lse=lse.t()), dict(lse=lse.double()),
                  dict(needs=(True,))):
        with pytest.raises(ValueError):
            _lib.attention_backward(**{**a, "dout": _z(5, 4, 64), "out": _z(5, 4, 64), "lse": lse, **wrong})


def test_decode_arguments(no_gpu):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    a = dict(q=_z(3, 4, 64), k_cache=_z(9, 2, 16, 64), v_cache=_z(9, 2, 16, 64), block_table=i(3, 4), lengths=i(3))
    for wrong in (dict(q=_z(3, 4, 64, dtype=F32)), dict(q=_z(3, 3, 64)), dict(q=_z(3, 4, 32)), dict(block_table=i(2, 4)),
                  dict(block_table=i(12)), dict(block_table=i(3, 4).long()), dict(lengths=i(4)), dict(lengths=i(3).long()),
                  dict(v_cache=_z(9, 2, 16, 64, dtype=HF)), dict(k_cache=_z(9, 16, 2, 64).transpose(1, 2))):
        with pytest.raises(ValueError):
            _lib.decode_attention(**{**a, **wrong})


def test_strides_that_a_size_of_one_leaves_open(monkeypatch):
    """A dimension of one has any stride: such tensors go on as dense ones."""
    monkeypatch.setattr(_lib, "_gpu_of", lambda *t: 0)
    got = []
    monkeypatch.setattr(_lib, "_launch", lambda what, index, fn, *args: got.append(args))
    q = _z(1000)[:256].as_strided((1, 4, 64), (3, 64, 1))
    assert q.is_contiguous()
    _lib.attention(q, q, q, torch.tensor([0, 1], dtype=torch.int32))
    assert got[0][1:3] == (256, 64) and got[0][0] % 16 == 0
    kc = _z(5000)[:2048].as_strided((1, 2, 16, 64), (7, 1024, 64, 1))
    _lib.decode_attention(q, kc, kc, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    assert got[1][4] == got[1][6] == 2048
    one = _z(5000)[:1024].as_strided((1, 1, 16, 64), (1024, 5, 64, 1))
    _lib.decode_attention(q, one, one, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


def test_cpu_tensors():
    cu = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        _lib.attention(_z(5, 4, 64), _z(5, 2, 64), _z(5, 2, 64), cu)
    with pytest.raises(RuntimeError, match="GPU only"):
        _lib.head_norm_rope(**_rope())


# ---------------------------------------------------------------- the differentiable forms


@pytest.fixture
def stand_ins(monkeypatch):
    monkeypatch.setattr(_lib, "head_norm_rope", lambda q, k, v, *a: (q.detach() * 1, k.detach() * 1,
                                                                      None if v is None else v.detach() * 1))
    monkeypatch.setattr(_lib, "attention", lambda q, *a, return_lse=False: (q.detach() * 1, torch.zeros(2)) if return_lse
                        else q.detach() * 1)
    monkeypatch.setattr(_lib, "attention_backward", lambda d, q, k, v, *a, needs: tuple(
        torch.ones_like(t) if n else None for t, n in zip((q, k, v), needs)))


def test_forward_mode_derivatives(stand_ins):
    q, w, cu = torch.zeros(5, 2, 64), torch.zeros(64), torch.tensor([0, 5], dtype=torch.int32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for f in (lambda: training.attention(dual, q, q, cu), lambda: training.attention(q, q, dual, cu),
                  lambda: training.head_norm_rope(q, dual, q, None, None, cu),
                  lambda: training.head_norm_rope(q, q, q, forward_ad.make_dual(w, w), w, cu)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                f()


def test_tables_have_no_gradient(stand_ins):
    q, t, cu = torch.zeros(5, 2, 64), torch.zeros(9, 8, requires_grad=True), torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError, match="cos"):
        training.head_norm_rope(q, q, q, t, t.detach(), cu)
    with pytest.raises(ValueError, match="sin"):
        training.head_norm_rope(q.requires_grad_(), q, q, t.detach(), t, cu)
    with torch.no_grad():
        training.head_norm_rope(q, q, q, t, t, cu)


def test_differentiable_once(stand_ins):
    q, cu = torch.zeros(5, 2, 64, requires_grad=True), torch.tensor([0, 5], dtype=torch.int32)
    g, = torch.autograd.grad(training.attention(q, q.detach(), q.detach(), cu).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        g.sum().backward()


@pytest.mark.parametrize("name", ["attention", "head_norm_rope"])
def test_no_pass_of_a_recorded_step_is_captured(stand_ins, monkeypatch, name):
    q, i = torch.zeros(5, 2, 64, requires_grad=True), torch.zeros(5, dtype=torch.int32)
    f = {"attention": lambda: training.attention(q, q, q, i), "head_norm_rope": lambda: training.head_norm_rope(
        q, q, q, None, None, i)[0]}[name]
    y, capturing = f(), [True]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    with pytest.raises(RuntimeError, match="cannot be captured"):
        f()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        y.sum().backward()
    with torch.no_grad():
        f()


# ---------------------------------------------------------------- tables, cache and module


def test_rope_tables():
    cos, sin = attention.rope_tables(131072, 64, 1e6)
    angle = 131071 * 1e6 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert cos.shape == sin.shape == (131072, 32) and cos.dtype == F32
    assert (cos[-1] - angle.cos()).abs().max() < 2 ** -24 and (sin[-1] - angle.sin()).abs().max() < 2 ** -24
    cos, sin = attention.rope_tables(7, 4, frequencies=torch.tensor([0.5, 0.0]))
    assert bool((cos[:, 1] == 1).all()) and not sin[:, 1].any() and abs(float(sin[3, 0]) - 0.9974949866) < 1e-7
    assert attention.rope_tables(7, 0)[0].shape == (7, 0)
    for kw in (dict(columns=3), dict(columns=-2), dict(columns=4, frequencies=torch.ones(3))):
        with pytest.raises(ValueError):
            attention.rope_tables(7, **kw)


def _cache(pages=6, sequences=3, longest=70):
    return attention.PagedKVCache(2, 1, 64, pages, sequences, longest, page_size=16)


def test_cache_pages():
    c = _cache()
    assert c.k.shape == c.v.shape == (2, 6, 1, 16, 64) and c.block_table.shape == (3, 5) and c.free_pages == 6
    pos, slots = c.append({1: 20, 0: 3, 2: 0})
    assert pos.tolist() == [*range(20), 0, 1, 2] and pos.dtype == slots.dtype == torch.int32
    assert c.lengths.tolist() == [3, 20, 0] and c.free_pages == 3
    table = c.block_table
    for (s, n), (at, p) in zip([(1, 20), (0, 3)], [(0, pos[:20]), (20, pos[20:])]):
        for i, j in enumerate(p.tolist()):
            assert int(slots[at + i]) == int(table[s, j // 16]) * 16 + j % 16
    used = [int(x) for x in table.flatten() if x >= 0]
    assert len(set(used)) == len(used) == 3 and bool((table[2] == -1).all())
    pos, slots = c.append({1: 13, 0: 1})
    assert pos.tolist() == [*range(20, 33), 3] and c.lengths.tolist() == [4, 33, 0] and c.free_pages == 2
    assert c.block_table is table and c.rows([0, 1, 2])[0] is table
    rows, lengths = c.rows([1])
    assert rows.tolist() == table[1:2].tolist() and lengths.tolist() == [33]
    c.free(1)
    assert c.free_pages == 5 and c.lengths.tolist() == [4, 0, 0] and bool((table[1] == -1).all()) and c.length(0) == 4
    assert [t.numel() for t in c.append({})] == [0, 0]


def test_cache_refuses_whole():
    c = _cache()
    c.append({0: 40})
    before = c.block_table.clone(), c.lengths.clone(), c.free_pages
    for counts, kind in (({1: 40, 2: 1}, RuntimeError), ({1: 5, 0: 31}, ValueError), ({1: 5, 3: 1}, ValueError),
                         ({1: 5, 2: -1}, ValueError), ({-1: 1}, ValueError)):
        with pytest.raises(kind):
            c.append(counts)
        assert torch.equal(c.block_table, before[0]) and torch.equal(c.lengths, before[1]) and c.free_pages == before[2]
        assert c.length(1) == c.length(2) == 0
    for kw in (dict(pages=0), dict(sequences=0), dict(longest=0)):
        with pytest.raises(ValueError):
            _cache(**kw)
    with pytest.raises(ValueError):
        attention.PagedKVCache(1, 1, 64, 4, 1, 64, page_size=24)
    with pytest.raises(ValueError):
        c.free(3)


def test_module_refuses():
    for heads, kv in ((3, 2), (4, 0)):
        with pytest.raises(ValueError):
            attention.Attention(64, heads, kv, 64)
    m = attention.Attention(64, 4, 2, 64)
    with pytest.raises(ValueError):
        m(_z(1, 5, 64), None, None, None, None)
