"""The paged cache and the latent stack's calls over it where something fails, on the CPU: the cache is then
as it was before the call."""
import pytest
import torch

from hybridagent_amd import attention, latent

BF = torch.bfloat16


def _cache(pages=6, sequences=3, longest=70):
    return attention.PagedKVCache(2, 1, 64, pages, sequences, longest, page_size=16)


def _state(c):
    return (c.block_table.tolist(), c.lengths.tolist(), [c.length(s) for s in range(len(c.lengths))], list(c._free),
            [list(p) for p in c._pages])


def test_take_back():
    c = _cache()
    c.append({0: 20, 2: 16})
    before = _state(c)
    c.append({1: 17, 0: 13, 2: 0})
    c.take_back({1: 17, 0: 13, 2: 0})
    assert _state(c) == before
    c.take_back({0: 4})
    assert c.length(0) == 16 and c.free_pages == 4 and c.block_table[0].tolist()[1:] == [-1] * 4
    for counts in ({0: 17}, {0: 1, 3: 1}, {2: -1}, {-1: 0}):
        state = _state(c)
        with pytest.raises(ValueError):
            c.take_back(counts)
        assert _state(c) == state
    pos, slots = c.append({0: 2})
    assert pos.tolist() == [16, 17] and slots.tolist() == [16 * c._pages[0][1], 16 * c._pages[0][1] + 1]


def test_append_that_cannot_reach_the_device(monkeypatch):
    c = _cache()
    c.append({0: 20})
    host = [list(c._lengths), list(c._free), [list(p) for p in c._pages]]
    lengths = c.lengths.tolist()

    def copy(*a):
        raise RuntimeError("out of memory")
    monkeypatch.setattr(c, "_copy", copy)
    with pytest.raises(RuntimeError, match="out of memory"):
        c.append({0: 30, 1: 5})
    assert [c._lengths, c._free, c._pages] == host and c.lengths.tolist() == lengths
    monkeypatch.undo()
    pos, _ = c.append({0: 1, 1: 5})
    assert pos.tolist() == [20, 0, 1, 2, 3, 4] and c.lengths.tolist() == [21, 5, 0]


def _stack():
    sizes = latent.AttentionSizes(heads=4, kv_heads=2, head_size=64, longest=128)
    return latent.LatentStack(2, 8, 256, 128, 2, 32, seed=5, device="cpu", tiled=False, attention=sizes)


def test_a_step_that_fails_leaves_the_cache(monkeypatch):
    """The kernels refuse tensors on the CPU, after the cache gave room; then a layer of several."""
    st = _stack()
    c = st.cache(8, 2, page_size=16)
    state = _state(c)
    for _ in range(2):  # the second is no "has tokens already"
        with pytest.raises(RuntimeError, match="GPU only"):
            st.prompt(torch.zeros(20, 256, dtype=BF), c, {0: 17, 1: 3})
        assert _state(c) == state
    monkeypatch.setattr(st, "_attended", lambda h, attend: h)
    st.prompt(torch.zeros(20, 256, dtype=BF), c, {0: 17, 1: 3})
    state = _state(c)
    monkeypatch.undo()
    for call in (st.decode, st.latent):
        with pytest.raises(RuntimeError, match="GPU only"):
            call(torch.zeros(2, 256, dtype=BF), c, [1, 0])
        assert _state(c) == state
    calls = []

    def attended(h, attend):
        calls.append(1)
        raise KeyboardInterrupt
    monkeypatch.setattr(st, "_attended", attended)
    with pytest.raises(KeyboardInterrupt):
        st.decode(torch.zeros(1, 256, dtype=BF), c, [0])
    assert calls == [1] and _state(c) == state


@pytest.mark.parametrize("wrong", [dict(dtype=torch.float32), dict(dtype=torch.float16), dict(device="meta")])
def test_residuals_of_another_kind(wrong):
    st = _stack()
    c = st.cache(8, 2, page_size=16)
    for call in (lambda: st.prompt(torch.zeros(3, 256, **{"dtype": BF, **wrong}), c, {0: 3}),
                 lambda: st.decode(torch.zeros(1, 256, **{"dtype": BF, **wrong}), c, [0])):
        with pytest.raises(ValueError, match="bfloat16"):
            call()
        assert c.length(0) == 0 and c.free_pages == 8


@pytest.mark.parametrize("which", [[-1], [3], [0, 3], [1, -4]])
def test_rows_of_no_sequence(which):
    c = _cache()
    c.append({0: 3, 2: 5})
    with pytest.raises(ValueError, match="no sequence"):
        c.rows(which)
    for s in which:
        if not 0 <= s < 3:
            with pytest.raises(ValueError, match="no sequence"):
                c.length(s)
    assert c.rows([2, 0])[1].tolist() == [5, 3]


def test_rope_tables_of_frequencies_elsewhere():
    """Without a device the tables are where the frequencies are."""
    f = torch.ones(4, device="meta")
    assert all(t.device == f.device and t.shape == (7, 4) for t in attention.rope_tables(7, 8, frequencies=f))
    assert attention.rope_tables(7, 8, frequencies=torch.ones(4))[0].device.type == "cpu"
    assert attention.rope_tables(7, 8, device="cpu", frequencies=torch.ones(4, dtype=torch.float64))[1].shape == (7, 4)
