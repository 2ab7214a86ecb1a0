"""What the compiler records of the attention half's kernels: the loops' registers are enough.  Three keep
a few values in scratch memory outside their steps (or in the branch of a masked step)."""
import pytest

from test_kernel_resources import kernels  # noqa: F401  (the fixture)

FEW = {"k_attention_dkv": ("Li256ELi2E", 6), "k_decode_attention": ("Li512E", 24)}


@pytest.mark.parametrize("name", ["k_attentionI", "k_attention_join", "k_attention_delta", "k_attention_dq", "k_attention_dkv",
                                  "k_decode_attention", "k_decode_join", "k_head_norm"])
def test_vector_register_spills(kernels, name):  # noqa: F811
    mine = {n: k for n, k in kernels.items() if name in n}
    assert mine
    where, most = FEW.get(name, ("", 0))
    for n, k in mine.items():
        allowed = most if where and where in n else 0
        assert k[".vgpr_spill_count"] <= allowed, (n, k[".vgpr_spill_count"])
        assert k[".private_segment_fixed_size"] <= 4 * (allowed + 1) * bool(allowed), n


def test_every_head_size_is_there(kernels):  # noqa: F811
    for name in ("k_attentionI", "k_attention_dq", "k_attention_dkv", "k_decode_attention"):
        for kind in ("DF16b", "DF16_"):
            for d in (64, 128, 256, 512):
                assert any(name in n and kind in n and f"Li{d}E" in n for n in kernels), (name, kind, d)
