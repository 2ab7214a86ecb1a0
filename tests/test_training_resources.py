"""What the compiler records of the training forms' kernels: none spills a vector register or
uses scratch memory (in the products a spilled accumulator would be read back in every stage)."""
import pytest

from test_kernel_resources import kernels  # noqa: F401  (the fixture)


@pytest.mark.parametrize("name", ["k_gemm_dense", "k_gemm_thin", "k_ln_forward", "k_ln_backward", "k_column"])
def test_no_vector_register_spills(kernels, name):  # noqa: F811
    mine = {n: k for n, k in kernels.items() if name in n}
    assert mine
    spilled = {n: k[".vgpr_spill_count"] for n, k in mine.items()
               if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not spilled, spilled
