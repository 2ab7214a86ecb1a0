"""The shapes that the GPU tests of the training forms run reach every tile, and a split's join, of
every product and epilogue on 256 CUs: the rules (rules.hpp) compiled for the CPU.  And the sizes of
what the forward passes keep."""
import shutil
import subprocess
from pathlib import Path

import pytest

import test_gpu_training as gpu
import test_gpu_training_use as use
from hybridagent_amd import _lib

CSRC = Path(__file__).resolve().parent.parent / "hybridagent_amd" / "csrc"
NT, NN, TN = 0, 1, 2

PROGRAM = """
#include <cstdio>
#include "rules.hpp"
using namespace w4a16;
int main() {
#define W4A16_DG(MI_, NI_, KG_, OCC_, ALONE_, EACH_) printf("%d %d %d\\n", MI_, NI_, KG_);
  W4A16_DG_TILES_NT(W4A16_DG)
  printf("-\\n");
  W4A16_DG_TILES_NN(W4A16_DG)
  printf("-\\n");
  W4A16_DG_TILES_TN(W4A16_DG)
#undef W4A16_DG
  printf("-\\n");
  // layout, 32-row stages, columns of a few-rows workgroup, products; each: rows, columns, operand's columns
  long long layout, nk, cols, n, r[3], c[3], w[3];
  while (scanf("%lld %lld %lld %lld", &layout, &nk, &cols, &n) == 4) {
    DenseShape sh[3];
    long long plane = 0;
    for (int i = 0; i < n; ++i) {
      if (scanf("%lld %lld %lld", r + i, c + i, w + i) != 3) return 1;
      sh[i] = DenseShape{r[i], w[i]};
      plane += r[i] * w[i];
    }
    if (layout != kPlanTN && dense_thin(r[0], c[0], (int)cols, 256)) {
      printf("0 0 0 1\\n");
      continue;
    }
    const DensePlan p = dense_plan(sh, (int)n, (int)nk, dense_part_planes(plane), 256, (int)layout);
    printf("%d %d %d %d\\n", p.mi, p.ni, p.kg, p.ksplit);
  }
}
"""


def _shapes(*tests):
    return [v for t in tests for mark in t.pytestmark if mark.name == "parametrize" for v in mark.args[1]]


def _mlp(T, H, I):
    k, wide = (T + 31) // 32, [(H, I, I), (I, H, H), (I, H, H)]
    return [("gate/up", NT, H // 32, 16, [(T, I, 2 * I)]), ("plain", NT, I // 32, 32, [(T, H, H)]),
            ("gate/up gradients", NN, H // 32, 32, [(T, I, I)]), ("plain", NN, 2 * (I // 32), 32, [(T, H, H)]),
            ("plain", TN, k, 32, wide)]


def _link(T, H):
    one = [(T, H, H)]
    return [("bias, GELU", NT, H // 32, 32, one), ("bias, residual", NT, H // 32, 32, one),
            ("GELU's slope", NN, H // 32, 32, one), ("sums", NN, H // 32, 32, one),
            ("plain", TN, (T + 31) // 32, 32, [(H, H, H)] * 2)]


def test_every_tile_of_every_product_is_reached(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{CSRC}", str(tmp_path / "plan.cpp"), "-o", str(tmp_path / "plan")],
                   check=True)
    calls = [c for s in _shapes(gpu.test_gated_mlp, gpu.test_gated_mlp_few_rows_of_wide_or_narrow_outputs,
                                gpu.test_gated_mlp_every_tile, use.test_gated_mlp_more_tiles) for c in _mlp(*s)]
    calls += [c for s in _shapes(gpu.test_hybridlink_training, gpu.test_hybridlink_every_tile,
                                 gpu.test_hybridlink_few_rows_of_wide_or_narrow_outputs) for c in _link(*s)]
    lines = [" ".join(map(str, (layout, nk, cols, len(p), *(v for q in p for v in q))))
             for _, layout, nk, cols, p in calls]
    out = subprocess.run([str(tmp_path / "plan")], input="\n".join(lines), text=True, capture_output=True,
                         check=True).stdout.split("\n-\n")
    *tiles, got = ([tuple(map(int, ln.split())) for ln in part.split("\n") if ln] for part in out)
    assert len(got) == len(calls)
    reached, split = {}, set()
    for (name, layout, *_), (mi, ni, kg, ksplit) in zip(calls, got):
        reached.setdefault((name, layout), set()).add((mi, ni, kg))
        if ksplit > 1:
            split.add(name)
    for (name, layout), seen in reached.items():
        few = set() if layout == TN else {(0, 0, 0)}
        assert seen == set(tiles[layout]) | few, (name, layout, (set(tiles[layout]) | few) - seen)
    assert split == {name for name, _ in reached}, {name for name, _ in reached} - split


def test_sizes_of_what_the_forward_passes_keep():
    """The gated MLP: two fp32 sums and a bf16 product per row and column of I; HybridLink: two bf16
    operands, two fp32 sums per element and two norms' statistics per row."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libw4a16moe.so not built")
    lib = _lib.load()
    for M, n in ((1, 32), (4, 96), (517, 2112)):
        assert 10 * M * n <= lib.w4a16_gated_mlp_saved_bytes(M, n) <= 10 * M * n + 3 * 256
        assert 12 * M * n + 16 * M <= lib.w4a16_hybridlink_saved_bytes(M, n) <= 12 * M * n + 16 * M + 8 * 256
