"""The host rules of the dense GEMMs (gemm_dense.hpp), compiled for the CPU: every plan is a
tile that is built, its partial sums fit, and it is among the fast ones where they were
measured on an MI355X."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "hybridagent_amd" / "csrc"

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
  long long n, rows, cols, nk, plane, cus, layout;
  while (scanf("%lld %lld %lld %lld %lld %lld %lld", &n, &rows, &cols, &nk, &plane, &cus, &layout) == 7) {
    DenseShape sh[3];
    for (int i = 0; i < n; ++i) sh[i] = DenseShape{rows, cols};
    const int planes = dense_part_planes(plane);
    const DensePlan p = dense_plan(sh, (int)n, (int)nk, planes, (int)cus, (int)layout);
    printf("%d %d %d %d %d\\n", p.mi, p.ni, p.kg, p.ksplit, planes);
  }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)

    def run(calls):
        out = subprocess.run([str(d / "plan")], input="\n".join(" ".join(map(str, c)) for c in calls), text=True,
                             capture_output=True, check=True).stdout.split("\n-\n")
        *tiles, got = ([tuple(map(int, ln.split())) for ln in part.split("\n") if ln] for part in out)
        return tiles, got

    return run


def test_every_plan_is_built_and_fits(plans):
    calls = [(n, m, c, nk, n * m * c, cus, nk % 3) for n in (1, 2, 3) for m in (1, 33, 200, 517, 2049, 8192, 100_000)
             for c in (32, 512, 2112, 4224, 32768) for nk in (0, 1, 7, 66, 256, 5000) for cus in (32, 256, 304)]
    tiles, got = plans(calls)
    assert all(len(t) == len(set(t)) for t in tiles)
    for (n, m, c, nk, plane, _, layout), (mi, ni, kg, ks, planes) in zip(calls, got):
        assert (mi, ni, kg) in tiles[layout]
        assert 1 <= ks <= planes <= 8
        assert planes == 1 or planes * plane <= 8 << 20
        assert ks == 1 or nk >= 2 * ks * kg


# x W^T, dy W and dy^T x at the model's shapes: the tiles (and splits) within 6 % of the fastest measured
MEASURED = [  # products, rows, columns, stages of 32 k, partial plane, layout (x W^T 0, dy W 1, dy^T x 2)
    ((1, 8192, 4224, 88, 8192 * 4224, 0), {"8x6x1", "6x8x1"}),
    ((1, 8192, 2816, 66, 8192 * 2816, 0), {"8x6x1", "6x8x1"}),
    ((1, 8192, 2112, 88, 8192 * 2112, 1), {"6x6x1"}),
    ((1, 2049, 2816, 88, 2049 * 2816, 0), {"6x4x1", "4x6x1"}),
    ((1, 2049, 2816, 88, 2049 * 2816, 1), {"6x4x1"}),
    ((1, 517, 2816, 66, 517 * 2816, 0), {"4x2x1"}),
    ((1, 517, 2112, 88, 517 * 2112, 1), {"2x4x2"}),
    ((1, 100, 2816, 66, 100 * 2816, 0), {"2x2x1"}),
    ((1, 1024, 2816, 88, 1024 * 2816, 0), {"4x4x1"}),
    ((3, 2816, 2112, 256, 3 * 2816 * 2112, 2), {"6x6x1"}),
    ((2, 2816, 2816, 65, 2 * 2816 * 2816, 2), {"8x8x1", "8x4x1", "4x8x1", "6x6x1"}),
    ((2, 2816, 2816, 1, 2 * 2816 * 2816, 2), {"8x4x1", "4x8x1", "6x6x1"}),
]


def test_plans_are_among_the_fast_ones(plans):
    _, got = plans([(*c[:5], 256, c[5]) for c, _ in MEASURED])
    for (c, fast), (mi, ni, kg, ks, _) in zip(MEASURED, got):
        assert f"{mi}x{ni}x{kg}" in fast and ks == 1, (c, mi, ni, kg, ks)
