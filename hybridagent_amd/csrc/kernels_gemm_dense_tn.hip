// Dense TN products (gemm_dense.hpp), the gradients of the linears' weights,
// and the plan and launch of all dense products.
#include "gemm_dense.hpp"
#include "rules.hpp"

namespace w4a16 {

hipError_t launch_gemm_dense_nt(int epi, const DgArgs& a, hipStream_t s);
hipError_t launch_gemm_dense_nn(int epi, const DgArgs& a, hipStream_t s);

static_assert(kPlanNT == (int)kDgNT && kPlanNN == (int)kDgNN && kPlanTN == (int)kDgTN, "dense_plan's layouts");

hipError_t launch_gemm_dense(int layout, int epi, DgArgs a, hipStream_t s) {
  if (a.nprob < 1 || a.nprob > kDgMaxProblems || a.K < 0) return hipErrorInvalidValue;
  const bool gu = epi == kDgGateUp;
  a.nk1 = (a.K + kDgKT - 1) / kDgKT;
  a.nk = layout == kDgNN && a.prob[0].A2 != nullptr ? 2 * a.nk1 : a.nk1;
  a.plane = 0;
  DenseShape sh[kDgMaxProblems];
  for (int i = 0; i < a.nprob; ++i) {
    DgProblem& p = a.prob[i];
    if (p.M <= 0 || p.N <= 0 || p.N % 8 != 0 || (layout != kDgTN && a.K % kDgKT != 0) ||
        (layout == kDgTN && p.M % 8 != 0))
      return hipErrorInvalidValue;
    // a tile's rows (rows format), a stage's (cols) stay within 32-bit offsets
    if ((int64_t)p.lda * 512 >= (int64_t(1) << 31) || (int64_t)p.ldb * 512 >= (int64_t(1) << 31))
      return hipErrorInvalidValue;
    p.part0 = a.plane;
    a.plane += (int64_t)p.M * p.N * (gu ? 2 : 1);
    sh[i] = DenseShape{p.M, gu ? 2 * (int64_t)p.N : p.N};
  }
  const bool thin =
      layout != kDgTN && a.nprob == 1 && dense_thin(a.prob[0].M, a.prob[0].N, gu ? 16 : 32, device_cus());
  a.mi = a.ni = 0;
  a.kg = a.ksplit = 1;
  if (!thin) {
    const DensePlan pl = dense_plan(sh, a.nprob, a.nk, a.part != nullptr ? dense_part_planes(a.plane) : 1, device_cus(),
                                    layout);
    a.mi = pl.mi;
    a.ni = pl.ni;
    a.kg = pl.kg;
    a.ksplit = pl.ksplit;
  }
  a.tiles = 0;
  for (int i = 0; i < a.nprob && !thin; ++i) {
    DgProblem& p = a.prob[i];
    const int bm = dg_bm(a.mi), bn = dg_bn(epi, a.ni);
    const int64_t t = (int64_t)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn);
    p.tile0 = a.tiles;
    if ((a.tiles + t) * a.ksplit > (int64_t(1) << 30)) return hipErrorInvalidValue;
    a.tiles += (int)t;
  }
  switch (layout) {
    case kDgNT: return launch_gemm_dense_nt(epi, a, s);
    case kDgNN: return launch_gemm_dense_nn(epi, a, s);
    case kDgTN: return epi == kDgPlain ? dg_launch_tile<kDgTN, kDgPlain>(a, s) : hipErrorInvalidValue;
    default: return hipErrorInvalidValue;
  }
}

}  // namespace w4a16
