// Dense NT products (gemm_dense.hpp; few rows: gemm_thin.hpp): the forward passes' linears.
#include "gemm_dense.hpp"
#include "gemm_thin.hpp"

namespace w4a16 {

hipError_t launch_gemm_dense_nt(int epi, const DgArgs& a, hipStream_t s) {
  const bool thin = a.mi == 0;
  switch (epi) {
    case kDgPlain: return thin ? thin_launch<kDgNT, kDgPlain>(a, s) : dg_launch_tile<kDgNT, kDgPlain>(a, s);
    case kDgGateUp: return thin ? thin_launch<kDgNT, kDgGateUp>(a, s) : dg_launch_tile<kDgNT, kDgGateUp>(a, s);
    case kDgBiasGelu: return thin ? thin_launch<kDgNT, kDgBiasGelu>(a, s) : dg_launch_tile<kDgNT, kDgBiasGelu>(a, s);
    case kDgBiasResidual: return thin ? thin_launch<kDgNT, kDgBiasResidual>(a, s) : dg_launch_tile<kDgNT, kDgBiasResidual>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace w4a16
