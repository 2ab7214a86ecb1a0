// Dense NT products (gemm_dense.hpp): the forward passes' linears.
#include "gemm_dense.hpp"

namespace w4a16 {

hipError_t launch_gemm_dense_nt(int epi, const DgArgs& a, hipStream_t s) {
  switch (epi) {
    case kDgPlain: return dg_launch_tile<kDgNT, kDgPlain>(a, s);
    case kDgGateUp: return dg_launch_tile<kDgNT, kDgGateUp>(a, s);
    case kDgBiasGelu: return dg_launch_tile<kDgNT, kDgBiasGelu>(a, s);
    case kDgBiasResidual: return dg_launch_tile<kDgNT, kDgBiasResidual>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace w4a16
