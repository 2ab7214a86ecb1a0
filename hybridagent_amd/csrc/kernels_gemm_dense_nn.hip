// Dense NN products (gemm_dense.hpp; few rows: gemm_thin.hpp): the gradients of the linears' inputs.
#include "gemm_dense.hpp"
#include "gemm_thin.hpp"

namespace w4a16 {

hipError_t launch_gemm_dense_nn(int epi, const DgArgs& a, hipStream_t s) {
  const bool thin = a.mi == 0;
  switch (epi) {
    case kDgPlain: return thin ? thin_launch<kDgNN, kDgPlain>(a, s) : dg_launch_tile<kDgNN, kDgPlain>(a, s);
    case kDgGateUpBack: return thin ? thin_launch<kDgNN, kDgGateUpBack>(a, s) : dg_launch_tile<kDgNN, kDgGateUpBack>(a, s);
    case kDgGeluBack: return thin ? thin_launch<kDgNN, kDgGeluBack>(a, s) : dg_launch_tile<kDgNN, kDgGeluBack>(a, s);
    case kDgSums: return thin ? thin_launch<kDgNN, kDgSums>(a, s) : dg_launch_tile<kDgNN, kDgSums>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace w4a16
