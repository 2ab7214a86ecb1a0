// Dense NN products (gemm_dense.hpp): the gradients of the linears' inputs.
#include "gemm_dense.hpp"

namespace w4a16 {

hipError_t launch_gemm_dense_nn(int epi, const DgArgs& a, hipStream_t s) {
  switch (epi) {
    case kDgPlain: return dg_launch_tile<kDgNN, kDgPlain>(a, s);
    case kDgGateUpBack: return dg_launch_tile<kDgNN, kDgGateUpBack>(a, s);
    case kDgGeluBack: return dg_launch_tile<kDgNN, kDgGeluBack>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace w4a16
