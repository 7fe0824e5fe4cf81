// Tensor-core products of f16 operands.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_product_f16(const Product& p, const Epilogue& e, cudaStream_t st) {
  return mma::launch_any<2, 256, 1, f16>(p, e, st);
}

}  // namespace gsb
