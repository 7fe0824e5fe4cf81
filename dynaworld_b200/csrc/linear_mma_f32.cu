// Tensor-core products of f32 operands.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_product_f32(const Product& p, const Epilogue& e, cudaStream_t st) {
  return mma::launch_any<2, 128, 3, float>(p, e, st);
}

}  // namespace gsb
