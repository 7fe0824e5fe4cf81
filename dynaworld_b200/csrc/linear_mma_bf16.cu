// Tensor-core products of bf16 operands.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_product_bf16(const Product& p, const Epilogue& e, cudaStream_t st) {
  return mma::launch_any<2, 256, 1, bf16>(p, e, st);
}

}  // namespace gsb
