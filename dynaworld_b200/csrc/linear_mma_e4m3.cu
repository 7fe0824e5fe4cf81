// Tensor-core products of e4m3 operands.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_product_e4m3(const Product& p, const Epilogue& e, cudaStream_t st) {
  switch (p.out_dtype) {
    case GSB_F32: return mma::launch_act<1, 2, 256, 1, float>(p, e, st);
    case GSB_BF16: return mma::launch_act<1, 2, 256, 1, bf16>(p, e, st);
    default: return mma::launch_act<1, 2, 256, 1, f16>(p, e, st);
  }
}

}  // namespace gsb
