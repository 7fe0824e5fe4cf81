// Tensor-core products of float operands, as three bf16 parts each.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_launch_f32(const Product* p, const Epilogue* e, int count, int, const int* splits, cudaStream_t st) {
  if (p->b_mn) return mma::launch<0, 2, 256, true, 3, float, GSB_ACT_NONE>(p, e, count, splits, st);
  return mma::launch_fwd<0, 2, 256, 3, float>(*p, *e, splits, st);
}

}  // namespace gsb
