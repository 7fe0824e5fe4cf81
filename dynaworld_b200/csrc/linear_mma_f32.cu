// Tensor-core products of float operands, as three bf16 parts each.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_launch_f32(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st) {
  if (p->b_mn) return mma::launch_plain<0, true, 3, float>(p, e, count, bn, splits, st);
  return mma::launch_fwd<0, 3, float>(*p, *e, bn, splits, st);
}

}  // namespace gsb
