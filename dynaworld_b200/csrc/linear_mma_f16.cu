// Tensor-core products of f16 operands.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_launch_f16(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st) {
  if (p->out_dtype == GSB_F32) return mma_launch_sums16(p, e, count, bn, splits, st);
  if (p->b_mn) return mma::launch_plain<0, true, 1, f16>(p, e, count, bn, splits, st);
  return mma::launch_fwd<0, 1, f16>(*p, *e, bn, splits, st);
}

}  // namespace gsb
