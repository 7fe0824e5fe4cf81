// Float sums of 16-bit products (bf16 and fp16 differ in the instruction descriptor only).
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_launch_sums16(const Product* p, const Epilogue* e, int count, int bn, const int* splits,
                             cudaStream_t st) {
  if (p->b_mn) return mma::launch_plain<0, true, 1, float>(p, e, count, bn, splits, st);
  return mma::launch_plain<0, false, 1, float>(p, e, 1, bn, splits, st);
}

}  // namespace gsb
