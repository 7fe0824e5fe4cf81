// Tensor-core products of e4m3 operands.
#include "linear_mma.cuh"

namespace gsb {

gsb_status mma_launch_e4m3(const Product* p, const Epilogue* e, int, int bn, const int* splits, cudaStream_t st) {
  switch (p->out_dtype) {
    case GSB_F32:  // the last layers' raw outputs, and sums: not worth an instance per activation
      if (e->vec) return mma::launch_tile<1, false, 1, float, mma::kAnyAct, true>(p, e, 1, bn, splits, st);
      return mma::launch_tile<1, false, 1, float, mma::kAnyAct, false>(p, e, 1, bn, splits, st);
    case GSB_BF16: return mma::launch_fwd<1, 1, bf16>(*p, *e, bn, splits, st);
    default: return mma::launch_fwd<1, 1, f16>(*p, *e, bn, splits, st);
  }
}

}  // namespace gsb
