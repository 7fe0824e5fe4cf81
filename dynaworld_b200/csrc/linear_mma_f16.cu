// Tensor-core products of f16 operands.
#include "linear_mma.cuh"

namespace gsb {

template <int BN, typename O>
static gsb_status of_width(const Product* p, const Epilogue* e, int count, const int* splits, cudaStream_t st) {
  if (p->b_mn) return mma::launch<0, 2, BN, true, 1, O, GSB_ACT_NONE>(p, e, count, splits, st);
  if constexpr (sizeof(O) == 4) return mma::launch<0, 2, BN, false, 1, O, GSB_ACT_NONE>(p, e, 1, splits, st);
  else return mma::launch_fwd<0, 2, BN, 1, O>(*p, *e, splits, st);
}

gsb_status mma_launch_f16(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st) {
  if (p->out_dtype == GSB_F32)
    return bn == 256 ? of_width<256, float>(p, e, count, splits, st) : of_width<128, float>(p, e, count, splits, st);
  return bn == 256 ? of_width<256, f16>(p, e, count, splits, st) : of_width<128, f16>(p, e, count, splits, st);
}

}  // namespace gsb
