// Tensor-core products of e4m3 operands.
#include "linear_mma.cuh"

namespace gsb {

template <int BN>
static gsb_status of_width(const Product& p, const Epilogue& e, const int* splits, cudaStream_t st) {
  switch (p.out_dtype) {
    case GSB_F32: return mma::launch_fwd<1, 2, BN, 1, float>(p, e, splits, st);
    case GSB_BF16: return mma::launch_fwd<1, 2, BN, 1, bf16>(p, e, splits, st);
    default: return mma::launch_fwd<1, 2, BN, 1, f16>(p, e, splits, st);
  }
}

gsb_status mma_launch_e4m3(const Product* p, const Epilogue* e, int, int bn, const int* splits, cudaStream_t st) {
  return bn == 256 ? of_width<256>(*p, *e, splits, st) : of_width<128>(*p, *e, splits, st);
}

}  // namespace gsb
