// Tensor-core products: what the types' files share.
#include "linear_mma.cuh"

namespace gsb {
namespace mma {

EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

}  // namespace mma

static __device__ int g_gave_up;

int* gave_up_flag() {
  static std::atomic<int*> at[64];  // by device
  int dev = 0;
  (void)cudaGetDevice(&dev);
  int* p = at[dev & 63].load(std::memory_order_relaxed);
  if (p) return p;
  void* q = nullptr;
  if (cudaGetSymbolAddress(&q, g_gave_up) != cudaSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  at[dev & 63].store(static_cast<int*>(q), std::memory_order_relaxed);
  return static_cast<int*>(q);
}

gsb_status gave_up_status(int* gave_up) {
  if (cudaMemcpyFromSymbol(gave_up, g_gave_up, sizeof(int)) != cudaSuccess) {
    (void)cudaGetLastError();
    return GSB_ERR_CUDA;
  }
  return GSB_OK;
}

gsb_status mma_product(const Product& p, const Epilogue& e, cudaStream_t st) {
  switch (p.dtype) {
    case GSB_F32: return mma_product_f32(p, e, st);
    case GSB_BF16: return mma_product_bf16(p, e, st);
    case GSB_F16: return mma_product_f16(p, e, st);
    default: return mma_product_e4m3(p, e, st);
  }
}

}  // namespace gsb
