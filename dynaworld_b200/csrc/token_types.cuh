// Element types, vector accesses and reductions shared by the token-side operators (norm.cu,
// linear*.cu): values are stored as float, bf16, fp16 or e4m3 and computed in float.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace gsb {

using bf16 = __nv_bfloat16;
using f16 = __half;
using e4m3 = __nv_fp8_e4m3;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(f16 v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(e4m3 v) { return float(v); }

// Round to nearest even; fp16 overflows to infinity as a torch cast does.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float v) { return __float2half_rn(v); }

// Two at once.
__device__ __forceinline__ void pack2(bf16* p, float lo, float hi) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(lo, hi);
}
__device__ __forceinline__ void pack2(f16* p, float lo, float hi) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(lo, hi);
}

// V elements moved by one access of V * sizeof(T) bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* p, float (&out)[V]) {
  const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_f32(t.v[i]);
}

// Data that is read once: it is the first to leave L2.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> read_once(const T* p) {
  if constexpr (sizeof(Vec<T, V>) == 16) {
    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const Vec<T, V>*>(&q);
  } else {
    return *reinterpret_cast<const Vec<T, V>*>(p);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_f32(T* p, const float (&in)[V]) {
  Vec<T, V> t;
  if constexpr (V % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < V; i += 2) pack2(&t.v[i], in[i], in[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = from_f32<T>(in[i]);
  }
  *reinterpret_cast<Vec<T, V>*>(p) = t;
}

// Two e4m3 codes, round to nearest even, values past 448 saturate, NaN stays NaN.
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint8_t e4m3x1(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Host: whether p and a row stride (elements) allow accesses of `bytes` bytes on every row.
inline bool vec_ok(const void* p, int64_t stride, int elem, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (stride * elem) % bytes == 0;
}

// SMs of the current device (a B200's without one).
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return 148;
  }
  int n = known[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      (void)cudaGetLastError();
      return 148;
    }
    known[dev & 63].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Column sums of the partial rows: 32 columns per block, 8 groups of rows added in a fixed order.
template <typename T>
static __global__ void __launch_bounds__(256) column_sum_kernel(const float* part, int parts, int dim, T* out) {
  __shared__ float s[8][33];
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float v = 0.0f;
  if (i < dim)
    for (int p = g; p < parts; p += 8) v += part[int64_t(p) * dim + i];
  s[g][threadIdx.x & 31] = v;
  __syncthreads();
  if (g == 0 && i < dim) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x & 31];
    out[i] = from_f32<T>(v);
  }
}

inline int elem_bytes(int dtype) { return dtype == 0 ? 4 : dtype == 3 ? 1 : 2; }

}  // namespace gsb
