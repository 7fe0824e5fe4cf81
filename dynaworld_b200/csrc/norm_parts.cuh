// What the norm's kernels share: arguments, reductions over a row's threads, code stores.
#pragma once

#include "gsb_common.cuh"
#include "gsb_internal.h"
#include "token_types.cuh"

namespace gsb {

constexpr int kThreads = 256;
constexpr float kTiny = 1e-30f;   // a row of zeros gets the scale 1e-30 / 448 and codes 0
constexpr float kE4M3Max = 448.0f;

struct NormArgs {
  int64_t rows;
  int dim;
  float eps, inv_dim;
  const void* x;
  int64_t x_stride;
  const void* res;
  int64_t res_stride;
  const void* w;
  void* y;        // [rows, dim]: values or e4m3 codes
  void* sum;      // [rows, dim] or NULL
  float* rstd;    // [rows] or NULL (forward); read in the backward
  float* scale;   // [rows], e4m3 outputs
  const void* dy;
  int64_t dy_stride;
  const void* dsum;  // or NULL
  int64_t dsum_stride;
  void* dx;       // [rows, dim]
  float* dw_part; // [blocks, dim]
};

// Sum / unsigned maximum over the GROUP threads (a warp or the block) that share a row.
template <int GROUP>
__device__ __forceinline__ float group_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (GROUP > 32) {
    constexpr int W = GROUP / 32;
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // the previous use of red has been read
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += red[i];
  }
  return v;
}

template <int GROUP>
__device__ __forceinline__ uint32_t group_max(uint32_t v, float* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (GROUP > 32) {
    constexpr int W = GROUP / 32;
    const int warp = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[warp] = __uint_as_float(v);
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) v = max(v, __float_as_uint(red[i]));
  }
  return v;
}

// |v| as bits: their unsigned order is the order of the magnitudes with NaN above infinity, so a
// maximum over them keeps a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&y)[V], float inv) {
  if constexpr (V == 1) {
    *p = e4m3x1(y[0] * inv);
  } else {
    Vec<uint16_t, V / 2> c;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) c.v[i] = e4m3x2(y[2 * i] * inv, y[2 * i + 1] * inv);
    *reinterpret_cast<Vec<uint16_t, V / 2>*>(p) = c;
  }
}

enum { kNorm = 0, kNormFp8 = 1, kQuantize = 2 };

// Many aligned rows: rows arrive through a ring of asynchronous copies (norm_ring.cu).  False where
// the sizes do not suit it and nothing was launched.
bool ring_fwd(const NormArgs& a, int dtype, int mode, cudaStream_t st);
// The same for the backward; *parts: rows of dw_part it writes.
bool ring_bwd(const NormArgs& a, int dtype, int* parts, cudaStream_t st);

}  // namespace gsb
