// What the matrix product's kernels share: operands, epilogue and the element-wise tail.
#pragma once

#include "activation.cuh"
#include "gsb_common.cuh"
#include "gsb_internal.h"
#include "token_types.cuh"

namespace gsb {

// What happens to a sum z: scales (e4m3 operands), bias, copy of z for the backward, activation,
// residual, rounding.  bias, res and out are of the output type.
struct Epilogue {
  const float* row_scale;
  const float* col_scale;
  const void* bias;
  const void* res;
  int64_t res_stride;
  void* preact;
  void* out;
  int64_t out_stride;
  int act;
  int vec;  // out, preact, bias and res rows allow 16-byte accesses
};

// D = A B^T, A [m, k] and B [n, k]; *_mn: stored [k, m] ([k, n]) with the rows of k.
struct Product {
  const void* a;
  int64_t a_ld;  // elements between stored rows
  bool a_mn;
  const void* b;
  int64_t b_ld;
  bool b_mn;
  int64_t m;
  int64_t n;
  int64_t k;
  int dtype;      // of a and b: GSB_BF16, GSB_F16, GSB_E4M3; GSB_F32: three bf16 parts each
  int out_dtype;
  int64_t a_plane, b_plane;  // GSB_F32: elements between the parts
};

// The pre-activation kept for the backward: float beside float operands, else fp16 saturated at
// its largest value.  fp16 and not bf16: its 11 bits keep the slope's error (at most 2^-11 |z|
// act'') an eighth of the rounding that dz gets, and beyond +-65504 every slope is constant.  ReLU's
// slope jumps at 0 however small z is: there a z that would round to 0 from above is kept as the least
// fp16 (bf16 operands reach z = 1e-38, and their gradients would be lost).
constexpr float kLeastHalf = 5.9604644775390625e-08f;  // 2^-24
__device__ __forceinline__ float on_its_side(float z) { return z > 0.0f ? fmaxf(z, kLeastHalf) : z; }

__device__ __forceinline__ float as_preact(float*, float z, bool) { return z; }
__device__ __forceinline__ f16 as_preact(f16*, float z, bool relu) {
  if (relu) z = on_its_side(z);
  uint16_t h;
  asm("cvt.rn.satfinite.f16.f32 %0, %1;" : "=h"(h) : "f"(z));
  return __ushort_as_half(h);
}

template <typename T>
struct PreactOf { using type = f16; };
template <>
struct PreactOf<float> { using type = float; };

template <typename O, int V>
__device__ __forceinline__ void apply_act(int act, float (&z)[V]) {
  switch (act) {
    case GSB_ACT_RELU: apply_value<GSB_ACT_RELU, O, V>(z); break;
    case GSB_ACT_GELU: apply_value<GSB_ACT_GELU, O, V>(z); break;
    case GSB_ACT_GELU_TANH: apply_value<GSB_ACT_GELU_TANH, O, V>(z); break;
    case GSB_ACT_SILU: apply_value<GSB_ACT_SILU, O, V>(z); break;
    default: break;
  }
}

// z as it is kept; relu: for ReLU's backward.
template <int V>
__device__ __forceinline__ Vec<float, V> kept_of(float*, const float (&z)[V], bool) {
  Vec<float, V> k;
#pragma unroll
  for (int u = 0; u < V; ++u) k.v[u] = z[u];
  return k;
}
template <int V>
__device__ __forceinline__ Vec<f16, V> kept_of(f16*, const float (&z)[V], bool relu) {
  Vec<f16, V> k;
  if constexpr (V == 1) {
    k.v[0] = as_preact(static_cast<f16*>(nullptr), z[0], relu);
  } else {
#pragma unroll
    for (int u = 0; u < V; u += 2) {
      const float lo = relu ? on_its_side(z[u]) : z[u], hi = relu ? on_its_side(z[u + 1]) : z[u + 1];
      asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(*reinterpret_cast<uint32_t*>(&k.v[u])) : "f"(hi), "f"(lo));
    }
  }
  return k;
}

// V adjacent sums of row i from column j on.
template <typename O, int V>
__device__ __forceinline__ void finish(const Epilogue& e, int64_t n, int64_t i, int64_t j, float (&z)[V]) {
  using Z = typename PreactOf<O>::type;
  if (e.row_scale) {
    const float rs = e.row_scale[i];
#pragma unroll
    for (int u = 0; u < V; ++u) z[u] *= rs * e.col_scale[j + u];
  }
  if (e.bias) {
    float b[V];
    load_f32<O, V>(static_cast<const O*>(e.bias) + j, b);
#pragma unroll
    for (int u = 0; u < V; ++u) z[u] += b[u];
  }
  if (e.preact) {
    *reinterpret_cast<Vec<Z, V>*>(static_cast<Z*>(e.preact) + i * n + j) =
        kept_of<V>(static_cast<Z*>(nullptr), z, e.act == GSB_ACT_RELU);
  }
  apply_act<O, V>(e.act, z);
  if (e.res) {
    float r[V];
    load_f32<O, V>(static_cast<const O*>(e.res) + i * e.res_stride + j, r);
#pragma unroll
    for (int u = 0; u < V; ++u) z[u] += r[u];
  }
  store_f32<O, V>(static_cast<O*>(e.out) + i * e.out_stride + j, z);
}

inline int k_blocks_of(const Product& p) {
  const int64_t per = p.dtype == GSB_E4M3 ? 128 : 64;
  return int((p.k + per - 1) / per);
}

// 2 to 32 aligned rows of 16-bit or e4m3 values (linear_few.cu).
bool few_rows_mma_serves(const gsb_linear& p);
void few_rows_mma(const gsb_linear& p, const Epilogue& e, cudaStream_t st);

// Blocks of K of one of its `splits` pieces, and how many pieces that makes.
inline int piece_of(const Product& p, int splits) { return (k_blocks_of(p) + splits - 1) / splits; }
inline int pieces_of(const Product& p, int splits) {
  const int per = piece_of(p, splits);
  return (k_blocks_of(p) + per - 1) / per;
}

// How the tensor-core kernel walks a product: tiles of 256 x 256 (bn 256) or 128 x bn, each in `splits` pieces along K whose
// float sums a second kernel adds (in order) and finishes.
struct Plan {
  int bn;
  int splits[2];  // of the launch's one or two products
  float cost;     // estimated, in blocks of K of a 256 x 256 tile
};
Plan plan_product(const Product& p);
// The backward's two products in one launch.
Plan plan_pair(const Product (&p)[2]);
size_t partial_bytes(const Product* p, int count, const Plan& plan);

// The products (linear_mma.cu).  The operands' rows (and parts) start on 16-byte boundaries; `part` is
// partial_bytes long.
gsb_status mma_products(const Product* p, const Epilogue* e, int count, const Plan& plan, void* part, cudaStream_t st);
// By operand type: products[0 .. count) of one launch, count 2 only with b_mn.  out_dtype F32 beside
// 16-bit operands writes sums (no epilogue).
gsb_status mma_launch_sums16(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st);
gsb_status mma_launch_bf16(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st);
gsb_status mma_launch_f16(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st);
gsb_status mma_launch_f32(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st);
gsb_status mma_launch_e4m3(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st);
// 1 when a bounded wait of a token-side kernel gave up on the current device since this last gave 1.
gsb_status gave_up_status(int* gave_up);

}  // namespace gsb
