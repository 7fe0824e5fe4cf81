// y = act(x w^T + b) + r and its backward.
#include "activation.cuh"
#include "gsb_common.cuh"
#include "gsb_internal.h"
#include "token_types.cuh"

namespace gsb {

namespace {

// C(i, j) = sum_k A(i, k) B(j, k) with any strides, A(i, k) = a[i a_i + k a_k].
struct Operands {
  const void* a;
  int64_t a_i, a_k;
  const void* b;
  int64_t b_j, b_k;
  int64_t m, n, k;
};

struct Epilogue {
  const float* row_scale;
  const float* col_scale;
  const void* bias;
  const void* res;
  int64_t res_stride;
  void* preact;
  void* out;
  int64_t out_stride;
};

constexpr float kHalfMax = 65504.0f;

// The pre-activation kept for the backward: float beside float operands, else fp16 saturated at
// its largest value.  fp16 and not bf16: its 11 bits keep the slope's error (at most 2^-11 |z|
// act'') an eighth of the rounding that dz gets, and beyond +-65504 every slope is constant.
__device__ __forceinline__ void put_preact(float* p, float z) { *p = z; }
__device__ __forceinline__ void put_preact(f16* p, float z) {
  *p = __float2half_rn(z != z ? z : fminf(fmaxf(z, -kHalfMax), kHalfMax));
}

template <typename T>
struct PreactOf { using type = f16; };
template <>
struct PreactOf<float> { using type = float; };

constexpr int kTile = 64, kDepth = 16;

template <typename T, typename O, int ACT>
__global__ void __launch_bounds__(256) product_kernel(Operands p, Epilogue e) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int64_t i0 = int64_t(blockIdx.x) * kTile;
  const int64_t j0 = int64_t(blockIdx.y) * kTile;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
    for (int s = threadIdx.x; s < kTile * kDepth; s += 256) {
      // the unit-stride index runs fastest over the threads
      const int ai = p.a_k == 1 ? s / kDepth : s % kTile, ak = p.a_k == 1 ? s % kDepth : s / kTile;
      const bool a_in = i0 + ai < p.m && k0 + ak < p.k;
      sa[ak][ai] = a_in ? to_f32(a[(i0 + ai) * p.a_i + (k0 + ak) * p.a_k]) : 0.0f;
      const int bj = p.b_k == 1 ? s / kDepth : s % kTile, bk = p.b_k == 1 ? s % kDepth : s / kTile;
      const bool b_in = j0 + bj < p.n && k0 + bk < p.k;
      sb[bk][bj] = b_in ? to_f32(b[(j0 + bj) * p.b_j + (k0 + bk) * p.b_k]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float av[4], bv[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        av[u] = sa[k][ty + 16 * u];
        bv[u] = sb[k][tx + 16 * u];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(av[u], bv[v], acc[u][v]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = i0 + ty + 16 * u;
    if (i >= p.m) continue;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t j = j0 + tx + 16 * v;
      if (j >= p.n) continue;
      float z = acc[u][v];
      if (e.row_scale) z *= e.row_scale[i] * e.col_scale[j];
      if (e.bias) z += to_f32(static_cast<const O*>(e.bias)[j]);
      if (e.preact) put_preact(static_cast<typename PreactOf<O>::type*>(e.preact) + i * p.n + j, z);
      float y = act_value<ACT>(z);
      if (e.res) y += to_f32(static_cast<const O*>(e.res)[i * e.res_stride + j]);
      static_cast<O*>(e.out)[i * e.out_stride + j] = from_f32<O>(y);
    }
  }
}

template <typename T, typename O, int ACT>
void product(const Operands& p, const Epilogue& e, cudaStream_t st) {
  product_kernel<T, O, ACT><<<dim3(unsigned((p.m + kTile - 1) / kTile), unsigned((p.n + kTile - 1) / kTile)), 256, 0,
                             st>>>(p, e);
  note_launch();
}

template <typename T, typename O>
void product_act(int act, const Operands& p, const Epilogue& e, cudaStream_t st) {
  switch (act) {
    case GSB_ACT_RELU: return product<T, O, GSB_ACT_RELU>(p, e, st);
    case GSB_ACT_GELU: return product<T, O, GSB_ACT_GELU>(p, e, st);
    case GSB_ACT_GELU_TANH: return product<T, O, GSB_ACT_GELU_TANH>(p, e, st);
    case GSB_ACT_SILU: return product<T, O, GSB_ACT_SILU>(p, e, st);
    default: return product<T, O, GSB_ACT_NONE>(p, e, st);
  }
}

// dz = dy act'(z) in the operands' type (dz NULL: only the column sums), and per block of rows the
// float column sums of the unrounded dz.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) dz_kernel(const T* dy, int64_t dy_stride, const typename PreactOf<T>::type* z,
                                                 T* dz, float* part, int64_t m, int n, int64_t rows_per_part) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  const int64_t lo = blockIdx.y * rows_per_part, hi = min(m, lo + rows_per_part);
  float s = 0.0f;
  for (int64_t i = lo; i < hi; ++i) {
    float v = to_f32(dy[i * dy_stride + j]);
    if constexpr (ACT != GSB_ACT_NONE) v *= act_slope<ACT>(to_f32(z[i * n + j]));
    if (dz) dz[i * n + j] = from_f32<T>(v);
    s += v;
  }
  if (part) part[int64_t(blockIdx.y) * n + j] = s;
}

constexpr int kDzParts = 128;

template <typename T, int ACT>
void launch_dz(const void* dy, int64_t dy_stride, const void* z, void* dz, float* part, int64_t m, int n,
               int64_t per, int parts, cudaStream_t st) {
  using Z = typename PreactOf<T>::type;
  dz_kernel<T, ACT><<<dim3((n + 255) / 256, parts), 256, 0, st>>>(static_cast<const T*>(dy), dy_stride,
                                                                static_cast<const Z*>(z), static_cast<T*>(dz), part, m,
                                                                n, per);
  note_launch();
}

struct BwdSpace {
  void* dz;
  float* part;
  size_t bytes;
};

BwdSpace bwd_space(const gsb_linear& p, void* ws, size_t cap) {
  Carver c(ws, cap);
  BwdSpace s{};
  s.part = c.take<float>(size_t(kDzParts) * p.n);
  if (p.activation != GSB_ACT_NONE) s.dz = c.take<char>(size_t(p.m) * p.n * elem_bytes(p.dtype));
  s.bytes = c.used;
  return s;
}

template <typename T>
gsb_status bwd_of_type(const gsb_linear& p, const void* z, const void* dy, int64_t dy_stride, void* dx, void* dw,
                       void* db, const BwdSpace& s, cudaStream_t st) {
  const int64_t per = (p.m + kDzParts - 1) / kDzParts;
  const int parts = int((p.m + per - 1) / per);
  const void* dz = dy;
  int64_t dz_stride = dy_stride;
  if (p.activation != GSB_ACT_NONE) {
    dz = s.dz;
    dz_stride = p.n;
  }
  if (db || p.activation != GSB_ACT_NONE) {
    void* out = p.activation != GSB_ACT_NONE ? s.dz : nullptr;
    float* part = db ? s.part : nullptr;
    switch (p.activation) {
      case GSB_ACT_RELU: launch_dz<T, GSB_ACT_RELU>(dy, dy_stride, z, out, part, p.m, p.n, per, parts, st); break;
      case GSB_ACT_GELU: launch_dz<T, GSB_ACT_GELU>(dy, dy_stride, z, out, part, p.m, p.n, per, parts, st); break;
      case GSB_ACT_GELU_TANH:
        launch_dz<T, GSB_ACT_GELU_TANH>(dy, dy_stride, z, out, part, p.m, p.n, per, parts, st);
        break;
      case GSB_ACT_SILU: launch_dz<T, GSB_ACT_SILU>(dy, dy_stride, z, out, part, p.m, p.n, per, parts, st); break;
      default: launch_dz<T, GSB_ACT_NONE>(dy, dy_stride, z, out, part, p.m, p.n, per, parts, st); break;
    }
    if (db) {
      column_sum_kernel<T><<<(p.n + 31) / 32, 256, 0, st>>>(s.part, parts, p.n, static_cast<T*>(db));
      note_launch();
    }
  }
  if (dx) {
    Epilogue e{};
    e.out = dx;
    e.out_stride = p.k;
    product<T, T, GSB_ACT_NONE>({dz, dz_stride, 1, p.weight, 1, p.weight_stride, p.m, p.k, p.n}, e, st);
  }
  if (dw) {
    Epilogue e{};
    e.out = dw;
    e.out_stride = p.k;
    product<T, T, GSB_ACT_NONE>({dz, 1, dz_stride, p.x, 1, p.x_stride, p.n, p.k, p.m}, e, st);
  }
  return launch_status();
}

gsb_status check_linear(const gsb_linear* p) {
  if (!p) return GSB_ERR_ARG;
  if (p->dtype < GSB_F32 || p->dtype > GSB_E4M3) return GSB_ERR_ARG;
  if (p->out_dtype < GSB_F32 || p->out_dtype > GSB_F16) return GSB_ERR_ARG;
  if (p->dtype != GSB_E4M3 && p->out_dtype != p->dtype) return GSB_ERR_ARG;
  if (p->activation < GSB_ACT_NONE || p->activation > GSB_ACT_SILU) return GSB_ERR_ARG;
  if (p->m < 0 || p->m > 0x7fffffff || p->n < 1 || p->k < 1 || p->n > (1 << 24) || p->k > (1 << 24))
    return GSB_ERR_SHAPE;
  return GSB_OK;
}

gsb_status check_operands(const gsb_linear* p) {
  if (!p->weight || (p->m > 0 && !p->x)) return GSB_ERR_ARG;
  if (p->dtype == GSB_E4M3 && p->m > 0 && (!p->x_scale || !p->weight_scale)) return GSB_ERR_ARG;
  return GSB_OK;
}

}  // namespace

size_t linear_fwd_workspace(const gsb_linear* p) {
  if (check_linear(p) != GSB_OK) return 0;
  return kAlign;
}

gsb_status linear_fwd(const gsb_linear* p, void* y, void* preact, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (gsb_status s = check_linear(p); s != GSB_OK) return s;
  if (gsb_status s = check_operands(p); s != GSB_OK) return s;
  if (p->dtype == GSB_E4M3 && preact) return GSB_ERR_ARG;
  if (p->m == 0) return GSB_OK;
  if (!y) return GSB_ERR_ARG;
  Operands o{p->x, p->x_stride, 1, p->weight, p->weight_stride, 1, p->m, p->n, p->k};
  Epilogue e{};
  if (p->dtype == GSB_E4M3) {
    e.row_scale = p->x_scale;
    e.col_scale = p->weight_scale;
  }
  e.bias = p->bias;
  e.res = p->residual;
  e.res_stride = p->residual_stride;
  e.preact = preact;
  e.out = y;
  e.out_stride = p->n;
  switch (p->dtype) {
    case GSB_F32: product_act<float, float>(p->activation, o, e, st); break;
    case GSB_BF16: product_act<bf16, bf16>(p->activation, o, e, st); break;
    case GSB_F16: product_act<f16, f16>(p->activation, o, e, st); break;
    default:
      if (p->out_dtype == GSB_F32) product_act<e4m3, float>(p->activation, o, e, st);
      else if (p->out_dtype == GSB_BF16) product_act<e4m3, bf16>(p->activation, o, e, st);
      else product_act<e4m3, f16>(p->activation, o, e, st);
  }
  return launch_status();
}

size_t linear_bwd_workspace(const gsb_linear* p) {
  if (check_linear(p) != GSB_OK) return 0;
  return bwd_space(*p, nullptr, 0).bytes;
}

gsb_status linear_bwd(const gsb_linear* p, const void* preact, const void* dy, int64_t dy_stride, void* dx,
                      void* dweight, void* dbias, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (gsb_status s = check_linear(p); s != GSB_OK) return s;
  if (p->dtype == GSB_E4M3) return GSB_ERR_ARG;
  if (p->m == 0) {
    const size_t e = elem_bytes(p->dtype);
    if (dweight) (void)cudaMemsetAsync(dweight, 0, size_t(p->n) * p->k * e, st);
    if (dbias) (void)cudaMemsetAsync(dbias, 0, size_t(p->n) * e, st);
    return launch_status();
  }
  if (!dy || (p->activation != GSB_ACT_NONE && !preact)) return GSB_ERR_ARG;
  if ((dx && !p->weight) || (dweight && !p->x)) return GSB_ERR_ARG;
  if (!ws || ws_bytes < linear_bwd_workspace(p)) return GSB_ERR_WORKSPACE;
  const BwdSpace s = bwd_space(*p, ws, ws_bytes);
  switch (p->dtype) {
    case GSB_F32: return bwd_of_type<float>(*p, preact, dy, dy_stride, dx, dweight, dbias, s, st);
    case GSB_BF16: return bwd_of_type<bf16>(*p, preact, dy, dy_stride, dx, dweight, dbias, s, st);
    default: return bwd_of_type<f16>(*p, preact, dy, dy_stride, dx, dweight, dbias, s, st);
  }
}

}  // namespace gsb
