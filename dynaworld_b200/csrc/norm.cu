// Root-mean-square norm of a residual stream, its backward, its e4m3 form, and row quantisation.
//
//   h = x + r                       (r optional; h is written back in the stream's type)
//   rstd = 1 / sqrt(mean(h^2) + eps)
//   y = h rstd w
//   dx = dr = rstd (dy w - h rstd^2 mean(dy w h)) + dh,   dw = sum over rows of dy h rstd
//   e4m3: top = max(max |y|, 1e-30), scale = top / 448, code = e4m3(y (448 / top))
//
// All of it is bound by HBM: a row is read once, kept in registers as float, reduced, and written.
// Many rows of up to 256 16-byte accesses go through norm_ring.cu.  Here: few rows, rows that start
// anywhere (one value per access) and wider ones.  A row belongs to one warp while 32 lanes x 4
// accesses hold it, to a block of 256 threads above that, and above what those hold in registers it is
// walked twice (the second walk finds it in L2).  Blocks walk rows with a grid stride so that the
// weight, and in the backward the weight gradient's partial sums, stay in registers over all rows of a
// block.  8,192 x 2,048 floats quantised: 13.2 us (6.4 TB/s); one row of 1,024: 3 us, a launch.
#include "norm_parts.cuh"

#include <type_traits>

namespace gsb {

namespace {

// One row per GROUP threads, held in registers: access j of lane t covers elements
// (j GROUP + t) V .. + V.
template <typename T, int V, int PV, int GROUP, int MODE>
__global__ void __launch_bounds__(kThreads) norm_fwd_kernel(NormArgs a) {
  __shared__ float red[kThreads / 32];
  constexpr int PER_BLOCK = kThreads / GROUP;
  const int t = threadIdx.x % GROUP, sub = threadIdx.x / GROUP;
  const int nv = a.dim / V;
  Vec<T, V> w[PV];
  if constexpr (MODE != kQuantize) {
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) w[j] = reinterpret_cast<const Vec<T, V>*>(a.w)[j * GROUP + t];
  }
  for (int64_t row = int64_t(blockIdx.x) * PER_BLOCK + sub; row < a.rows; row += int64_t(gridDim.x) * PER_BLOCK) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float h[PV][V];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const int i = j * GROUP + t;
      if (i < nv) {
        load_f32<T, V>(x + int64_t(i) * V, h[j]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) h[j][e] = 0.0f;
      }
    }
    if constexpr (MODE != kQuantize) {
      if (a.res) {
        const T* r = static_cast<const T*>(a.res) + row * a.res_stride;
#pragma unroll
        for (int j = 0; j < PV; ++j) {
          const int i = j * GROUP + t;
          if (i < nv) {
            float rv[V];
            load_f32<T, V>(r + int64_t(i) * V, rv);
#pragma unroll
            for (int e = 0; e < V; ++e) h[j][e] += rv[e];
            if (a.sum) store_f32<T, V>(static_cast<T*>(a.sum) + row * a.dim + int64_t(i) * V, h[j]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < PV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fmaf(h[j][e], h[j][e], ss);
      ss = group_sum<GROUP>(ss, red);
      const float rstd = 1.0f / sqrtf(ss * a.inv_dim + a.eps);
      if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const int i = j * GROUP + t;
        if (i < nv) {
#pragma unroll
          for (int e = 0; e < V; ++e) h[j][e] = h[j][e] * rstd * to_f32(w[j].v[e]);
          if constexpr (MODE == kNorm) store_f32<T, V>(static_cast<T*>(a.y) + row * a.dim + int64_t(i) * V, h[j]);
        }
      }
    }
    if constexpr (MODE != kNorm) {
      uint32_t top = __float_as_uint(kTiny);
#pragma unroll
      for (int j = 0; j < PV; ++j)
        if (j * GROUP + t < nv) {
#pragma unroll
          for (int e = 0; e < V; ++e) top = max(top, abs_bits(h[j][e]));
        }
      top = group_max<GROUP>(top, red);
      const float most = __uint_as_float(top);
      const float inv = kE4M3Max / most;
      if (t == 0) a.scale[row] = most / kE4M3Max;
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const int i = j * GROUP + t;
        if (i < nv) store_codes<V>(static_cast<uint8_t*>(a.y) + row * a.dim + int64_t(i) * V, h[j], inv);
      }
    }
  }
}

// Rows too wide for registers: one block per row, two (e4m3: three) walks over it.
template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads) norm_fwd_wide_kernel(NormArgs a) {
  __shared__ float red[kThreads / 32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = a.res ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;
  const T* w = static_cast<const T*>(a.w);
  float rstd = 1.0f;
  if constexpr (MODE != kQuantize) {
    float ss = 0.0f;
    for (int i = threadIdx.x; i < a.dim; i += kThreads) {
      float h = to_f32(x[i]);
      if (r) {
        h += to_f32(r[i]);
        if (a.sum) static_cast<T*>(a.sum)[row * a.dim + i] = from_f32<T>(h);
      }
      ss = fmaf(h, h, ss);
    }
    ss = group_sum<kThreads>(ss, red);
    rstd = 1.0f / sqrtf(ss * a.inv_dim + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  }
  const auto value = [&](int i) {
    float h = to_f32(x[i]);
    if constexpr (MODE == kQuantize) return h;
    if (r) h += to_f32(r[i]);
    return h * rstd * to_f32(w[i]);
  };
  if constexpr (MODE == kNorm) {
    for (int i = threadIdx.x; i < a.dim; i += kThreads)
      static_cast<T*>(a.y)[row * a.dim + i] = from_f32<T>(value(i));
  } else {
    uint32_t top = __float_as_uint(kTiny);
    for (int i = threadIdx.x; i < a.dim; i += kThreads) top = max(top, abs_bits(value(i)));
    top = group_max<kThreads>(top, red);
    const float most = __uint_as_float(top);
    const float inv = kE4M3Max / most;
    if (threadIdx.x == 0) a.scale[row] = most / kE4M3Max;
    for (int i = threadIdx.x; i < a.dim; i += kThreads)
      static_cast<uint8_t*>(a.y)[row * a.dim + i] = e4m3x1(value(i) * inv);
  }
}

// Backward of one row per GROUP threads.  h is formed again from x and the residual (the rounded
// stream would put half a step of error into every term of dw and dx).  Every thread
// adds its columns' dy h rstd over its rows in registers; a block's threads of one column are
// added in shared memory in a fixed order and leave one row of dw_part, so the weight gradient is
// the same on every run.
template <typename T, int V, int PV, int GROUP>
__global__ void __launch_bounds__(kThreads) norm_bwd_kernel(NormArgs a) {
  __shared__ float red[kThreads / 32];
  extern __shared__ float s_dw[];  // [PER_BLOCK][dim] when a block holds several rows
  constexpr int PER_BLOCK = kThreads / GROUP;
  const int t = threadIdx.x % GROUP, sub = threadIdx.x / GROUP;
  const int nv = a.dim / V;
  Vec<T, V> w[PV];
  float acc[PV][V];
#pragma unroll
  for (int j = 0; j < PV; ++j) {
    if (j * GROUP + t < nv) w[j] = reinterpret_cast<const Vec<T, V>*>(a.w)[j * GROUP + t];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[j][e] = 0.0f;
  }
  for (int64_t row = int64_t(blockIdx.x) * PER_BLOCK + sub; row < a.rows; row += int64_t(gridDim.x) * PER_BLOCK) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    const float rstd = a.rstd[row];
    Vec<T, V> g[PV], ds[PV];
    float h[PV][V];
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const int i = j * GROUP + t;
      if (i < nv) {
        load_f32<T, V>(x + int64_t(i) * V, h[j]);
        g[j] = *reinterpret_cast<const Vec<T, V>*>(dy + int64_t(i) * V);
      }
    }
    if (a.res) {
      const T* r = static_cast<const T*>(a.res) + row * a.res_stride;
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const int i = j * GROUP + t;
        if (i < nv) {
          float rv[V];
          load_f32<T, V>(r + int64_t(i) * V, rv);
#pragma unroll
          for (int e = 0; e < V; ++e) h[j][e] += rv[e];
        }
      }
    }
    if (a.dsum) {
      const T* d = static_cast<const T*>(a.dsum) + row * a.dsum_stride;
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const int i = j * GROUP + t;
        if (i < nv) ds[j] = *reinterpret_cast<const Vec<T, V>*>(d + int64_t(i) * V);
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float gh = to_f32(g[j].v[e]) * h[j][e];
          dot = fmaf(gh, to_f32(w[j].v[e]), dot);
          acc[j][e] = fmaf(gh, rstd, acc[j][e]);
        }
      }
    dot = group_sum<GROUP>(dot, red);
    const float c = rstd * rstd * (dot * a.inv_dim);
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const int i = j * GROUP + t;
      if (i < nv) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          o[e] = rstd * (to_f32(g[j].v[e]) * to_f32(w[j].v[e]) - h[j][e] * c);
          if (a.dsum) o[e] += to_f32(ds[j].v[e]);
        }
        store_f32<T, V>(static_cast<T*>(a.dx) + row * a.dim + int64_t(i) * V, o);
      }
    }
  }
  float* part = a.dw_part + int64_t(blockIdx.x) * a.dim;
  if constexpr (PER_BLOCK == 1) {
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) part[(j * GROUP + t) * V + e] = acc[j][e];
      }
  } else {
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) s_dw[sub * a.dim + (j * GROUP + t) * V + e] = acc[j][e];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += kThreads) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < PER_BLOCK; ++k) s += s_dw[k * a.dim + i];
      part[i] = s;
    }
  }
}

// Rows too wide for registers: dx with one block per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_bwd_wide_kernel(NormArgs a) {
  __shared__ float red[kThreads / 32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
  const T* d = a.dsum ? static_cast<const T*>(a.dsum) + row * a.dsum_stride : nullptr;
  const T* w = static_cast<const T*>(a.w);
  const T* r = a.res ? static_cast<const T*>(a.res) + row * a.res_stride : nullptr;
  const auto h = [&](int i) { return r ? to_f32(x[i]) + to_f32(r[i]) : to_f32(x[i]); };
  const float rstd = a.rstd[row];
  float dot = 0.0f;
  for (int i = threadIdx.x; i < a.dim; i += kThreads) dot = fmaf(to_f32(dy[i]) * h(i), to_f32(w[i]), dot);
  dot = group_sum<kThreads>(dot, red);
  const float c = rstd * rstd * (dot * a.inv_dim);
  for (int i = threadIdx.x; i < a.dim; i += kThreads) {
    float o = rstd * (to_f32(dy[i]) * to_f32(w[i]) - h(i) * c);
    if (d) o += to_f32(d[i]);
    static_cast<T*>(a.dx)[row * a.dim + i] = from_f32<T>(o);
  }
}

// ... and their weight gradient's partial sums: block (column group, row group).
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_dw_wide_kernel(NormArgs a, int64_t rows_per_part) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.dim) return;
  const int64_t lo = blockIdx.y * rows_per_part, hi = min(a.rows, lo + rows_per_part);
  float s = 0.0f;
  for (int64_t row = lo; row < hi; ++row) {
    float h = to_f32(static_cast<const T*>(a.x)[row * a.x_stride + i]);
    if (a.res) h += to_f32(static_cast<const T*>(a.res)[row * a.res_stride + i]);
    s = fmaf(to_f32(static_cast<const T*>(a.dy)[row * a.dy_stride + i]) * h, a.rstd[row], s);
  }
  a.dw_part[int64_t(blockIdx.y) * a.dim + i] = s;
}

// How a row is spread over threads.
struct Split {
  int v;      // elements per access (16 bytes, or 1 where the addresses do not allow it)
  int group;  // threads per row: 32, 256, or 0 (too wide for registers)
  int pv;     // accesses per thread
};

Split split_of(int dim, int elem, bool wide_ok) {
  const int v = wide_ok ? 16 / elem : 1;
  const int nv = dim / v;
  for (int pv = 1; pv <= 4; pv *= 2)
    if (nv <= 32 * pv) return {v, 32, pv};
  for (int pv = 1; pv <= 8; pv *= 2)
    if (nv <= kThreads * pv) return {v, kThreads, pv};
  return {v, 0, 0};
}

// Blocks per launch: enough to fill the GPU (eight of 256 threads per SM); the rows beyond are
// walked with the grid stride.
int fwd_blocks(int64_t rows, int per_block) {
  const int64_t need = (rows + per_block - 1) / per_block;
  return int(std::min<int64_t>(need, int64_t(sm_count()) * 8));
}

// Backward: two blocks per SM (register-bound); more would only add rows to the partial sums.
int bwd_blocks(int64_t rows, int per_block) {
  const int64_t need = (rows + per_block - 1) / per_block;
  return int(std::min<int64_t>(need, int64_t(sm_count()) * 2));
}

constexpr int kWideParts = 64;

template <typename T, int V, int PV, int GROUP, int MODE>
void run_fwd(const NormArgs& a, cudaStream_t st) {
  norm_fwd_kernel<T, V, PV, GROUP, MODE><<<fwd_blocks(a.rows, kThreads / GROUP), kThreads, 0, st>>>(a);
}

template <typename T, int V, int MODE>
void pick_fwd(const NormArgs& a, const Split& s, cudaStream_t st) {
  if (s.group == 32) {
    if (s.pv == 1) return run_fwd<T, V, 1, 32, MODE>(a, st);
    if (s.pv == 2) return run_fwd<T, V, 2, 32, MODE>(a, st);
    return run_fwd<T, V, 4, 32, MODE>(a, st);
  }
  if (s.pv == 1) return run_fwd<T, V, 1, kThreads, MODE>(a, st);
  if (s.pv == 2) return run_fwd<T, V, 2, kThreads, MODE>(a, st);
  if (s.pv == 4) return run_fwd<T, V, 4, kThreads, MODE>(a, st);
  return run_fwd<T, V, 8, kThreads, MODE>(a, st);
}

template <typename T, int MODE>
gsb_status fwd_of_type(const NormArgs& a, cudaStream_t st) {
  constexpr int E = sizeof(T);
  bool ok = a.dim % (16 / E) == 0 && vec_ok(a.x, a.x_stride, E, 16) && (!a.res || vec_ok(a.res, a.res_stride, E, 16)) &&
            vec_ok(a.w, 0, E, 16) && vec_ok(a.sum, 0, E, 16) && vec_ok(a.y, 0, E, 16);
  const int code = sizeof(T) == 4 ? GSB_F32 : std::is_same<T, bf16>::value ? GSB_BF16 : GSB_F16;
  if (ok && ring_fwd(a, code, MODE, st)) return launch_status();
  const Split s = split_of(a.dim, E, ok);
  if (s.group == 0)
    norm_fwd_wide_kernel<T, MODE><<<unsigned(a.rows), kThreads, 0, st>>>(a);
  else if (s.v == 1)
    pick_fwd<T, 1, MODE>(a, s, st);
  else
    pick_fwd<T, 16 / E, MODE>(a, s, st);
  note_launch();
  return launch_status();
}

template <int MODE>
gsb_status fwd(const NormArgs& a, int dtype, cudaStream_t st) {
  if (dtype == GSB_F32) return fwd_of_type<float, MODE>(a, st);
  if (dtype == GSB_BF16) return fwd_of_type<bf16, MODE>(a, st);
  return fwd_of_type<f16, MODE>(a, st);
}

template <typename T, int V, int PV, int GROUP>
int run_bwd(const NormArgs& a, cudaStream_t st) {
  constexpr int PER_BLOCK = kThreads / GROUP;
  const int blocks = bwd_blocks(a.rows, PER_BLOCK);
  const size_t smem = PER_BLOCK > 1 ? size_t(PER_BLOCK) * a.dim * 4 : 0;  // at most 8 x 1024 floats
  norm_bwd_kernel<T, V, PV, GROUP><<<blocks, kThreads, smem, st>>>(a);
  return blocks;
}

template <typename T, int V>
int pick_bwd(const NormArgs& a, const Split& s, cudaStream_t st) {
  if (s.group == 32) {
    if (s.pv == 1) return run_bwd<T, V, 1, 32>(a, st);
    if (s.pv == 2) return run_bwd<T, V, 2, 32>(a, st);
    return run_bwd<T, V, 4, 32>(a, st);
  }
  if (s.pv == 1) return run_bwd<T, V, 1, kThreads>(a, st);
  if (s.pv == 2) return run_bwd<T, V, 2, kThreads>(a, st);
  if (s.pv == 4) return run_bwd<T, V, 4, kThreads>(a, st);
  return run_bwd<T, V, 8, kThreads>(a, st);
}

template <typename T>
gsb_status bwd_of_type(const NormArgs& a, void* dw, cudaStream_t st) {
  constexpr int E = sizeof(T);
  const bool ok = a.dim % (16 / E) == 0 && vec_ok(a.x, a.x_stride, E, 16) && vec_ok(a.dy, a.dy_stride, E, 16) &&
                  (!a.res || vec_ok(a.res, a.res_stride, E, 16)) && (!a.dsum || vec_ok(a.dsum, a.dsum_stride, E, 16)) &&
                  vec_ok(a.w, 0, E, 16) && vec_ok(a.dx, 0, E, 16);
  const int code = sizeof(T) == 4 ? GSB_F32 : std::is_same<T, bf16>::value ? GSB_BF16 : GSB_F16;
  const Split s = split_of(a.dim, E, ok);
  int parts;
  if (ok && ring_bwd(a, code, &parts, st)) {
    if (dw) {
      column_sum_kernel<T><<<(a.dim + 31) / 32, 256, 0, st>>>(a.dw_part, parts, a.dim, static_cast<T*>(dw));
      note_launch();
    }
    return launch_status();
  }
  if (s.group == 0) {
    norm_bwd_wide_kernel<T><<<unsigned(a.rows), kThreads, 0, st>>>(a);
    note_launch();
    const int64_t per = (a.rows + kWideParts - 1) / kWideParts;
    parts = int((a.rows + per - 1) / per);
    norm_dw_wide_kernel<T><<<dim3((a.dim + kThreads - 1) / kThreads, parts), kThreads, 0, st>>>(a, per);
  } else if (s.v == 1) {
    parts = pick_bwd<T, 1>(a, s, st);
  } else {
    parts = pick_bwd<T, 16 / E>(a, s, st);
  }
  note_launch();
  if (dw) {
    column_sum_kernel<T><<<(a.dim + 31) / 32, 256, 0, st>>>(a.dw_part, parts, a.dim, static_cast<T*>(dw));
    note_launch();
  }
  return launch_status();
}

gsb_status check_norm(const gsb_norm* n) {
  if (!n) return GSB_ERR_ARG;
  if (n->dtype != GSB_F32 && n->dtype != GSB_BF16 && n->dtype != GSB_F16) return GSB_ERR_ARG;
  if (n->rows < 0 || n->rows > 0x7fffffff || n->dim < 1 || n->dim > (1 << 24)) return GSB_ERR_SHAPE;
  if (n->rows > 0 && !n->x) return GSB_ERR_ARG;
  return GSB_OK;
}

NormArgs args_of(const gsb_norm& n) {
  NormArgs a{};
  a.rows = n.rows;
  a.dim = n.dim;
  a.eps = n.eps;
  a.inv_dim = 1.0f / float(n.dim);
  a.x = n.x;
  a.x_stride = n.x_stride;
  a.res = n.residual;
  a.res_stride = n.residual_stride;
  a.w = n.weight;
  return a;
}

}  // namespace

gsb_status rms_norm_fwd(const gsb_norm* n, void* y, void* summed, float* rstd, cudaStream_t st) {
  if (gsb_status s = check_norm(n); s != GSB_OK) return s;
  if (n->rows == 0) return GSB_OK;
  if (!n->weight || !y || !(n->eps >= 0.0f)) return GSB_ERR_ARG;
  NormArgs a = args_of(*n);
  a.y = y;
  a.sum = summed;
  a.rstd = rstd;
  return fwd<kNorm>(a, n->dtype, st);
}

gsb_status rms_norm_fp8(const gsb_norm* n, void* codes, float* scales, void* summed, cudaStream_t st) {
  if (gsb_status s = check_norm(n); s != GSB_OK) return s;
  if (n->rows == 0) return GSB_OK;
  if (!n->weight || !codes || !scales || !(n->eps >= 0.0f)) return GSB_ERR_ARG;
  NormArgs a = args_of(*n);
  a.y = codes;
  a.scale = scales;
  a.sum = summed;
  return fwd<kNormFp8>(a, n->dtype, st);
}

gsb_status quantize_rows_fp8(const gsb_norm* n, void* codes, float* scales, cudaStream_t st) {
  if (gsb_status s = check_norm(n); s != GSB_OK) return s;
  if (n->rows == 0) return GSB_OK;
  if (!codes || !scales) return GSB_ERR_ARG;
  NormArgs a = args_of(*n);
  a.res = a.w = nullptr;
  a.y = codes;
  a.scale = scales;
  return fwd<kQuantize>(a, n->dtype, st);
}

size_t rms_norm_bwd_workspace(const gsb_norm* n) {
  if (check_norm(n) != GSB_OK) return 0;
  // as many rows of sums as any of the kernels leaves (the ring: one per SM)
  const size_t parts = std::max<size_t>(kWideParts, bwd_blocks(n->rows, 1));
  return align_up(parts * size_t(n->dim) * 4);
}

gsb_status rms_norm_bwd(const gsb_norm* n, const float* rstd, const void* dy, int64_t dy_stride, const void* dsummed,
                        int64_t dsummed_stride, void* dx, void* dweight, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (gsb_status s = check_norm(n); s != GSB_OK) return s;
  if (!n->weight) return GSB_ERR_ARG;
  if (n->rows == 0) {
    if (dweight) (void)cudaMemsetAsync(dweight, 0, size_t(n->dim) * elem_bytes(n->dtype), st);
    return launch_status();
  }
  if (!rstd || !dy || !dx || !ws) return GSB_ERR_ARG;
  if (ws_bytes < rms_norm_bwd_workspace(n)) return GSB_ERR_WORKSPACE;
  NormArgs a = args_of(*n);
  a.rstd = const_cast<float*>(rstd);
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.dsum = dsummed;
  a.dsum_stride = dsummed_stride;
  a.dx = dx;
  a.dw_part = static_cast<float*>(ws);
  if (n->dtype == GSB_F32) return bwd_of_type<float>(a, dweight, st);
  if (n->dtype == GSB_BF16) return bwd_of_type<bf16>(a, dweight, st);
  return bwd_of_type<f16>(a, dweight, st);
}

}  // namespace gsb
