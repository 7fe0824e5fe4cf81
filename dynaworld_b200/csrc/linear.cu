// y = act(x w^T + b) + r and its backward.
#include "linear_parts.cuh"

#include <type_traits>

namespace gsb {

namespace {

// Which kernels serve a forward: the weights walked row by row without the tensor cores (one row; float
// or unaligned rows, up to 64 while the weights stay in L2 between eight rows and the next), the
// warp-wide MMA, or tcgen05 tiles.  1,024 x 1,024 float, 16 rows: 6.0 us, 17 on tiles; 64 rows: 12.8.
enum class Path { kWalk, kFewMma, kTiles };
Path path_of(const gsb_linear& p) {
  if (few_rows_mma_serves(p)) return Path::kFewMma;
  const int b = elem_bytes(p.dtype);
  const bool aligned = p.dtype != GSB_F32 && p.k % (16 / b) == 0 && vec_ok(p.x, p.x_stride, b, 16) &&
                       vec_ok(p.weight, p.weight_stride, b, 16);
  const int64_t most = aligned ? 1 : int64_t(p.n) * p.k * b <= (8 << 20) ? 64 : 8;
  return p.m <= most ? Path::kWalk : Path::kTiles;
}

// ---- one row; a few float or unaligned rows ------------------------------------------------------
// Bound by the weights' bytes (1,024 x 4,096 bf16: 3.0 us, most of it a launch and the way to HBM and
// back).  A warp owns C columns and walks their weight rows in 16-byte accesses, all ROWS tokens at
// once, so that the weights are read once; the tokens come from L1.  Float operands stay float.
template <typename T, typename O, int V, int ROWS, int C>
__global__ void __launch_bounds__(128) few_rows_kernel(const T* x, int64_t x_stride, const T* w, int64_t w_stride, int m,
                                                       int n, int k, Epilogue e) {
  const int lane = threadIdx.x & 31;
  const int j0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * C;
  if (j0 >= n) return;
  const int r0 = blockIdx.y * ROWS;  // float rows beyond ROWS: the weights come from L2 for each ROWS more
  x += int64_t(r0) * x_stride;
  m -= r0;
  float acc[ROWS][C];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[r][c] = 0.0f;
  const T* wr[C];
#pragma unroll
  for (int c = 0; c < C; ++c) wr[c] = w + int64_t(min(j0 + c, n - 1)) * w_stride;
#pragma unroll(C* ROWS <= 4 ? 4 : 2)
  for (int i = lane * V; i < k; i += 32 * V) {
    float wv[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) load_f32<T, V>(wr[c] + i, wv[c]);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float xv[V];
      load_f32<T, V>(x + int64_t(min(r, m - 1)) * x_stride + i, xv);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int u = 0; u < V; ++u) acc[r][c] = fmaf(xv[u], wv[c][u], acc[r][c]);
    }
  }
  // lane r C + c keeps that sum, so that the lanes finish theirs together
  float z[1] = {0.0f};
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float s = warp_sum(acc[r][c]);
      if (lane == r * C + c) z[0] = s;
    }
  const int r = lane / C, c = lane % C;
  if (r < ROWS && r < m && j0 + c < n) finish<O, 1>(e, n, r0 + r, j0 + c, z);
}

template <typename T, typename O, int V>
void few_rows_v(const gsb_linear& p, const Epilogue& e, cudaStream_t st) {
  const auto run = [&](auto kernel, int cols) {
    const dim3 grid((p.n + 4 * cols - 1) / (4 * cols), unsigned((p.m + 7) / 8));
    kernel<<<grid, 128, 0, st>>>(static_cast<const T*>(p.x), p.x_stride, static_cast<const T*>(p.weight), p.weight_stride,
                                 int(p.m), p.n, p.k, e);
    note_launch();
  };
  if (p.m == 1) return run(few_rows_kernel<T, O, V, 1, 2>, 2);
  if constexpr (V == 1 || sizeof(T) == 4) {  // more aligned rows of the other types: linear_few.cu
    if (p.m == 2) return run(few_rows_kernel<T, O, V, 2, 2>, 2);
    if (p.m <= 4) return run(few_rows_kernel<T, O, V, 4, 4>, 4);
    run(few_rows_kernel<T, O, V, 8, 4>, 4);
  }
}

template <typename T, typename O>
void few_rows(const gsb_linear& p, const Epilogue& e, cudaStream_t st) {
  constexpr int E = sizeof(T);
  if (p.k % (16 / E) == 0 && vec_ok(p.x, p.x_stride, E, 16) && vec_ok(p.weight, p.weight_stride, E, 16))
    return few_rows_v<T, O, 16 / E>(p, e, st);
  few_rows_v<T, O, 1>(p, e, st);
}

// ---- operands for the tensor cores ------------------------------------------------------------

// The next multiple of 16 bytes of a row of `cols` values (float operands: of their bf16 parts).
int64_t pitch_of(int64_t cols, int dtype) {
  const int64_t per = dtype == GSB_E4M3 ? 16 : 8;
  return (cols + per - 1) / per * per;
}

bool fits_tma(const void* p, int64_t stride, int dtype) {
  const int e = dtype == GSB_E4M3 ? 1 : 2;
  return dtype != GSB_F32 && stride > 0 && vec_ok(p, stride, e, 16);
}

size_t copy_bytes(int64_t rows, int64_t cols, int dtype) {
  return size_t(rows) * size_t(pitch_of(cols, dtype)) * (dtype == GSB_F32 ? 6 : dtype == GSB_E4M3 ? 1 : 2);
}

// v as a sum of three bf16 values, each the rounding of what the ones before leave: 3 x 8 bits and
// signs hold all 24 of a float's.  A first part that would round to infinity is truncated
// instead.  Infinities and NaN go to the third part alone: it meets only the other operand's first part,
// which is 0 only where that value is, while its second and third are 0 for every value exact in bf16 (and
// infinity times 0 is NaN).  Two infinities that meet give NaN so.
struct Parts { bf16 p[3]; };
__device__ __forceinline__ Parts split3(float v) {
  Parts s;
  const bool finite = fabsf(v) <= 3.402823466e38f;
  const float f = finite ? v : 0.0f;
  s.p[0] = __float2bfloat16_rn(f);
  if (fabsf(__bfloat162float(s.p[0])) > 3.402823466e38f) s.p[0] = __float2bfloat16_rz(f);
  const float rest = f - __bfloat162float(s.p[0]);
  s.p[1] = __float2bfloat16_rn(rest);
  s.p[2] = __float2bfloat16_rn(finite ? rest - __bfloat162float(s.p[1]) : v);
  return s;
}

struct CopyJob {
  const void* in;
  int64_t stride, rows, cols, pitch;
  void* out;
};

// Rows of up to two matrices copied to a pitch that TMA takes (16-bit and 8-bit values): a warp per
// row, the unaligned reads a value per lane.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(CopyJob a, CopyJob b, int a_blocks) {
  const bool second = blockIdx.x >= a_blocks;
  const CopyJob& s = second ? b : a;
  const int64_t block = second ? blockIdx.x - a_blocks : blockIdx.x;
  const int64_t blocks = second ? gridDim.x - a_blocks : a_blocks;
  const int lane = threadIdx.x & 31;
  for (int64_t i = block * 8 + (threadIdx.x >> 5); i < s.rows; i += blocks * 8) {
    const T* in = static_cast<const T*>(s.in) + i * s.stride;
    T* out = static_cast<T*>(s.out) + i * s.pitch;
#pragma unroll 8
    for (int64_t j = lane; j < s.cols; j += 32) out[j] = in[j];
  }
}

// Two float matrices (the second may be empty) as three bf16 planes each.
__global__ void __launch_bounds__(256) split_kernel(CopyJob a, CopyJob b, int a_blocks) {
  const bool second = blockIdx.x >= a_blocks;
  const CopyJob& s = second ? b : a;
  const int64_t block = second ? blockIdx.x - a_blocks : blockIdx.x;
  const int64_t blocks = second ? gridDim.x - a_blocks : a_blocks;
  const int64_t plane = s.rows * s.pitch;
  bf16* out = static_cast<bf16*>(s.out);
  const int64_t quads = s.pitch / 4, total = s.rows * quads;
  const bool vec = (reinterpret_cast<uintptr_t>(s.in) & 15) == 0 && (s.stride & 3) == 0 && (s.cols & 3) == 0;
  for (int64_t t = block * 256 + threadIdx.x; t < total; t += blocks * 256) {
    const int64_t i = t / quads, j = (t - i * quads) * 4;
    const float* in = static_cast<const float*>(s.in) + i * s.stride + j;
    float v[4] = {};
    if (vec && j < s.cols) {
      load_f32<float, 4>(in, v);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u < s.cols) v[u] = in[u];
    }
    Vec<bf16, 4> o[3];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const Parts q = split3(v[u]);
#pragma unroll
      for (int k = 0; k < 3; ++k) o[k].v[u] = q.p[k];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<Vec<bf16, 4>*>(out + k * plane + i * s.pitch + j) = o[k];
  }
}

int copy_blocks(int64_t steps) { return int(std::min<int64_t>((steps + 255) / 256, int64_t(sm_count()) * 8)); }

CopyJob job_of(const void* in, int64_t stride, int64_t rows, int64_t cols, int dtype, void* out) {
  return {in, stride, rows, cols, pitch_of(cols, dtype), out};
}

void split(const CopyJob& a, const CopyJob& b, cudaStream_t st) {
  const int na = a.rows ? copy_blocks(a.rows * (a.pitch / 4)) : 0, nb = b.rows ? copy_blocks(b.rows * (b.pitch / 4)) : 0;
  split_kernel<<<na + nb, 256, 0, st>>>(a, b, na);
  note_launch();
}

void pack(const CopyJob& a, const CopyJob& b, int dtype, cudaStream_t st) {
  const int na = a.rows ? copy_blocks(a.rows * 32) : 0, nb = b.rows ? copy_blocks(b.rows * 32) : 0;
  if (na + nb == 0) return;
  if (dtype == GSB_E4M3) pack_kernel<uint8_t><<<na + nb, 256, 0, st>>>(a, b, na);
  else pack_kernel<uint16_t><<<na + nb, 256, 0, st>>>(a, b, na);
  note_launch();
}

// One operand as the tensor-core kernel reads it.
struct Ready {
  const void* p;
  int64_t ld, plane;
};

// Two operands at once: in place where their rows are aligned, else copied (split) to the space given.
void ready_pair(CopyJob a, CopyJob b, int dtype, Ready& ra, Ready& rb, cudaStream_t st) {
  const auto in_place = [&](CopyJob& s, Ready& r) {
    const bool fits = fits_tma(s.in, s.stride, dtype);
    r = fits ? Ready{s.in, s.stride, 0} : Ready{s.out, s.pitch, s.rows * s.pitch};
    if (fits) s.rows = 0;
  };
  in_place(a, ra);
  in_place(b, rb);
  if (dtype == GSB_F32) split(a, b, st);
  else pack(a, b, dtype, st);
}

// ---- backward: dz and the bias gradient -------------------------------------------------------

// dz = dy act'(z) rounded to the operands' type (float: its three bf16 parts), rows at `pitch`
// (dz NULL: only the sums), and per block of rows the float column sums of the unrounded dz.
// A block is 32 lanes x V columns by 8 rows; its rows' sums are added in a fixed order.
// Each thread's next two rows are on their way while it works on one (left to the compiler, the loads
// waited for the arithmetic: SiLU took 95 us at 16384 x 4096 bf16 where the bytes take 62, float
// GELU 195 us where they take 144).
template <typename T, int ACT, int V>
__global__ void __launch_bounds__(256, 4)
    dz_kernel(const T* dy, int64_t dy_stride, const typename PreactOf<T>::type* z, void* dz, int64_t pitch, float* part,
              int64_t m, int n, int64_t rows_per_part) {
  using Z = typename PreactOf<T>::type;
  constexpr bool SPLIT = sizeof(T) == 4;
  using D = typename std::conditional<SPLIT, bf16, T>::type;
  __shared__ float s_sum[8][32 * V + 1];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int j = (blockIdx.x * 32 + lane) * V;
  const int64_t lo = blockIdx.y * rows_per_part;
  const int rows = int(min(m, lo + rows_per_part) - lo);
  float s[V];
#pragma unroll
  for (int u = 0; u < V; ++u) s[u] = 0.0f;
  if (j < n) {
    const T* from = dy + (lo + g) * dy_stride + j;
    const Z* zs = z + (lo + g) * n + j;
    D* to = static_cast<D*>(dz) + (lo + g) * pitch + j;
    const int64_t dy_step = 8 * dy_stride, z_step = 8 * int64_t(n), dz_step = 8 * pitch, plane = m * pitch;
    const auto work = [&](const Vec<T, V>& d, const Vec<Z, V>& at) {
      float v[V];
#pragma unroll
      for (int u = 0; u < V; ++u) v[u] = to_f32(d.v[u]);
      if constexpr (ACT != GSB_ACT_NONE) {
        float slope[V];
#pragma unroll
        for (int u = 0; u < V; ++u) slope[u] = to_f32(at.v[u]);
        apply_slope<ACT, T, V>(slope);
#pragma unroll
        for (int u = 0; u < V; ++u) v[u] = __fmul_rn(v[u], slope[u]);
      }
#pragma unroll
      for (int u = 0; u < V; ++u) s[u] = __fadd_rn(s[u], v[u]);  // not fused: the same sum with and without dz
      if (dz) {
        if constexpr (SPLIT) {
          Vec<bf16, V> o[3];
#pragma unroll
          for (int u = 0; u < V; ++u) {
            const Parts p = split3(v[u]);
#pragma unroll
            for (int k = 0; k < 3; ++k) o[k].v[u] = p.p[k];
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) *reinterpret_cast<Vec<bf16, V>*>(to + k * plane) = o[k];
        } else {
          store_f32<T, V>(to, v);
        }
      }
      to += dz_step;
    };
    Vec<T, V> d0, d1;
    Vec<Z, V> z0, z1;
    const auto fetch = [&](Vec<T, V>& d, Vec<Z, V>& at) {
      d = read_once<T, V>(from);
      if constexpr (ACT != GSB_ACT_NONE) at = read_once<Z, V>(zs);
      from += dy_step;
      zs += z_step;
    };
    if (g < rows) fetch(d0, z0);
    if (g + 8 < rows) fetch(d1, z1);
    for (int i = g; i < rows; i += 16) {
      Vec<T, V> d = d0;
      Vec<Z, V> at = z0;
      if (i + 16 < rows) fetch(d0, z0);
      work(d, at);
      if (i + 8 >= rows) break;
      d = d1;
      at = z1;
      if (i + 24 < rows) fetch(d1, z1);
      work(d, at);
    }
  }
  if (!part) return;
#pragma unroll
  for (int u = 0; u < V; ++u) s_sum[g][u * 32 + lane] = s[u];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * V; c += 256) {
    const int jj = (blockIdx.x * 32 + (c & 31)) * V + (c >> 5);
    if (jj < n) {
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += s_sum[k][c];
      part[int64_t(blockIdx.y) * n + jj] = t;
    }
  }
}

struct DzJob {
  const void* dy;
  int64_t dy_stride;
  const void* z;
  void* dz;
  int64_t pitch;
  float* part;
  int64_t m;
  int n;
  int64_t per;
  int parts;
};

template <typename T, int ACT, int V>
void launch_dz_v(const DzJob& d, cudaStream_t st) {
  using Z = typename PreactOf<T>::type;
  dz_kernel<T, ACT, V><<<dim3((d.n + 32 * V - 1) / (32 * V), d.parts), 256, 0, st>>>(
      static_cast<const T*>(d.dy), d.dy_stride, static_cast<const Z*>(d.z), d.dz, d.pitch, d.part, d.m, d.n, d.per);
  note_launch();
}

template <typename T, int ACT>
void launch_dz(const DzJob& d, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // z and dz are this library's own, aligned whenever n is a multiple of V
  if (d.n % V == 0 && vec_ok(d.dy, d.dy_stride, sizeof(T), V * sizeof(T)) && vec_ok(d.z, 0, 1, 16))
    launch_dz_v<T, ACT, V>(d, st);
  else launch_dz_v<T, ACT, 1>(d, st);
}

template <typename T>
void launch_dz_act(int act, const DzJob& d, cudaStream_t st) {
  switch (act) {
    case GSB_ACT_RELU: return launch_dz<T, GSB_ACT_RELU>(d, st);
    case GSB_ACT_GELU: return launch_dz<T, GSB_ACT_GELU>(d, st);
    case GSB_ACT_GELU_TANH: return launch_dz<T, GSB_ACT_GELU_TANH>(d, st);
    case GSB_ACT_SILU: return launch_dz<T, GSB_ACT_SILU>(d, st);
    default: return launch_dz<T, GSB_ACT_NONE>(d, st);
  }
}

// Blocks of rows whose column sums are kept apart: enough blocks to fill the GPU eight times over,
// at least 32 rows each.
int dz_parts(int64_t m, int n, int dtype) {
  const int v = dtype == GSB_F32 ? 4 : 8;
  const int64_t across = (n + 32 * v - 1) / (32 * v);
  const int64_t want = std::max<int64_t>(1, int64_t(sm_count()) * 8 / across);
  return int(std::max<int64_t>(1, std::min<int64_t>(want, (m + 31) / 32)));
}

// ---- workspaces -------------------------------------------------------------------------------

struct FwdSpace {
  void *x, *w, *part;
  Plan plan;
  size_t bytes;
};

// The forward's product without its operands' addresses, and the backward's two.
Product fwd_shape(const gsb_linear& p) {
  Product q{};
  q.m = p.m, q.n = p.n, q.k = p.k, q.dtype = p.dtype, q.out_dtype = p.out_dtype;
  return q;
}
Product dx_shape(const gsb_linear& p) {
  Product q{};
  q.b_mn = true;
  q.m = p.m, q.n = p.k, q.k = p.n, q.dtype = p.dtype, q.out_dtype = p.dtype;
  return q;
}
Product dw_shape(const gsb_linear& p) {
  Product q{};
  q.a_mn = q.b_mn = true;
  q.m = p.n, q.n = p.k, q.k = p.m, q.dtype = p.dtype, q.out_dtype = p.dtype;
  return q;
}

FwdSpace fwd_space(const gsb_linear& p, void* ws, size_t cap) {
  Carver c(ws, cap);
  FwdSpace s{};
  if (path_of(p) == Path::kTiles) {
    if (!fits_tma(p.x, p.x_stride, p.dtype)) s.x = c.take<char>(copy_bytes(p.m, p.k, p.dtype));
    if (!fits_tma(p.weight, p.weight_stride, p.dtype)) s.w = c.take<char>(copy_bytes(p.n, p.k, p.dtype));
    const Product q = fwd_shape(p);
    s.plan = plan_product(q);
    if (const size_t sums = partial_bytes(&q, 1, s.plan)) s.part = c.take<char>(sums);
  }
  s.bytes = c.used;
  return s;
}

struct BwdSpace {
  void *dz, *x, *w, *sums;  // sums: of products in pieces
  float* part;
  Plan dx, dw, pair;
  bool together;  // both products in one launch
  size_t bytes;
};

bool keeps_dy(const gsb_linear& p, const void* dy, int64_t dy_stride) {
  return p.activation == GSB_ACT_NONE && fits_tma(dy, dy_stride, p.dtype);
}

BwdSpace bwd_space(const gsb_linear& p, const void* dy, int64_t dy_stride, void* ws, size_t cap) {
  Carver c(ws, cap);
  BwdSpace s{};
  s.part = c.take<float>(size_t(dz_parts(p.m, p.n, p.dtype)) * p.n);
  if (!keeps_dy(p, dy, dy_stride)) s.dz = c.take<char>(copy_bytes(p.m, p.n, p.dtype));
  if (!fits_tma(p.x, p.x_stride, p.dtype)) s.x = c.take<char>(copy_bytes(p.m, p.k, p.dtype));
  if (!fits_tma(p.weight, p.weight_stride, p.dtype)) s.w = c.take<char>(copy_bytes(p.n, p.k, p.dtype));
  const Product two[2] = {dx_shape(p), dw_shape(p)};
  s.dx = plan_product(two[0]);
  s.dw = plan_product(two[1]);
  s.pair = plan_pair(two);
  s.together = s.pair.cost < s.dx.cost + s.dw.cost;
  // for either gradient alone too: which are wanted is not known here
  const size_t sums = std::max({partial_bytes(two, 1, s.dx), partial_bytes(two + 1, 1, s.dw),
                                s.together ? partial_bytes(two, 2, s.pair) : 0});
  if (sums) s.sums = c.take<char>(sums);
  s.bytes = c.used;
  return s;
}

Epilogue plain_output(void* out, int64_t cols, int dtype) {
  Epilogue e{};
  e.out = out;
  e.out_stride = cols;
  const int b = elem_bytes(dtype);
  e.vec = cols % (16 / b) == 0 && vec_ok(out, cols, b, 16);
  return e;
}

gsb_status bwd(const gsb_linear& p, const void* z, const void* dy, int64_t dy_stride, void* dx, void* dw, void* db,
               const BwdSpace& s, cudaStream_t st) {
  const bool keep = keeps_dy(p, dy, dy_stride);
  const bool products = dx || dw;
  const int64_t pitch = keep ? dy_stride : pitch_of(p.n, p.dtype);
  DzJob d{dy, dy_stride, z, keep || !products ? nullptr : s.dz, pitch, db ? s.part : nullptr, p.m, p.n, 0, 0};
  d.parts = dz_parts(p.m, p.n, p.dtype);
  d.per = (p.m + d.parts - 1) / d.parts;
  d.parts = int((p.m + d.per - 1) / d.per);
  if (d.dz || db) {
    switch (p.dtype) {
      case GSB_F32: launch_dz_act<float>(p.activation, d, st); break;
      case GSB_BF16: launch_dz_act<bf16>(p.activation, d, st); break;
      default: launch_dz_act<f16>(p.activation, d, st); break;
    }
  }
  if (db) {
    const int blocks = (p.n + 31) / 32;
    switch (p.dtype) {
      case GSB_F32: column_sum_kernel<float><<<blocks, 256, 0, st>>>(s.part, d.parts, p.n, static_cast<float*>(db)); break;
      case GSB_BF16: column_sum_kernel<bf16><<<blocks, 256, 0, st>>>(s.part, d.parts, p.n, static_cast<bf16*>(db)); break;
      default: column_sum_kernel<f16><<<blocks, 256, 0, st>>>(s.part, d.parts, p.n, static_cast<f16*>(db)); break;
    }
    note_launch();
  }
  if (!products) return launch_status();
  const Ready g = keep ? Ready{dy, dy_stride, 0} : Ready{s.dz, pitch, p.m * pitch};
  CopyJob jx = job_of(p.x, p.x_stride, dw ? p.m : 0, p.k, p.dtype, s.x);
  CopyJob jw = job_of(p.weight, p.weight_stride, dx ? p.n : 0, p.k, p.dtype, s.w);
  Ready x, w;
  ready_pair(jx, jw, p.dtype, x, w, st);
  gsb_status status = launch_status();
  Product p2[2] = {dx_shape(p), dw_shape(p)};
  p2[0].a = p2[1].a = g.p;
  p2[0].a_ld = p2[1].a_ld = g.ld;
  p2[0].a_plane = p2[1].a_plane = g.plane;
  p2[0].b = w.p, p2[0].b_ld = w.ld, p2[0].b_plane = w.plane;
  p2[1].b = x.p, p2[1].b_ld = x.ld, p2[1].b_plane = x.plane;
  const Epilogue e2[2] = {plain_output(dx, p.k, p.dtype), plain_output(dw, p.k, p.dtype)};
  if (dx && dw && s.together) return status == GSB_OK ? mma_products(p2, e2, 2, s.pair, s.sums, st) : status;
  if (dx && status == GSB_OK) status = mma_products(p2, e2, 1, s.dx, s.sums, st);
  if (dw && status == GSB_OK) status = mma_products(p2 + 1, e2 + 1, 1, s.dw, s.sums, st);
  return status;
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

// Workspaces hold rows that TMA and 16-byte accesses read and write.
bool aligned16(const void* ws) { return reinterpret_cast<uintptr_t>(ws) % 16 == 0; }

gsb_status check_operands(const gsb_linear* p) {
  if (!p->weight || (p->m > 0 && !p->x)) return GSB_ERR_ARG;
  if (p->dtype == GSB_E4M3 && p->m > 0 && (!p->x_scale || !p->weight_scale)) return GSB_ERR_ARG;
  return GSB_OK;
}

}  // namespace

size_t linear_fwd_workspace(const gsb_linear* p) {
  if (check_linear(p) != GSB_OK) return 0;
  return fwd_space(*p, nullptr, 0).bytes;
}

gsb_status linear_fwd(const gsb_linear* p, void* y, void* preact, void* ws, size_t ws_bytes, cudaStream_t st) {
  if (gsb_status s = check_linear(p); s != GSB_OK) return s;
  if (gsb_status s = check_operands(p); s != GSB_OK) return s;
  if (p->dtype == GSB_E4M3 && preact) return GSB_ERR_ARG;
  if (p->m == 0) return GSB_OK;
  if (!y) return GSB_ERR_ARG;
  Epilogue e = plain_output(y, p->n, p->out_dtype);
  if (p->dtype == GSB_E4M3) {
    e.row_scale = p->x_scale;
    e.col_scale = p->weight_scale;
  }
  e.bias = p->bias;
  e.res = p->residual;
  e.res_stride = p->residual_stride;
  e.preact = preact;
  e.act = p->activation;
  const int b = elem_bytes(p->out_dtype);
  e.vec = e.vec && vec_ok(p->bias, 0, b, 16) && vec_ok(preact, 0, b, 16) &&
          (!p->residual || vec_ok(p->residual, p->residual_stride, b, 16));
  const Path path = path_of(*p);
  if (path == Path::kFewMma) {
    few_rows_mma(*p, e, st);
    return launch_status();
  }
  if (path == Path::kWalk) {
    switch (p->dtype) {
      case GSB_F32: few_rows<float, float>(*p, e, st); break;
      case GSB_BF16: few_rows<bf16, bf16>(*p, e, st); break;
      case GSB_F16: few_rows<f16, f16>(*p, e, st); break;
      default:
        if (p->out_dtype == GSB_F32) few_rows<e4m3, float>(*p, e, st);
        else if (p->out_dtype == GSB_BF16) few_rows<e4m3, bf16>(*p, e, st);
        else few_rows<e4m3, f16>(*p, e, st);
    }
    return launch_status();
  }
  const FwdSpace s = fwd_space(*p, ws, ws_bytes);
  if (s.bytes && (!ws || ws_bytes < s.bytes)) return GSB_ERR_WORKSPACE;
  if (s.bytes && !aligned16(ws)) return GSB_ERR_ARG;
  Ready x, w;
  ready_pair(job_of(p->x, p->x_stride, p->m, p->k, p->dtype, s.x),
             job_of(p->weight, p->weight_stride, p->n, p->k, p->dtype, s.w), p->dtype, x, w, st);
  if (gsb_status q = launch_status(); q != GSB_OK) return q;
  Product q = fwd_shape(*p);
  q.a = x.p, q.a_ld = x.ld, q.a_plane = x.plane;
  q.b = w.p, q.b_ld = w.ld, q.b_plane = w.plane;
  return mma_products(&q, &e, 1, s.plan, s.part, st);
}

size_t linear_bwd_workspace(const gsb_linear* p, const void* dy, int64_t dy_stride) {
  if (check_linear(p) != GSB_OK) return 0;
  return bwd_space(*p, dy, dy_stride, nullptr, 0).bytes;
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
  if (!ws || ws_bytes < linear_bwd_workspace(p, dy, dy_stride)) return GSB_ERR_WORKSPACE;
  if (!aligned16(ws)) return GSB_ERR_ARG;
  return bwd(*p, preact, dy, dy_stride, dx, dweight, dbias, bwd_space(*p, dy, dy_stride, ws, ws_bytes), st);
}

gsb_status token_status() {
  int gave_up = 0;
  if (gsb_status s = gave_up_status(&gave_up); s != GSB_OK) return s;
  return gave_up ? GSB_ERR_TIMEOUT : GSB_OK;
}

}  // namespace gsb
