// y = act(x w^T + b) + r for a handful of rows (up to 32) of 16-bit or e4m3 values.
//
// Bound by the weights' bytes, and by latency: 16 rows through 8,192 x 2,048 e4m3 weights are 2.6 us of
// HBM.  A tcgen05 tile spends about 128 cycles per MMA on its 128 rows whatever few of them are live
// and cannot start before its ring, barriers and TMEM are set up: 12.0 us there, 6.4 here.  A warp reads the
// weights into registers as the fragments of the warp-wide MMA (m16n8k16) want them and the eight
// warps of a block share K, so that a block's loads are all on their way at once.
//
// Fragments without a shuffle: the MMA sums over 16 k in any order as long as both operands agree, so
// lane l takes 16 adjacent bytes of row l / 4 of either operand and the MMA's k slots (2 (l % 4) + {0, 1},
// + 8) are read as the lane's own values: its first two 32-bit words for one MMA, the next two for
// another.  e4m3 becomes fp16 on the way, exactly.
#include "linear_parts.cuh"

namespace gsb {

namespace {

constexpr int kWarps = 8;
constexpr int kBatch = 4;  // steps whose loads are in flight together

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1, bf16*) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1, f16*) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes as 16-bit pairs: as they are, or eight words of fp16 from 16 e4m3 codes.
template <typename T>
struct Words {
  static constexpr int kCount = sizeof(T) == 1 ? 8 : 4;
  uint32_t w[kCount];
  __device__ __forceinline__ explicit Words(uint4 v) {
    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 1) {
        asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\ncvt.rn.f16x2.e4m3x2 %1, hi;\n}"
            : "=r"(w[2 * i]), "=r"(w[2 * i + 1])
            : "r"(in[i]));
      } else {
        w[i] = in[i];
      }
    }
  }
};

template <typename T> struct MmaType { using type = T; };
template <> struct MmaType<e4m3> { using type = f16; };

// MB blocks of 16 rows by C blocks of 8 columns.
template <typename T, typename O, int MB, int C>
__global__ void __launch_bounds__(32 * kWarps) few_mma_kernel(const T* x, int64_t x_stride, const T* w, int64_t w_stride,
                                                             int m, int n, int k, Epilogue e) {
  constexpr int V = 16 / sizeof(T);  // values per lane and step
  using M = typename MmaType<T>::type;
  __shared__ float part[kWarps][16 * MB][8 * C + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j0 = blockIdx.x * 8 * C;
  const int sub = (lane & 3) * V;  // this lane's k within a step
  const T* wr[C];
  const T* xr[MB][2];
#pragma unroll
  for (int c = 0; c < C; ++c) wr[c] = w + int64_t(min(j0 + c * 8 + (lane >> 2), n - 1)) * w_stride;
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) xr[b][h] = x + int64_t(min(b * 16 + h * 8 + (lane >> 2), m - 1)) * x_stride;
  float acc[MB][C][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int k0 = warp * 4 * V; k0 < k; k0 += kBatch * kWarps * 4 * V) {
    uint4 wv[kBatch][C], xv[kBatch][MB][2];
#pragma unroll
    for (int s = 0; s < kBatch; ++s) {
      const int at = k0 + s * kWarps * 4 * V + sub;
      const bool in = at < k;  // k is a multiple of V
#pragma unroll
      for (int c = 0; c < C; ++c) wv[s][c] = in ? __ldcs(reinterpret_cast<const uint4*>(wr[c] + at)) : zero;
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) xv[s][b][h] = in ? *reinterpret_cast<const uint4*>(xr[b][h] + at) : zero;
    }
#pragma unroll
    for (int s = 0; s < kBatch; ++s) {
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        const Words<T> lo(xv[s][b][0]), hi(xv[s][b][1]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const Words<T> bw(wv[s][c]);
#pragma unroll
          for (int q = 0; q < Words<T>::kCount; q += 2)
            mma16(acc[b][c], lo.w[q], hi.w[q], lo.w[q + 1], hi.w[q + 1], bw.w[q], bw.w[q + 1],
                  static_cast<M*>(nullptr));
        }
      }
    }
  }
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        part[warp][b * 16 + (lane >> 2) + 8 * (q >> 1)][c * 8 + (lane & 3) * 2 + (q & 1)] = acc[b][c][q];
  __syncthreads();
  for (int t = threadIdx.x; t < 16 * MB * 8 * C; t += 32 * kWarps) {
    const int r = t / (8 * C), c = t % (8 * C);
    if (r >= m || j0 + c >= n) continue;
    float z[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < kWarps; ++v) z[0] += part[v][r][c];
    finish<O, 1>(e, n, r, j0 + c, z);
  }
}

template <typename T, typename O>
void launch(const gsb_linear& p, const Epilogue& e, cudaStream_t st) {
  const auto run = [&](auto kernel, int cols) {
    kernel<<<(p.n + cols - 1) / cols, 32 * kWarps, 0, st>>>(static_cast<const T*>(p.x), p.x_stride,
                                                           static_cast<const T*>(p.weight), p.weight_stride, int(p.m),
                                                           p.n, p.k, e);
    note_launch();
  };
  // 32 columns per block read the rows' values once for four blocks of weights; where that leaves SMs
  // without a block, 8
  if (p.m > 16) return run(few_mma_kernel<T, O, 2, 1>, 8);
  if (p.n >= 32 * sm_count()) return run(few_mma_kernel<T, O, 1, 4>, 32);
  run(few_mma_kernel<T, O, 1, 1>, 8);
}

}  // namespace

bool few_rows_mma_serves(const gsb_linear& p) {
  const int b = elem_bytes(p.dtype);
  if (p.dtype == GSB_F32 || p.k % (16 / b) != 0 || !vec_ok(p.x, p.x_stride, b, 16) ||
      !vec_ok(p.weight, p.weight_stride, b, 16))
    return false;
  // from 2 rows (2,048 x 8,192 e4m3: 6.0 us, 8.4 one row after the other); 17 to 32 rows: their values'
  // way through L1 outweighs the weights' once those are large (1,024 x 1,024 bf16: 3.7 us here, 9.3 on
  // tcgen05 tiles; 2,048 x 8,192: 16.0 and 14.8)
  return p.m >= 2 && p.m <= (int64_t(p.n) * p.k * b <= (8 << 20) ? 32 : 16);
}

void few_rows_mma(const gsb_linear& p, const Epilogue& e, cudaStream_t st) {
  switch (p.dtype) {
    case GSB_BF16: launch<bf16, bf16>(p, e, st); break;
    case GSB_F16: launch<f16, f16>(p, e, st); break;
    default:
      if (p.out_dtype == GSB_F32) launch<e4m3, float>(p, e, st);
      else if (p.out_dtype == GSB_BF16) launch<e4m3, bf16>(p, e, st);
      else launch<e4m3, f16>(p, e, st);
  }
}

}  // namespace gsb
