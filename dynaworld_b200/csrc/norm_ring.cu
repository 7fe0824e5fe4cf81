// The norm over many rows: every SM keeps one block, whose rows come in through a ring of
// asynchronous copies (cp.async.bulk of whole rows, one barrier per slot).
//
// The kernels of norm.cu load a row, wait, reduce, store; with 92 registers a thread only 16 warps
// fit an SM and their loads pause while they reduce.  Here a warp owns a row and up to 200 KB of rows
// are on their way to each SM whatever the warps do.  Norm of 16,384 x 1,024 bf16 values with a
// residual: 32.5 -> 20.1 us (6.7 TB/s), its backward 37 -> 34 us though it reads a fifth more
// (4.9 TB/s); e4m3 norm of 65,536 x 2,048: 234 -> 146 us (6.4 TB/s).
#include "async_copy.cuh"
#include "norm_parts.cuh"

#include <atomic>

namespace gsb {

namespace {

constexpr int kBudget = 200 * 1024;  // bytes of row slots per block
constexpr int kMaxSlots = 6;
constexpr int kBarBytes = 1024;      // barriers at the front of the shared memory: 16 groups x 6 slots

// A warp's walk over its rows.  Slot s holds `streams` rows of `bytes` bytes one after the other.
template <int THREADS>
struct Ring {
  static constexpr int kGroups = THREADS / 32;
  uint32_t bars, data;
  const uint8_t* smem;
  int slots, streams;
  uint32_t bytes;
  int* gave_up;
  bool ok;

  __device__ __forceinline__ void init(uint8_t* raw, int slots_, int streams_, uint32_t bytes_, int* flag) {
    const int g = threadIdx.x / 32;
    slots = slots_;
    streams = streams_;
    bytes = bytes_;
    gave_up = flag;
    ok = true;
    bars = smem_addr(raw) + g * kMaxSlots * 8;
    smem = raw + kBarBytes + size_t(g) * slots * streams * bytes;
    data = smem_addr(smem);
    if (threadIdx.x % 32 == 0)
      for (int s = 0; s < slots; ++s) bar_init(bars + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
  }
  __device__ __forceinline__ void expect(int s) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bars + 8 * s), "r"(streams * bytes)
                 : "memory");
  }
  __device__ __forceinline__ void load(int s, int q, const void* src) {
    bulk_load(data + (s * streams + q) * bytes, src, bytes, bars + 8 * s);
  }
  __device__ __forceinline__ void wait(int s, uint32_t parity) {
    if (ok) ok = bar_wait(bars + 8 * s, parity, gave_up);
  }
  template <typename T, int V>
  __device__ __forceinline__ const Vec<T, V>* row(int s, int q) const {
    return reinterpret_cast<const Vec<T, V>*>(smem + (s * streams + q) * size_t(bytes));
  }
};

struct RingArgs {
  NormArgs a;
  int slots;
  int* gave_up;
};

template <typename T, int PV, int THREADS, int MODE>
__global__ void __launch_bounds__(THREADS, 1) ring_fwd_kernel(const __grid_constant__ RingArgs ra) {
  constexpr int V = 16 / sizeof(T);
  const NormArgs& a = ra.a;
  extern __shared__ __align__(128) uint8_t raw[];
  using R = Ring<THREADS>;
  constexpr int GROUP = 32;
  const int t = threadIdx.x % GROUP, g = threadIdx.x / GROUP;
  const int nv = a.dim / V;
  const bool has_res = MODE != kQuantize && a.res;
  R ring;
  ring.init(raw, ra.slots, has_res ? 2 : 1, a.dim * uint32_t(sizeof(T)), ra.gave_up);
  const int64_t first = int64_t(blockIdx.x) * R::kGroups + g, step = int64_t(gridDim.x) * R::kGroups;
  const auto fetch = [&](int64_t row, int s) {
    ring.expect(s);
    ring.load(s, 0, static_cast<const T*>(a.x) + row * a.x_stride);
    if (has_res) ring.load(s, 1, static_cast<const T*>(a.res) + row * a.res_stride);
  };
  if (t == 0)
    for (int s = 0; s < ra.slots; ++s)
      if (first + s * step < a.rows) fetch(first + s * step, s);
  Vec<T, V> w[PV];
  if constexpr (MODE != kQuantize) {
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) w[j] = reinterpret_cast<const Vec<T, V>*>(a.w)[j * GROUP + t];
  }
  int s = 0;
  uint32_t parity = 0;
  for (int64_t row = first; row < a.rows; row += step) {
    ring.wait(s, parity);
    float h[PV][V];
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const int i = j * GROUP + t;
      if (i < nv) {
        const Vec<T, V> v = ring.template row<T, V>(s, 0)[i];
#pragma unroll
        for (int e = 0; e < V; ++e) h[j][e] = to_f32(v.v[e]);
        if (has_res) {
          const Vec<T, V> r = ring.template row<T, V>(s, 1)[i];
#pragma unroll
          for (int e = 0; e < V; ++e) h[j][e] += to_f32(r.v[e]);
        }
        if (!ring.ok) {
#pragma unroll
          for (int e = 0; e < V; ++e) h[j][e] = __int_as_float(0x7fc00000);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) h[j][e] = 0.0f;
      }
    }
    __syncwarp();  // every lane has read the slot
    if (t == 0 && ring.ok && row + ra.slots * step < a.rows) fetch(row + ra.slots * step, s);
    if (++s == ra.slots) s = 0, parity ^= 1;
    if constexpr (MODE != kQuantize) {
      if (has_res && a.sum) {
#pragma unroll
        for (int j = 0; j < PV; ++j)
          if (j * GROUP + t < nv) store_f32<T, V>(static_cast<T*>(a.sum) + row * a.dim + int64_t(j * GROUP + t) * V, h[j]);
      }
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < PV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fmaf(h[j][e], h[j][e], ss);
      ss = warp_sum(ss);
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
      top = __reduce_max_sync(0xffffffffu, top);
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
  if (!ring.ok) let_copies_land();
}

template <typename T, int PV, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) ring_bwd_kernel(const __grid_constant__ RingArgs ra) {
  constexpr int V = 16 / sizeof(T);
  const NormArgs& a = ra.a;
  extern __shared__ __align__(128) uint8_t raw[];
  using R = Ring<THREADS>;
  constexpr int GROUP = 32;
  const int t = threadIdx.x % GROUP, g = threadIdx.x / GROUP;
  const int nv = a.dim / V;
  const int q_res = 2, q_ds = a.res ? 3 : 2;
  R ring;
  ring.init(raw, ra.slots, 2 + (a.res != nullptr) + (a.dsum != nullptr), a.dim * uint32_t(sizeof(T)), ra.gave_up);
  const int64_t first = int64_t(blockIdx.x) * R::kGroups + g, step = int64_t(gridDim.x) * R::kGroups;
  const auto fetch = [&](int64_t row, int s) {
    ring.expect(s);
    ring.load(s, 0, static_cast<const T*>(a.x) + row * a.x_stride);
    ring.load(s, 1, static_cast<const T*>(a.dy) + row * a.dy_stride);
    if (a.res) ring.load(s, q_res, static_cast<const T*>(a.res) + row * a.res_stride);
    if (a.dsum) ring.load(s, q_ds, static_cast<const T*>(a.dsum) + row * a.dsum_stride);
  };
  if (t == 0)
    for (int s = 0; s < ra.slots; ++s)
      if (first + s * step < a.rows) fetch(first + s * step, s);
  Vec<T, V> w[PV];
  float acc[PV][V];
#pragma unroll
  for (int j = 0; j < PV; ++j) {
    if (j * GROUP + t < nv) w[j] = reinterpret_cast<const Vec<T, V>*>(a.w)[j * GROUP + t];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[j][e] = 0.0f;
  }
  int s = 0;
  uint32_t parity = 0;
  for (int64_t row = first; row < a.rows; row += step) {
    const float rstd = a.rstd[row];
    ring.wait(s, parity);
    float h[PV][V], gr[PV][V];
    Vec<T, V> ds[PV];
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const int i = j * GROUP + t;
      if (i < nv) {
        const Vec<T, V> v = ring.template row<T, V>(s, 0)[i], u = ring.template row<T, V>(s, 1)[i];
#pragma unroll
        for (int e = 0; e < V; ++e) h[j][e] = to_f32(v.v[e]), gr[j][e] = to_f32(u.v[e]);
        if (a.res) {
          const Vec<T, V> r = ring.template row<T, V>(s, q_res)[i];
#pragma unroll
          for (int e = 0; e < V; ++e) h[j][e] += to_f32(r.v[e]);
        }
        if (a.dsum) ds[j] = ring.template row<T, V>(s, q_ds)[i];
        if (!ring.ok) {
#pragma unroll
          for (int e = 0; e < V; ++e) h[j][e] = __int_as_float(0x7fc00000);
        }
      }
    }
    __syncwarp();  // every lane has read the slot
    if (t == 0 && ring.ok && row + ra.slots * step < a.rows) fetch(row + ra.slots * step, s);
    if (++s == ra.slots) s = 0, parity ^= 1;
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float gh = gr[j][e] * h[j][e];
          dot = fmaf(gh, to_f32(w[j].v[e]), dot);
          acc[j][e] = fmaf(gh, rstd, acc[j][e]);
        }
      }
    dot = warp_sum(dot);
    const float c = rstd * rstd * (dot * a.inv_dim);
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      const int i = j * GROUP + t;
      if (i < nv) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          o[e] = rstd * (gr[j][e] * to_f32(w[j].v[e]) - h[j][e] * c);
          if (a.dsum) o[e] += to_f32(ds[j].v[e]);
        }
        store_f32<T, V>(static_cast<T*>(a.dx) + row * a.dim + int64_t(i) * V, o);
      }
    }
  }
  if (!ring.ok) let_copies_land();
  // the block's column sums, its groups added in order; the slots are free once every row is read
  float* part = a.dw_part + int64_t(blockIdx.x) * a.dim;
  {
    __syncthreads();
    float* s_dw = reinterpret_cast<float*>(raw + kBarBytes);
#pragma unroll
    for (int j = 0; j < PV; ++j)
      if (j * GROUP + t < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) s_dw[g * a.dim + (j * GROUP + t) * V + e] = acc[j][e];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < a.dim; i += THREADS) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < R::kGroups; ++k) v += s_dw[k * a.dim + i];
      part[i] = v;
    }
  }
}

template <typename K>
bool start(K kernel, const NormArgs& a, int groups, int threads, int streams, int elem, int slots, int blocks,
           std::atomic<uint64_t>& ready, cudaStream_t st) {
  RingArgs ra{a, slots, gave_up_flag()};
  if (!ra.gave_up) return false;
  int dev = 0;
  (void)cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBarBytes + kBudget) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const size_t bytes = kBarBytes + size_t(groups) * slots * streams * a.dim * elem;
  kernel<<<blocks, threads, bytes, st>>>(ra);
  note_launch();
  return true;
}

int slots_of(int groups, int streams, int row_bytes) {
  return std::min(kMaxSlots, kBudget / (groups * streams * row_bytes));
}

template <typename T, int MODE>
bool fwd_of(const NormArgs& a, cudaStream_t st) {
  constexpr int E = sizeof(T), V = 16 / E;
  const int nv = a.dim / V, row = a.dim * E, streams = MODE != kQuantize && a.res ? 2 : 1;
  // per instance: the devices whose copy of the kernel has its shared memory
  const auto go = [&](auto kernel, int groups, int threads, std::atomic<uint64_t>& ready) {
    const int slots = slots_of(groups, streams, row);
    const int64_t blocks = std::min<int64_t>(sm_count(), (a.rows + groups - 1) / groups);
    return slots >= 2 && start(kernel, a, groups, threads, streams, E, slots, int(blocks), ready, st);
  };
  static std::atomic<uint64_t> ready[3];
  if (nv <= 64) return go(ring_fwd_kernel<T, 2, 512, MODE>, 16, 512, ready[0]);
  if (nv <= 128) return go(ring_fwd_kernel<T, 4, 512, MODE>, 16, 512, ready[1]);
  return go(ring_fwd_kernel<T, 8, 384, MODE>, 12, 384, ready[2]);  // eight warps with a slot more: 172 us instead of 146
}

template <typename T>
bool bwd_of(const NormArgs& a, int* parts, cudaStream_t st) {
  constexpr int E = sizeof(T), V = 16 / E;
  const int nv = a.dim / V, row = a.dim * E, streams = 2 + (a.res != nullptr) + (a.dsum != nullptr);
  const auto go = [&](auto kernel, int groups, std::atomic<uint64_t>& ready) {
    const int slots = slots_of(groups, streams, row);
    const int64_t blocks = std::min<int64_t>(sm_count(), (a.rows + groups - 1) / groups);
    *parts = int(blocks);
    return slots >= 2 && start(kernel, a, groups, 256, streams, E, slots, int(blocks), ready, st);
  };
  static std::atomic<uint64_t> ready[2];
  if (nv <= 64) return go(ring_bwd_kernel<T, 2, 256>, 8, ready[0]);
  return go(ring_bwd_kernel<T, 4, 256>, 8, ready[1]);
}

// A ring pays once every warp walks a few rows (below that the register kernels' single round is
// shorter), a row is worth a copy of its own and a warp's registers hold it (a block per row, with one
// ring per SM, took 31 us for the 13 us of norm.cu's blocks: 8,192 x 2,048 floats quantised).
bool worth_it(const NormArgs& a, int elem, int most_vectors) {
  const int nv = a.dim * elem / 16;
  return a.dim * elem >= 512 && nv <= most_vectors && a.rows >= int64_t(sm_count()) * 32;
}

}  // namespace

bool ring_fwd(const NormArgs& a, int dtype, int mode, cudaStream_t st) {
  if (!worth_it(a, elem_bytes(dtype), 256)) return false;
  const auto of = [&](auto value) {
    using T = decltype(value);
    if (mode == kNorm) return fwd_of<T, kNorm>(a, st);
    if (mode == kNormFp8) return fwd_of<T, kNormFp8>(a, st);
    return fwd_of<T, kQuantize>(a, st);
  };
  if (dtype == GSB_F32) return of(float{});
  if (dtype == GSB_BF16) return of(bf16{});
  return of(f16{});
}

bool ring_bwd(const NormArgs& a, int dtype, int* parts, cudaStream_t st) {
  if (!worth_it(a, elem_bytes(dtype), 128)) return false;
  if (dtype == GSB_F32) return bwd_of<float>(a, parts, st);
  if (dtype == GSB_BF16) return bwd_of<bf16>(a, parts, st);
  return bwd_of<f16>(a, parts, st);
}

}  // namespace gsb
