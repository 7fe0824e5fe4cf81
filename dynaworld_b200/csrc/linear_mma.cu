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
  // every stream: the copy waits for the legacy default stream only, and torch's are non-blocking ones
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(gave_up, g_gave_up, sizeof(int)) != cudaSuccess) {
    (void)cudaGetLastError();
    return GSB_ERR_CUDA;
  }
  const int none = 0;  // reported once
  if (*gave_up && cudaMemcpyToSymbol(g_gave_up, &none, sizeof(int)) != cudaSuccess) {
    (void)cudaGetLastError();
    return GSB_ERR_CUDA;
  }
  return GSB_OK;
}

// One thread waits, as the kernels do, on a barrier that nothing completes.
static __global__ void timeout_probe_kernel(uint64_t limit_ns, int* gave_up) {
  __shared__ __align__(8) uint64_t bar;
  bar_init(smem_addr(&bar), 1);
  (void)bar_wait(smem_addr(&bar), 0, gave_up, limit_ns);
}

gsb_status token_timeout_probe(uint32_t limit_us, cudaStream_t st) {
  int* flag = gave_up_flag();
  if (!flag) return GSB_ERR_CUDA;
  timeout_probe_kernel<<<1, 1, 0, st>>>(uint64_t(std::min<uint32_t>(limit_us, 1000000)) * 1000, flag);
  return launch_status();
}

// ---- plans ------------------------------------------------------------------------------------
//
// Costs in units of one 64-element block of K of a 256 x 256 tile (about 0.27 us).
// A launch ends with one exposed epilogue (about 2 us, less for narrower tiles); pieces along K
// cost a second kernel (about 4 us) and their sums' way through L2.
constexpr float kReduce = 14.0f;
constexpr float kPartialPerMB = 1.0f;  // written and read once

struct Walk {
  int bn;
  int rows;     // of a tile
  float block, tail;
};

// What a block of K of each tile costs.  An MMA takes about 128 cycles whether its B has 64 columns or
// 256 (A's 128 rows have to be read for each; 8192 x 4096 x 4096 bf16 took 195 us in 256-wide tiles
// and 351 us in 128-wide ones), so narrow tiles only serve to fill the GPU and to end sooner.
static const Walk kWalks[3] = {{256, 256, 1.0f, 8.0f}, {128, 128, 0.95f, 4.0f}, {64, 128, 0.9f, 2.5f}};
constexpr float kFloatBlock = 6.0f;  // six products

static float block_cost(const Product& p, const Walk& w) { return p.dtype == GSB_F32 ? kFloatBlock * w.block : w.block; }
static int64_t workers_of(const Walk& w) { return w.rows == 256 ? sm_count() / 2 : sm_count(); }

static int64_t tiles_of(const Product& p, const Walk& w) {
  return ((p.m + w.rows - 1) / w.rows) * ((p.n + w.bn - 1) / w.bn);
}

// The second kernel and its sums' traffic.
static float reduce_cost(const Product& p, int splits) {
  return kReduce + kPartialPerMB * float(splits) * float(p.m) * float(p.n) * 4e-6f;
}

static bool may_split(const Product& p, int splits, int64_t tiles, int64_t clusters) {
  return splits == 1 || (k_blocks_of(p) >= 4 * splits && tiles * splits <= 2 * clusters);
}

Plan plan_product(const Product& p) {
  Plan best{0, {1, 1}, 0.0f};
  for (const Walk& w : kWalks) {
    const int64_t workers = workers_of(w), tiles = tiles_of(p, w);
    for (int s = 1; s <= 16 && may_split(p, s, tiles, workers); s *= 2) {
      const int64_t rounds = (tiles * s + workers - 1) / workers;
      float cost = float(rounds) * float(piece_of(p, s)) * block_cost(p, w) + w.tail;
      if (s > 1) cost += reduce_cost(p, s);
      if (best.bn == 0 || cost < best.cost) best = {w.bn, {s, 1}, cost};
    }
  }
  return best;
}

// Whether a product of the launch leaves float sums: its own pieces, or, where the output is not float,
// the other's (one kernel writes both).
static bool leaves_sums(const Product* p, int count, const Plan& plan, int i) {
  if (plan.splits[i] > 1) return true;
  return count == 2 && plan.splits[1 - i] > 1 && p[i].out_dtype != GSB_F32;
}

Plan plan_pair(const Product (&p)[2]) {
  Plan best{0, {1, 1}, 0.0f};
  for (const Walk& w : kWalks) {
    const int64_t workers = workers_of(w), t0 = tiles_of(p[0], w), t1 = tiles_of(p[1], w);
    for (int s0 = 1; s0 <= 16 && may_split(p[0], s0, t0, workers); s0 *= 2)
      for (int s1 = 1; s1 <= 16 && may_split(p[1], s1, t1, workers); s1 *= 2) {
        const Plan plan{w.bn, {s0, s1}, 0.0f};
        const float a = float(piece_of(p[0], s0)) * block_cost(p[0], w), b = float(piece_of(p[1], s1)) * block_cost(p[1], w);
        const float all = (float(t0 * s0) * a + float(t1 * s1) * b) / float(workers);
        // an even share, at least the longer piece, and half of the shorter one lost at the end
        float cost = std::max(all + 0.5f * std::min(a, b), std::max(a, b)) + w.tail;
        for (int k = 0; k < 2; ++k)
          if (leaves_sums(p, 2, plan, k)) cost += reduce_cost(p[k], plan.splits[k]);
        if (best.bn == 0 || cost < best.cost) best = {w.bn, {s0, s1}, cost};
      }
  }
  return best;
}

size_t partial_bytes(const Product* p, int count, const Plan& plan) {
  size_t n = 0;
  for (int i = 0; i < count; ++i)
    if (leaves_sums(p, count, plan, i)) n += align_up(size_t(plan.splits[i]) * size_t(p[i].m) * size_t(p[i].n) * 4);
  return n;
}

// ---- the sums of a product's pieces, finished --------------------------------------------------

template <typename O, int V>
static __global__ void __launch_bounds__(256) add_parts_kernel(const float* part, int splits, int64_t m, int64_t n,
                                                              Epilogue e) {
  const int64_t per_row = n / V, total = m * per_row, plane = m * n;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < total; t += int64_t(gridDim.x) * 256) {
    const int64_t i = t / per_row, j = (t - i * per_row) * V;
    const float* p = part + i * n + j;
    float z[V];
#pragma unroll
    for (int u = 0; u < V; ++u) z[u] = 0.0f;
    for (int s = 0; s < splits; ++s) {
      if constexpr (V > 1) {
#pragma unroll
        for (int u = 0; u < V; u += 4) {
          const float4 q = *reinterpret_cast<const float4*>(p + s * plane + u);
          z[u] += q.x, z[u + 1] += q.y, z[u + 2] += q.z, z[u + 3] += q.w;
        }
      } else {
        z[0] += p[s * plane];
      }
    }
    finish<O, V>(e, n, i, j, z);
  }
}

template <typename O>
static void add_parts(const float* part, int splits, const Product& p, const Epilogue& e, cudaStream_t st) {
  constexpr int V = 16 / sizeof(O);
  const int64_t steps = e.vec ? p.m * p.n / V : p.m * p.n;
  const int blocks = int(std::min<int64_t>((steps + 255) / 256, int64_t(sm_count()) * 8));
  if (e.vec) add_parts_kernel<O, V><<<blocks, 256, 0, st>>>(part, splits, p.m, p.n, e);
  else add_parts_kernel<O, 1><<<blocks, 256, 0, st>>>(part, splits, p.m, p.n, e);
  note_launch();
}

static gsb_status launch_of(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st) {
  switch (p->dtype) {
    case GSB_F32: return mma_launch_f32(p, e, count, bn, splits, st);
    case GSB_BF16: return mma_launch_bf16(p, e, count, bn, splits, st);
    case GSB_F16: return mma_launch_f16(p, e, count, bn, splits, st);
    default: return mma_launch_e4m3(p, e, count, bn, splits, st);
  }
}

gsb_status mma_products(const Product* p, const Epilogue* e, int count, const Plan& plan, void* part, cudaStream_t st) {
  Product q[2];
  Epilogue f[2];
  float* sums[2] = {};
  char* next = static_cast<char*>(part);
  for (int i = 0; i < count; ++i) {
    q[i] = p[i];
    f[i] = e[i];
    if (!leaves_sums(p, count, plan, i)) continue;
    sums[i] = reinterpret_cast<float*>(next);
    next += align_up(size_t(plan.splits[i]) * size_t(p[i].m) * size_t(p[i].n) * 4);
    q[i].out_dtype = GSB_F32;
    f[i] = Epilogue{};
    f[i].out = sums[i];
    f[i].out_stride = p[i].n;
    f[i].vec = p[i].n % 4 == 0;
  }
  if (gsb_status s = launch_of(q, f, count, plan.bn, plan.splits, st); s != GSB_OK) return s;
  for (int i = 0; i < count; ++i) {
    if (!sums[i]) continue;
    const int pieces = pieces_of(p[i], plan.splits[i]);
    if (p[i].out_dtype == GSB_F32) add_parts<float>(sums[i], pieces, p[i], e[i], st);
    else if (p[i].out_dtype == GSB_BF16) add_parts<bf16>(sums[i], pieces, p[i], e[i], st);
    else add_parts<f16>(sums[i], pieces, p[i], e[i], st);
  }
  return launch_status();
}

}  // namespace gsb
