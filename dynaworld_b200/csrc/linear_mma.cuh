// Matrix product on the fifth-generation tensor cores (sm_100a): D = A B^T in float.
//
// Persistent kernel, one CTA per SM; CG = 2 pairs the CTAs of a cluster on one 256 x BN tile, so
// that each loads half of B, CG = 1 gives each a 128 x BN tile.  Warp roles of a CTA (384 threads):
//   warp 0      loads: TMA copies of 128-byte wide boxes (swizzled) into a ring of slots
//   warp 1      issues tcgen05.mma, accumulators in TMEM (two buffers: the next tile's products
//               run while this tile's epilogue reads)
//   warp 2      allocates and frees TMEM
//   warps 4-11  epilogue: TMEM -> registers -> a shared-memory transpose, so that the stores (and
//               the residual's loads) are rows of 16-byte accesses
// Operands are K-major (rows of k) or MN-major (rows of m or n, as the backward's products have
// them): the TMA box and the shared-memory descriptor differ, nothing is transposed in memory.
//
// Float operands (PLANES = 3) are sums of three bf16 parts.  The tensor core's additions truncate, and
// a chain of them loses about steps x 2^-25 of what the accumulator holds.  So every block of 64 k has a
// chain of its own, the products (3,1) (1,3) (2,2) (1,2) (2,1), which are small, before the four
// steps of (1,1), and the epilogue warps add each block's sums in float registers while the next
// block runs: 128 sums per thread, for which they take registers from the other warps.
//
// Bounds.  16-bit and e4m3 products are bound by the tensor cores and, kept up, by the power limit:
// 16,384 x 1,024 x 4,096 bf16 takes 102 us alone (1.35 PFLOP/s; cuBLAS 99), 126 in a loop of 0.3 s
// (cuBLAS 117); 8,192 x 2,048 x 8,192 e4m3 113 and 133 us (cuBLAS 103 and 122).  Then by the epilogue: GELU
// and the kept pre-activation add 16 to 26 us, a residual 13 to 24.  Float products do 6 times the work:
// 4,096 x 512 x 2,560 in 58 us, 1.11 PFLOP/s of bf16 work in three rounds of which the last is a sixth full;
// with GELU 66, in a training loop that keeps z 79.
// 256 x 256 tiles over CTA pairs because an MMA takes as long for 64 columns as for 256, and half of B
// per CTA because the operands' way from L2 would bound a CTA on its own.
//
// Every wait is bounded (4 s).  A wait that gives up sets a sticky flag, its CTA's remaining tiles
// become NaN, and every role leaves its loop.
#pragma once

#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "async_copy.cuh"
#include "linear_parts.cuh"

namespace gsb {
namespace mma {

constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kStageBytes = kEpiWarps * 32 * 32 * 4;  // a 32 x 32 block of floats per epilogue warp
constexpr int kRowBytes = 128;              // one swizzled row of a box
constexpr int kABytes = 128 * kRowBytes;
// Registers per thread after the split (PLANES = 3); 128 x 56 + 256 x 224 are the 384 x 168 of the launch.
constexpr int kFewRegs = 56, kManyRegs = 224;


// One product of a launch: m_tiles x n_tiles tiles, each walked in `splits` pieces of `per_split` blocks of
// K (more than one: every piece writes its float sums to a plane of its own, part_stride apart).
struct Job {
  int64_t m, n;
  int64_t part_stride;
  int64_t units;    // tiles x splits
  int k_blocks, per_split, splits;
  int m_tiles, n_tiles;
  int group;        // m tiles walked together, for reuse in L2
  int a_mn;         // A is MN-major (backward launches)
  uint32_t idesc;
  Epilogue e;
};

// A launch's products over C clusters.  The units of job 0 (the longer ones) go round; clusters that
// got one less take `extra` rounds of job 1 before all share the rest of it.
template <int JOBS>
struct Args {
  Job job[JOBS];
  CUtensorMap a[JOBS], b[JOBS];
  int extra;
  int* gave_up;

  // The cluster's i-th unit; false past its last one.
  __device__ __forceinline__ bool unit(int c, int clusters, int64_t i, int& which, int64_t& u) const {
    which = 0;
    if constexpr (JOBS == 1) {
      u = c + i * clusters;
      return u < job[0].units;
    } else {
      const int64_t all = job[0].units / clusters;
      const int hi = int(job[0].units - all * clusters);
      const int64_t mine = all + (c < hi);
      if (i < mine) {
        u = c + i * clusters;
        return true;
      }
      which = 1;
      i -= mine;
      const int early = clusters - hi;
      if (c >= hi) {
        if (i < extra) {
          u = i * early + (c - hi);
          return u < job[1].units;
        }
        i -= extra;
      }
      u = int64_t(extra) * early + i * clusters + (c >= hi ? c - hi : c + early);
      return u < job[1].units;
    }
  }
};

// ---- PTX ----

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// bar: an address in the cluster's shared window.  Relaxed: what the arrival hands over is TMEM that has
// been read, and nothing in global or shared memory, which is what a release would order.  TMEM accesses of
// different threads are ordered by tcgen05's own rules (PTX, tcgen05 memory consistency model): the reads are
// complete after tcgen05.wait::ld, tcgen05.fence::before_thread_sync orders them before the arrival, and the
// waiting thread's fence::after_thread_sync orders its next MMA after the wait that saw it.  A release would
// also wait for the warp's stores of outputs, about a microsecond per tile.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}

// 32 columns of the warp's lanes, asynchronously: the registers hold them after tmem_wait32 on the same
// array, whose operands keep the compiler from reading them earlier.
__device__ __forceinline__ void tmem_start32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}

template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int plane, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(plane), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(plane), "r"(bar)
        : "memory");
}

template <int KIND, int CG>
__device__ __forceinline__ void mma_issue(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define GSB_MMA(cg, kind)                                                                                     \
  asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"                                                     \
               "tcgen05.mma.cta_group::" cg ".kind::" kind " [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), \
               "r"(idesc), "r"(accumulate)                                                                     \
               : "memory")
  if constexpr (KIND == 1) {
    if constexpr (CG == 1) GSB_MMA("1", "f8f6f4");
    else GSB_MMA("2", "f8f6f4");
  } else {
    if constexpr (CG == 1) GSB_MMA("1", "f16");
    else GSB_MMA("2", "f16");
  }
#undef GSB_MMA
}

// Arrives on bar (both CTAs' barriers at this offset with CG = 2) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(uint16_t(3))
        : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle (layout type 2 in bits 61-63, version 1 in bits
// 46-47).  K-major: 8-row groups 1024 bytes apart (the stride offset).  MN-major: blocks of 64
// columns 8192 bytes apart (the leading offset), groups of 8 k 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, bool mn) {
  const uint64_t lead = mn ? 8192 / 16 : 1, stride = 1024 / 16;
  return uint64_t((addr >> 4) & 0x3fff) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}

// Descriptor advance per MMA (16 k of 16-bit, 32 of 8-bit values): 32 bytes along a K-major row,
// two 8-k groups MN-major; in units of 16 bytes.
__host__ __device__ constexpr uint32_t desc_step(bool mn) { return mn ? 2048 / 16 : 32 / 16; }

__device__ __forceinline__ void tile_of(const Job& p, int64_t t, int64_t& mt, int64_t& nt) {
  const int64_t per = int64_t(p.group) * p.n_tiles;
  const int64_t band = t / per, r = t - band * per;
  const int64_t first = band * p.group;
  const int64_t rows = min(int64_t(p.group), int64_t(p.m_tiles) - first);
  mt = first + r % rows;
  nt = r / rows;
}

// Where the q-th 16 bytes of row r of a warp's block are: a permutation by row, so that eight lanes
// meet eight banks groups whether they hold eight rows (writing) or adjacent parts of one (reading).
__device__ __forceinline__ int stage_at(int r, int q) { return r * 32 + ((q ^ (r & 7)) << 2); }

// A warp's part of the epilogue.  A 32 x 32 block of sums (lane = row) goes through shared memory so
// that global accesses are 16 bytes per lane: V values, 32 / V lanes per row, kSteps rows per lane.
// The residual and bias of the next block are loaded while this one is finished: a block takes
// about 600 cycles, the residual's way from HBM more.
constexpr int kAnyAct = -1;  // the activation is chosen at run time

template <int ACT>
__device__ __forceinline__ bool is_relu(const Job& p) {
  return (ACT == kAnyAct ? p.e.act : ACT) == GSB_ACT_RELU;
}

template <int ACT, typename O, int V>
__device__ __forceinline__ void activate(const Job& p, float (&z)[V]) {
  if constexpr (ACT == kAnyAct) apply_act<O, V>(p.e.act, z);
  else apply_value<ACT, O, V>(z);
}

// VEC: the output's rows (and the residual's, bias, kept sums) allow accesses of 16 bytes.
// SCALED: e4m3 operands with their rows' scales.
template <typename O, int ACT, bool VEC, bool SCALED>
struct Rows {
  static constexpr int V = 16 / int(sizeof(O));
  static constexpr int kPerRow = 32 / V;
  static constexpr int kAtOnce = 32 / kPerRow;  // rows in one access of the warp
  static constexpr int kSteps = 32 / kAtOnce;
  using Z = typename PreactOf<O>::type;
  struct Ahead {  // what the next block reads, of aligned rows
    uint4 res[kSteps];
    uint4 bias;
  };
  int row0, col;  // this lane's first row and column within the block
  int steps;      // its rows inside the matrix
  int64_t i;      // its first row
  int64_t plane;  // offset of this piece's output
  float rs[kSteps];

  __device__ __forceinline__ void start(const Job& p, int64_t i0, int64_t plane_) {
    plane = plane_;
    const int lane = threadIdx.x & 31;
    row0 = lane / kPerRow;
    col = (lane % kPerRow) * V;
    i = i0 + row0;
    steps = int(max(int64_t(0), min(int64_t(kSteps), (p.m - i + kAtOnce - 1) / kAtOnce)));
    if (SCALED && p.e.row_scale) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) rs[s] = s < steps ? p.e.row_scale[i + s * kAtOnce] : 0.0f;
    }
  }

  __device__ __forceinline__ void prefetch(const Job& p, int64_t j0, Ahead& a) const {
    if constexpr (!VEC) return;
    const int64_t j = j0 + col;
    const bool in = j < p.n;
    if (p.e.bias && in) a.bias = __ldg(reinterpret_cast<const uint4*>(static_cast<const O*>(p.e.bias) + j));
    if (p.e.res) {
      const O* r = static_cast<const O*>(p.e.res) + i * p.e.res_stride + j;
      const int64_t step = kAtOnce * p.e.res_stride;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (in && s < steps) a.res[s] = __ldg(reinterpret_cast<const uint4*>(r + s * step));
    }
  }

  // The block's sums into shared memory ...
  __device__ __forceinline__ static void put(float* stage, const uint32_t (&v)[32]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<uint4*>(stage + stage_at(lane, q)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    __syncwarp();
  }

  // ... and from there to the output.
  __device__ __forceinline__ void emit(const Job& p, const float* stage, int64_t i0, int64_t j0, const Ahead& a) const {
    const int lane = threadIdx.x & 31;
    if constexpr (VEC) {
      const int64_t j = j0 + col;
      if (j < p.n) {
        float bias[V], cs[V];
        if (p.e.bias) {
          const Vec<O, V> b = *reinterpret_cast<const Vec<O, V>*>(&a.bias);
#pragma unroll
          for (int u = 0; u < V; ++u) bias[u] = to_f32(b.v[u]);
        }
        if (SCALED && p.e.row_scale) {
#pragma unroll
          for (int u = 0; u < V; ++u) cs[u] = p.e.col_scale[j + u];
        }
        O* out = static_cast<O*>(p.e.out) + plane + i * p.e.out_stride + j;
        Z* keep = static_cast<Z*>(p.e.preact) + i * p.n + j;
        // two rows' arithmetic at a time, no branch between them: a warp's latencies overlap
#pragma unroll
        for (int s0 = 0; s0 < kSteps; s0 += 2) {
          float z[2 * V];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int v = 0; v < V; v += 4) {
              const float4 q =
                  *reinterpret_cast<const float4*>(stage + stage_at(row0 + (s0 + h) * kAtOnce, (col + v) >> 2));
              float* to = z + h * V + v;
              to[0] = q.x, to[1] = q.y, to[2] = q.z, to[3] = q.w;
            }
          if (SCALED && p.e.row_scale) {
#pragma unroll
            for (int v = 0; v < 2 * V; ++v) z[v] *= rs[s0 + v / V] * cs[v % V];
          }
          if (p.e.bias) {
#pragma unroll
            for (int v = 0; v < 2 * V; ++v) z[v] += bias[v % V];
          }
          if (p.e.preact) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (s0 + h < steps)
                *reinterpret_cast<Vec<Z, V>*>(keep + (s0 + h) * kAtOnce * p.n) =
                    kept_of<V>(static_cast<Z*>(nullptr), reinterpret_cast<const float(&)[V]>(z[h * V]), is_relu<ACT>(p));
          }
          activate<ACT, O, 2 * V>(p, z);
          if (p.e.res) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const Vec<O, V> r = *reinterpret_cast<const Vec<O, V>*>(&a.res[s0 + h]);
#pragma unroll
              for (int v = 0; v < V; ++v) z[h * V + v] += to_f32(r.v[v]);
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (s0 + h < steps)
              store_f32<O, V>(out + (s0 + h) * kAtOnce * p.e.out_stride, reinterpret_cast<const float(&)[V]>(z[h * V]));
        }
      }
    } else {
      // rows that start anywhere: a lane per column, the residual's 32 rows asked for at once
      const int64_t j = j0 + lane;
      if (j < p.n) {
        O add[32];
        if (p.e.res) {
          const O* r = static_cast<const O*>(p.e.res) + i0 * p.e.res_stride + j;
#pragma unroll
          for (int q = 0; q < 32; ++q)
            if (i0 + q < p.m) add[q] = r[q * p.e.res_stride];
        }
        const float b = p.e.bias ? to_f32(static_cast<const O*>(p.e.bias)[j]) : 0.0f;
        const float cs = SCALED && p.e.row_scale ? p.e.col_scale[j] : 1.0f;
        O* out = static_cast<O*>(p.e.out) + plane + i0 * p.e.out_stride + j;
        Z* keep = static_cast<Z*>(p.e.preact) + i0 * p.n + j;
        const int rows = int(min(int64_t(32), p.m - i0));
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 8) {
          float z[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            z[r] = stage[stage_at(r0 + r, lane >> 2) + (lane & 3)];
            if (SCALED && p.e.row_scale && r0 + r < rows) z[r] *= p.e.row_scale[i0 + r0 + r] * cs;
            z[r] += b;
          }
          if (p.e.preact) {
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (r0 + r < rows) keep[(r0 + r) * p.n] = as_preact(static_cast<Z*>(nullptr), z[r], is_relu<ACT>(p));
          }
          activate<ACT, O, 8>(p, z);
          if (p.e.res) {
#pragma unroll
            for (int r = 0; r < 8; ++r) z[r] += to_f32(add[r0 + r]);
          }
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r0 + r < rows) out[(r0 + r) * p.e.out_stride] = from_f32<O>(z[r]);
        }
      }
    }
    __syncwarp();
  }
};

template <int CG, int BN, int PLANES>
struct Shape {
  static constexpr int kBRows = BN / CG;              // rows of B that one CTA loads
  static constexpr int kBBytes = kBRows * kRowBytes;
  static constexpr int kSlot = kABytes + kBBytes;
  static constexpr int kBudget = 232448 - 1024 - kStageBytes - 256;
  static constexpr int kSlots = kBudget / kSlot < 8 ? kBudget / kSlot : 8;
  static constexpr int kBufs = 2;
  static constexpr int kAccCols = BN;  // TMEM columns of one accumulator buffer
  static constexpr int kCols = kBufs * kAccCols;
  static constexpr int kBytes = 1024 + kSlots * kSlot + kStageBytes + 256;
  static_assert(kCols <= 512 && (kCols & (kCols - 1)) == 0 && kCols >= 32, "TMEM columns");
  static_assert(PLANES == 1 || kSlots >= 4, "a block's three slots and one ahead");
};

// KIND 0: 16-bit operands, 1: e4m3.  BWD: up to two products, B MN-major; else one, both K-major.
template <int KIND, int CG, int BN, bool BWD, int PLANES, typename O, int ACT, bool VEC>
__global__ void __launch_bounds__(kThreads, 1) mma_kernel(const __grid_constant__ Args<1 + BWD> p) {
  using S = Shape<CG, BN, PLANES>;
  constexpr int kElems = KIND == 1 ? 128 : 64;  // k per block
  constexpr int JOBS = 1 + BWD;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  uint8_t* smem = raw + (base - smem_addr(raw));
  float* stage_all = reinterpret_cast<float*>(smem + S::kSlots * S::kSlot);
  const uint32_t bars = base + S::kSlots * S::kSlot + kStageBytes;
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (S::kSlots + s); };
  const auto acc_full = [&](int b) { return bars + 8 * (2 * S::kSlots + b); };
  const auto acc_empty = [&](int b) { return bars + 8 * (2 * S::kSlots + 2 + b); };
  const uint32_t tmem_slot = bars + 8 * (2 * S::kSlots + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cluster_rank();

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kSlots; ++s) {
      bar_init(full(s), 1);
      bar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(acc_full(b), 1);
      bar_init(acc_empty(b), kEpiWarps * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) tmem_alloc<CG>(tmem_slot, S::kCols);
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_barrier();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));

  const int cluster = blockIdx.x / CG, clusters = gridDim.x / CG;
  int which;
  int64_t u;

  if (warp >= 4) {
    if constexpr (PLANES > 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
    const int w = warp - 4, quad = warp & 3, half = w >> 2;  // quad: the 32 TMEM lanes this warp may read
    float* stage = stage_all + w * 32 * 32;
    const uint32_t lanes = uint32_t(quad * 32) << 16;
    constexpr int kHalfCols = BN / 2;
    bool ok = true;
    int buf = 0;
    uint32_t acc_phase = 0;
    Rows<O, ACT, VEC, KIND == 1> rows;
    typename Rows<O, ACT, VEC, KIND == 1>::Ahead ahead;
    for (int64_t i = 0; p.unit(cluster, clusters, i, which, u); ++i) {
      const Job& job = p.job[which];
      int64_t mt, nt;
      tile_of(job, u / job.splits, mt, nt);
      const int64_t plane = (u % job.splits) * job.part_stride;
      const int64_t i0 = (mt * CG + rank) * 128 + quad * 32;
      const int64_t j0 = nt * BN + half * kHalfCols;
      const auto release = [&](int b) {
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(map_to_rank(acc_empty(b), 0));
      };
      if constexpr (PLANES == 1) {
        rows.start(job, i0, plane);
        rows.prefetch(job, j0, ahead);
        ok = __all_sync(0xffffffffu, ok && bar_wait(acc_full(buf), acc_phase, p.gave_up));
        fence_after();
        const uint32_t acc = tmem + lanes + buf * S::kAccCols + half * kHalfCols;
        uint32_t v[32];
        tmem_start32(acc, v);
#pragma unroll 1
        for (int c = 0; c < kHalfCols; c += 32) {
          const typename Rows<O, ACT, VEC, KIND == 1>::Ahead now = ahead;
          if (c + 32 < kHalfCols) rows.prefetch(job, j0 + c + 32, ahead);
          tmem_wait32(v);
          if (!ok) {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] = 0x7fc00000;
          }
          rows.put(stage, v);
          if (c + 32 < kHalfCols) tmem_start32(acc + c + 32, v);
          else release(buf);
          if (i0 < job.m && j0 + c < job.n) rows.emit(job, stage, i0, j0 + c, now);
        }
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      } else {
        constexpr int kAtOnce = kHalfCols < 64 ? kHalfCols : 64;  // columns on their way from TMEM
        float sum[kHalfCols];
#pragma unroll
        for (int q = 0; q < kHalfCols; ++q) sum[q] = 0.0f;
        const int kb0 = int(u % job.splits) * job.per_split, kb1 = min(job.k_blocks, kb0 + job.per_split);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = __all_sync(0xffffffffu, ok && bar_wait(acc_full(buf), acc_phase, p.gave_up));
          fence_after();
          const uint32_t acc = tmem + lanes + buf * S::kAccCols + half * kHalfCols;
#pragma unroll
          for (int c = 0; c < kHalfCols; c += kAtOnce) {
            uint32_t v[kAtOnce / 32][32];
#pragma unroll
            for (int h = 0; h < kAtOnce / 32; ++h) tmem_start32(acc + c + 32 * h, v[h]);
#pragma unroll
            for (int h = 0; h < kAtOnce / 32; ++h) tmem_wait32(v[h]);
#pragma unroll
            for (int q = 0; q < kAtOnce; ++q) sum[c + q] += __uint_as_float(v[q / 32][q % 32]);
          }
          release(buf);
          buf ^= 1;
          if (buf == 0) acc_phase ^= 1;
        }
        if (!ok) {
#pragma unroll
          for (int q = 0; q < kHalfCols; ++q) sum[q] = __int_as_float(0x7fc00000);
        }
        rows.start(job, i0, plane);
#pragma unroll
        for (int c = 0; c < kHalfCols; c += 32) {
          rows.put(stage, reinterpret_cast<const uint32_t(&)[32]>(sum[c]));
          rows.prefetch(job, j0 + c, ahead);
          if (i0 < job.m && j0 + c < job.n) rows.emit(job, stage, i0, j0 + c, ahead);
        }
      }
    }
  } else {
    if constexpr (PLANES > 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    if (warp == 0) {
      if (lane == 0) {
        bool ok = true;
        int s = 0;
        uint32_t phase = 0;
        for (int64_t i = 0; ok && p.unit(cluster, clusters, i, which, u); ++i) {
          const Job& job = p.job[which];
          const CUtensorMap* map_a = which ? &p.a[JOBS - 1] : &p.a[0];
          const CUtensorMap* map_b = which ? &p.b[JOBS - 1] : &p.b[0];
          int64_t mt, nt;
          tile_of(job, u / job.splits, mt, nt);
          const int i0 = int((mt * CG + rank) * 128);
          const int j0 = int(nt * BN + rank * S::kBRows);
          const int kb0 = int(u % job.splits) * job.per_split, kb1 = min(job.k_blocks, kb0 + job.per_split);
          const auto walk = [&](auto mn) {
            for (int kb = kb0; ok && kb < kb1; ++kb) {
              const int k0 = kb * kElems;
#pragma unroll
              for (int q = 0; q < PLANES; ++q) {
                const int plane = PLANES == 1 ? 0 : (q == 0 ? 2 : q - 1);  // parts 3, 1, 2
                if (!(ok = bar_wait(empty(s), phase ^ 1, p.gave_up))) break;
                const uint32_t bar = CG == 1 ? full(s) : map_to_rank(full(s), 0);
                if (rank == 0) bar_expect(full(s), CG * S::kSlot);
                const uint32_t a = base + s * S::kSlot, b = a + kABytes;
                if constexpr (decltype(mn)::value) {
#pragma unroll
                  for (int v = 0; v < 2; ++v) tma_load<CG>(a + v * 8192, map_a, i0 + 64 * v, k0, plane, bar);
                } else {
                  tma_load<CG>(a, map_a, k0, i0, plane, bar);
                }
                if constexpr (BWD) {
#pragma unroll
                  for (int v = 0; v < S::kBRows / 64; ++v) tma_load<CG>(b + v * 8192, map_b, j0 + 64 * v, k0, plane, bar);
                } else {
                  tma_load<CG>(b, map_b, k0, j0, plane, bar);
                }
                if (++s == S::kSlots) s = 0, phase ^= 1;
              }
            }
          };
          if (BWD && job.a_mn) walk(std::true_type{});
          else walk(std::false_type{});
        }
        // every slot released: no arrival of a commit comes after the CTA's end
        for (int q = 0; ok && q < S::kSlots; ++q) {
          ok = bar_wait(empty(s), phase ^ 1, p.gave_up);
          if (++s == S::kSlots) s = 0, phase ^= 1;
        }
        if (!ok) let_copies_land();
      }
    } else if (warp == 1) {
      if (rank == 0 && lane == 0) {
        bool ok = true;
        int s = 0, buf = 0;
        uint32_t phase = 0, acc_phase = 0;
        const auto next = [&](int x) { return x + 1 == S::kSlots ? 0 : x + 1; };
        for (int64_t i = 0; ok && p.unit(cluster, clusters, i, which, u); ++i) {
          const Job& job = p.job[which];
          const uint32_t idesc = job.idesc;
          const int kb0 = int(u % job.splits) * job.per_split, kb1 = min(job.k_blocks, kb0 + job.per_split);
          const auto walk = [&](auto mn) {
            constexpr bool a_mn = decltype(mn)::value;
            constexpr uint32_t a_step = desc_step(a_mn), b_step = desc_step(BWD);
            for (int kb = kb0; ok && kb < kb1;) {
              if (!(ok = bar_wait(acc_empty(buf), acc_phase ^ 1, p.gave_up))) break;
              fence_after();
              const uint32_t acc = tmem + buf * S::kAccCols;
              const int stop = PLANES == 1 ? kb1 : kb + 1;
              uint32_t more = 0;
              for (; kb < stop; ++kb) {
                if constexpr (PLANES == 1) {
                  if (!(ok = bar_wait(full(s), phase, p.gave_up))) break;
                  fence_after();
                  const uint64_t a = smem_desc(base + s * S::kSlot, a_mn);
                  const uint64_t b = smem_desc(base + s * S::kSlot + kABytes, BWD);
#pragma unroll
                  for (int v = 0; v < 4; ++v) {
                    mma_issue<KIND, CG>(acc, a + v * a_step, b + v * b_step, idesc, more);
                    more = 1;
                  }
                  mma_commit<CG>(empty(s));
                  if (++s == S::kSlots) s = 0, phase ^= 1;
                } else {
                  const int s3 = s, s1 = next(s3), s2 = next(s1);
                  const uint32_t ph1 = phase ^ (s1 < s3), ph2 = ph1 ^ (s2 < s1);
                  const auto da = [&](int q) { return smem_desc(base + q * S::kSlot, a_mn); };
                  const auto db = [&](int q) { return smem_desc(base + q * S::kSlot + kABytes, BWD); };
                  const auto run = [&](uint64_t a, uint64_t b) {
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                      mma_issue<KIND, CG>(acc, a + v * a_step, b + v * b_step, idesc, more);
                      more = 1;
                    }
                  };
                  if (!(ok = bar_wait(full(s3), phase, p.gave_up) && bar_wait(full(s1), ph1, p.gave_up))) break;
                  fence_after();
                  run(da(s3), db(s1));
                  run(da(s1), db(s3));
                  mma_commit<CG>(empty(s3));
                  if (!(ok = bar_wait(full(s2), ph2, p.gave_up))) break;
                  fence_after();
                  run(da(s2), db(s2));
                  run(da(s1), db(s2));
                  run(da(s2), db(s1));
                  mma_commit<CG>(empty(s2));
                  run(da(s1), db(s1));
                  mma_commit<CG>(empty(s1));
                  s = next(s2);
                  phase = ph2 ^ (s < s2);
                }
              }
              mma_commit<CG>(acc_full(buf));
              buf ^= 1;
              if (buf == 0) acc_phase ^= 1;
            }
          };
          if (BWD && job.a_mn) walk(std::true_type{});
          else walk(std::false_type{});
        }
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_barrier();
  fence_after();
  if (warp == 2) tmem_free<CG>(tmem, S::kCols);
}

// ---- host ----

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn();  // NULL when the driver does not offer it

// An operand [rows, k] as boxes of 128 bytes: K-major 128-byte rows of k, MN-major 64 rows of k by 64
// columns.  Values outside the matrix read as 0.
inline bool make_map(CUtensorMap* map, const void* ptr, int dtype, bool mn, int64_t rows, int64_t k, int64_t ld,
                     int box_rows, int planes, int64_t plane_stride) {
  EncodeFn encode = encode_fn();
  if (!encode) return false;
  const int e = dtype == GSB_E4M3 ? 1 : 2;
  const CUtensorMapDataType type = dtype == GSB_E4M3  ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : dtype == GSB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t dims[3] = {cuuint64_t(mn ? rows : k), cuuint64_t(mn ? k : rows), cuuint64_t(planes)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * e, cuuint64_t(planes > 1 ? plane_stride : ld) * e};
  const cuuint32_t box[3] = {cuuint32_t(128 / e), cuuint32_t(mn ? 64 : box_rows), 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode(map, type, 3, const_cast<void*>(ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// kind::f16: D float (bit 4), A and B formats (0 fp16, 1 bf16; e4m3 is 0 of kind::f8f6f4), MN-major
// flags in bits 15 and 16, N / 8 from bit 17, M / 16 from bit 24.
inline uint32_t instr_desc(int dtype, bool a_mn, bool b_mn, int m, int n) {
  const uint32_t f = (dtype == GSB_BF16 || dtype == GSB_F32) ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

template <int KIND, int CG, int BN, int PLANES>
bool make_job(Job& j, CUtensorMap* a, CUtensorMap* b, const Product& p, const Epilogue& e, int splits) {
  using S = Shape<CG, BN, PLANES>;
  if (!make_map(a, p.a, p.dtype, p.a_mn, p.m, p.k, p.a_ld, 128, PLANES, p.a_plane) ||
      !make_map(b, p.b, p.dtype, p.b_mn, p.n, p.k, p.b_ld, S::kBRows, PLANES, p.b_plane))
    return false;
  j.m = p.m;
  j.n = p.n;
  j.k_blocks = k_blocks_of(p);
  j.per_split = piece_of(p, splits);
  j.splits = (j.k_blocks + j.per_split - 1) / j.per_split;
  j.part_stride = j.splits > 1 ? p.m * p.n : 0;
  j.m_tiles = int((p.m + 128 * CG - 1) / (128 * CG));
  j.n_tiles = int((p.n + BN - 1) / BN);
  j.units = int64_t(j.m_tiles) * j.n_tiles * j.splits;
  j.group = 8;
  j.a_mn = p.a_mn;
  j.idesc = instr_desc(p.dtype, p.a_mn, p.b_mn, 128 * CG, BN);
  j.e = e;
  return true;
}

// products[0 .. count): one forward product, or one or two of the backward's.
template <int KIND, int CG, int BN, bool BWD, int PLANES, typename O, int ACT, bool VEC>
gsb_status launch(const Product* products, const Epilogue* e, int count, const int* splits, cudaStream_t st) {
  using S = Shape<CG, BN, PLANES>;
  auto* kernel = mma_kernel<KIND, CG, BN, BWD, PLANES, O, ACT, VEC>;
  int dev = 0;
  (void)cudaGetDevice(&dev);
  static std::atomic<uint64_t> ready{0};  // devices whose copy of the kernel has its shared memory
  const uint64_t bit = 1ull << (dev & 63);
  if (!(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess) {
      (void)cudaGetLastError();
      return GSB_ERR_CUDA;
    }
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  Args<1 + BWD> a{};
  int64_t units = 0;
  // the product of the longer pieces first
  const bool swap = count == 2 && piece_of(products[1], splits[1]) > piece_of(products[0], splits[0]);
  for (int i = 0; i < count; ++i) {
    const int from = swap ? 1 - i : i;
    if (!make_job<KIND, CG, BN, PLANES>(a.job[i], &a.a[i], &a.b[i], products[from], e[from], splits[from]))
      return GSB_ERR_CUDA;
    units += a.job[i].units;
  }
  a.gave_up = gave_up_flag();
  if (!a.gave_up) return GSB_ERR_CUDA;
  const int clusters = int(std::min<int64_t>(units, sm_count() / CG));
  if constexpr (BWD) {
    const int early = clusters - int(a.job[0].units % clusters);
    if (count == 2 && early < clusters) {
      const int64_t d0 = a.job[0].per_split, d1 = a.job[1].per_split;
      a.extra = int(std::min<int64_t>((d0 + d1 / 2) / d1, (a.job[1].units + early - 1) / early));
    }
    if (count == 1) a.job[1].splits = 1;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(clusters * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, a);
  note_launch();
  if (err != cudaSuccess) {
    (void)cudaGetLastError();
    return GSB_ERR_CUDA;
  }
  return launch_status();
}

// By tile: 256 is 256 x 256 over a pair of CTAs, 128 and 64 are 128 rows by that many columns on one
// CTA.
template <int KIND, bool BWD, int PLANES, typename O, int ACT, bool VEC>
gsb_status launch_tile(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st) {
  if (bn == 128) return launch<KIND, 1, 128, BWD, PLANES, O, ACT, VEC>(p, e, count, splits, st);
  if (bn == 64) return launch<KIND, 1, 64, BWD, PLANES, O, ACT, VEC>(p, e, count, splits, st);
  return launch<KIND, 2, 256, BWD, PLANES, O, ACT, VEC>(p, e, count, splits, st);
}

// One product without an epilogue (BWD: one or two).
template <int KIND, bool BWD, int PLANES, typename O>
gsb_status launch_plain(const Product* p, const Epilogue* e, int count, int bn, const int* splits, cudaStream_t st) {
  if (e[0].vec && e[count - 1].vec)
    return launch_tile<KIND, BWD, PLANES, O, GSB_ACT_NONE, true>(p, e, count, bn, splits, st);
  return launch_tile<KIND, BWD, PLANES, O, GSB_ACT_NONE, false>(p, e, count, bn, splits, st);
}

// The forward.  Large aligned outputs have an instance per activation, the others choose at run time.
template <int KIND, int PLANES, typename O>
gsb_status launch_fwd(const Product& p, const Epilogue& e, int bn, const int* splits, cudaStream_t st) {
  if (!e.vec) return launch_tile<KIND, false, PLANES, O, kAnyAct, false>(&p, &e, 1, bn, splits, st);
  if (bn == 128) return launch<KIND, 1, 128, false, PLANES, O, kAnyAct, true>(&p, &e, 1, splits, st);
  if (bn == 64) return launch<KIND, 1, 64, false, PLANES, O, kAnyAct, true>(&p, &e, 1, splits, st);
  switch (e.act) {
    case GSB_ACT_RELU: return launch<KIND, 2, 256, false, PLANES, O, GSB_ACT_RELU, true>(&p, &e, 1, splits, st);
    case GSB_ACT_GELU: return launch<KIND, 2, 256, false, PLANES, O, GSB_ACT_GELU, true>(&p, &e, 1, splits, st);
    case GSB_ACT_GELU_TANH: return launch<KIND, 2, 256, false, PLANES, O, GSB_ACT_GELU_TANH, true>(&p, &e, 1, splits, st);
    case GSB_ACT_SILU: return launch<KIND, 2, 256, false, PLANES, O, GSB_ACT_SILU, true>(&p, &e, 1, splits, st);
    default: return launch<KIND, 2, 256, false, PLANES, O, GSB_ACT_NONE, true>(&p, &e, 1, splits, st);
  }
}

}  // namespace mma
}  // namespace gsb
