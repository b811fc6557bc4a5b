// Half-precision tensor-core products with a fused epilogue: the main loop that
// the dense layer (dense.cu) and the Newton-Schulz products (muon.cu) share.
//
//   D(m, n) = sum_k A(m, k) B(n, k),  fp32 accumulation in TMEM (kind::f16)
//
// Persistent: one CTA (CG = 1) or a pair of CTAs on two SMs (CG = 2, one
// cta_group::2 accumulator tile of 256 rows) per SM or SM pair walks work items
// (group, batch entry, m-tile, n-tile, k-split):
//   warp 0      TMA producer: k-slices of 64 values (one 128-byte swizzle row)
//               of A and B into a ring of shared-memory stages;
//   warp 1      one thread issues the UMMAs (K = 16) of a stage, commits the
//               stage back to the producers and each finished accumulator to
//               the epilogue (two accumulators: an item's epilogue runs beside
//               the next item's products);
//   warps 2..   epilogue: tcgen05.ld (thread = row), the layer's own arithmetic,
//               and the result through shared memory to global memory.
// Operands are K-major (contiguous along k) or MN-major (contiguous along m or
// n), so x W^T, g W and g^T x read their operands as they are stored.
// PLANES = 2: every operand is a pair of fp16 planes hi + lo (22 significant
// bits) and a k-slice makes the products lo hi + hi lo + hi hi; the dropped
// lo lo term is 2^-22 relative. The tensor core truncates as it adds to an
// accumulator (a sum of positive terms over k = 3072, 576 additions, came out
// 2e-5 low), so accumulators then hold a few k-slices at a time and the
// epilogue warps add them up in registers, rounded to nearest.
// A pair of SMs halves the B bytes each SM stages per flop: a 256 x 256 tile
// takes 32 KB of shared memory per 64-wide slice and SM against 48 KB for the
// 128 x 256 tile of one SM, so that a ring of five stages fits beside the
// epilogue's blocks (three stages: 12% slower).
// Measured (bf16, one plane): 8192^3 in 709 us, 1.55 PFLOP/s, 94% of the measured
// cuBLAS rate; 65536 x 3072 x 768 in 230 us, 1.34 PFLOP/s, where the output's
// way through shared memory takes 27 us from the products.
// Every wait is bounded: on timeout the kernel records an error in the
// translation unit's error word, lets its copies land and unwinds.
#pragma once

#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "sm100.cuh"

namespace cg {
namespace half {

using namespace cg::sm100;

constexpr int kBK = 64;        // half-precision values per k-slice: 128 bytes
constexpr int kRows = 128;     // accumulator rows per CTA
// warps of a block: producer, issuer and `epi` epilogue warps (a multiple of
// four, epi / 4 per TMEM lane quarter)
__host__ __device__ constexpr int threads_of(int epi) { return 32 * (2 + epi); }
constexpr int kBand = 8;       // m-tiles of one band of the tile walk (a power of two)

// Bounded wait of a whole warp, with one outcome for all its lanes: 2^24 polls
// are about half a second at the least, hundreds of times the longest tile.
__device__ inline bool wait(uint64_t* bar, uint32_t parity, int* error_word) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, error_word, 1u << 24));
}

// One lane of a converged warp, the same one every time.
__device__ inline bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// ---- PTX of the cta_group::2 forms -----------------------------------------
__device__ inline uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ inline void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrive on the barrier at this shared-memory offset in CTA `rank` of the cluster,
// ordering nothing but the tensor memory accesses before a tc_fence_before().
__device__ inline void mbar_arrive_remote(uint64_t* bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %0, %1;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)),
      "r"(rank)
      : "memory");
}
template <int CG>
__device__ inline void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  if (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
  } else {
    // both CTAs of the pair report to the leader's barrier (bit 24 of the
    // shared-window address is the CTA's place in the pair)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar) & 0xFEFFFFFFu), "r"(x), "r"(y), "r"(z)
        : "memory");
  }
}
// A block between this CTA's shared memory and global memory; out-of-range
// parts are read as zero and not written. Stores are one bulk group each.
__device__ inline void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until all this thread's stores have read their shared memory / are complete.
__device__ inline void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ inline void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

template <int CG>
__device__ inline void tmem_alloc_cg(uint32_t* slot, uint32_t cols) {
  if (CG == 1) {
    tmem_alloc(slot, cols);
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ inline void tmem_dealloc_cg(uint32_t taddr, uint32_t cols) {
  if (CG == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
template <int CG>
__device__ inline void umma_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  if (CG == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
  }
}
// Arrive on `bar` (in both CTAs of a pair) once this thread's UMMAs have completed.
template <int CG>
__device__ inline void umma_commit_cg(uint64_t* bar) {
  if (CG == 1) {
    umma_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  }
}

// Instruction descriptor of kind::f16 with fp32 accumulation; both operands
// have the same type (bf16 or fp16).
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool bf16, bool a_mn_major, bool b_mn_major) {
  return (1u << 4)                         // D format: f32
         | ((bf16 ? 1u : 0u) << 7)         // A format: f16 / bf16
         | ((bf16 ? 1u : 0u) << 10)        // B format
         | ((a_mn_major ? 1u : 0u) << 15)  // A major
         | ((b_mn_major ? 1u : 0u) << 16)  // B major
         | ((uint32_t)(n >> 3) << 17)      // N / 8
         | ((uint32_t)(m >> 4) << 24);     // M / 16
}

// ---- chained launches -----------------------------------------------------------
// A kernel launched with launch_chained may start while the kernel before it in
// the stream still runs, if that one allows it (allow_next): it sets itself up
// and then waits (wait_previous) for the other's end and memory, before it reads
// or writes any global memory. It hides a launch's gap and set-up, about 3 us of
// each kernel of a chain of small products.
__device__ inline void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// The same for kernels of many small blocks, which are held up by the next
// kernel's blocks that wait on their SMs: only where all run at once (the
// prepare passes of 42 million values: 77 us, 105 us when they allow it always).
__device__ inline void allow_next_if_few() {
  if (gridDim.x * gridDim.y <= 512) allow_next();
}
__device__ inline void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Allow a kernel its dynamic shared memory, once per device and kernel (one Tag
// each; the call takes about half a microsecond).
template <class Tag, class K>
int allow_shared(K* kernel, int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  CG_CUDA(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  if (done.load(std::memory_order_acquire) & bit) return kOk;
  CG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_release);
  return kOk;
}

template <class... P, class... A>
int launch_chained(const char* name, void (*kernel)(P...), dim3 grid, int threads, int smem, dim3 cluster,
                   cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster.x;
  attr[1].val.clusterDim.y = cluster.y;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster.x * cluster.y > 1 ? 2 : 1;
  CG_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<A&&>(args)...));
  CG_LAUNCHED(name);
  return kOk;
}

// ---- tiles ------------------------------------------------------------------
template <int CG, int BN, int PLANES, class Epi>
struct Tile {
  static constexpr int kBRows = BN / CG;                       // B rows this CTA stages
  static constexpr int kA = kRows * kBK * 2;
  static constexpr int kBBlocks = (kBRows + 63) / 64;          // 64-wide boxes of an MN-major operand
  static constexpr int kB = kBBlocks * 64 * kBK * 2;
  static constexpr int kStage = PLANES * (kA + kB);
  static constexpr int kStaging = Epi::kWarps * Epi::kStagingBytes;  // the epilogue warps' own blocks
  static constexpr int kStagesFit = (227 * 1024 - kStaging - 1024 - 512) / kStage;
  static constexpr int kStages = kStagesFit < 8 ? kStagesFit : 8;
  static constexpr int kBytes = kStages * kStage + kStaging + 1024 /*alignment*/ + 512 /*barriers*/;
  static constexpr uint32_t kAccCols = BN <= 64 ? 64 : BN <= 128 ? 128 : 256;  // of one accumulator
  static constexpr uint32_t kTmemCols = 2 * kAccCols;
  static_assert(kBRows % 32 == 0, "rows of B");
  static_assert(kStages >= 3 && kTmemCols <= 512, "tile");
};

// Division of 0 <= n < 2^31 by a fixed d >= 1, without the dozens of
// instructions of an integer division: floor(n m / 2^(32 + s)) with m = the
// ceiling of 2^(32 + s) / d, s = ceil(log2 d) - 1 (Granlund and Montgomery,
// Division by invariant integers using multiplication).
struct Divisor {
  uint32_t d, m, s;
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> s); }
};
inline Divisor divisor(int64_t d) {
  Divisor r = {(uint32_t)d, 0, 0};
  if (d > 1) {
    while ((2ll << r.s) < d) ++r.s;
    r.m = (uint32_t)(((1ull << (32 + r.s)) + (uint64_t)d - 1) / (uint64_t)d);
  }
  return r;
}

// One problem of a launch: `batch` products of one shape.
template <class EpiArgs>
struct Group {
  CUtensorMap map_a, map_b;  // 3-D: (contiguous, rows, batch entry x plane)
  int m, n, k;
  int m_tiles, n_tiles;      // in tiles of CG * 128 x BN
  int batch;
  int a_mn, b_mn;            // MN-major operands
  int splits, kt_per;        // k-slices per split
  int lower;                 // symmetric result: only tiles that reach the lower triangle
  int tiles;                 // items per batch entry and split
  Divisor by_tiles, by_batch, by_band, by_last;  // by tiles, batch, a band's tiles, the last band's height
  int first_item;
  int first_tile;            // PLANES = 2 with splits: place of its partial tiles and counters
  EpiArgs epi;
};

// A launch: up to GROUPS problems of different shapes, walked in order.
template <class EpiArgs, int GROUPS>
struct Launch {
  Group<EpiArgs> g[GROUPS];
  int groups, items;
  int bf16;
  // PLANES = 2 with splits: a tile's splits leave their sums here, and the one
  // that counts last finishes it (counters are zero before the launch and after)
  float4* partial;
  unsigned* counters;
  int most_splits;  // room per tile
  int sum_slices;   // PLANES = 2: k-slices summed in one accumulator
};
template <class Epi>
using LaunchOf = Launch<typename Epi::Args, Epi::kGroups>;

struct Item {
  int g, batch, split, m0, n0, kt0, kt1;
  int tile;  // place of the output tile among its group's
};

// Tiles of a symmetric result that reach its lower triangle: row block i (of
// `bm` rows) holds those with n0 <= m0 + bm - 1.
__host__ __device__ inline int lower_tiles_of_row(int i, int bm, int bn, int n_tiles) {
  const int c = ((i + 1) * bm + bn - 1) / bn;
  return c < n_tiles ? c : n_tiles;
}

template <int BM, int BN, class EpiArgs, int GROUPS>
__device__ inline Item item_of(const Launch<EpiArgs, GROUPS>& L, int w) {
  Item it;
  it.g = 0;
  if (GROUPS > 1)
    while (it.g + 1 < L.groups && w >= L.g[it.g + 1].first_item) ++it.g;
  const Group<EpiArgs>& g = L.g[it.g];
  w -= g.first_item;
  const int which = g.by_tiles.div(w);
  int t = w - which * g.tiles;
  it.split = g.by_batch.div(which);
  it.batch = which - it.split * g.batch;
  it.tile = it.batch * g.tiles + t;
  int mt, nt;
  if (g.lower) {
    mt = 0;
    int c;
    while (t >= (c = lower_tiles_of_row(mt, BM, BN, g.n_tiles))) {
      t -= c;
      ++mt;
    }
    nt = t;
  } else {
    // bands of kBand m-tiles, each walked m first: a wave of tiles then covers
    // a near-square block and reads few rows of either operand
    const int band = g.by_band.div(t);
    t -= band * kBand * g.n_tiles;
    const int high = g.m_tiles - band * kBand;
    nt = high >= kBand ? t / kBand : g.by_last.div(t);
    mt = band * kBand + t - nt * (high >= kBand ? kBand : high);
  }
  it.m0 = mt * BM;
  it.n0 = nt * BN;
  const int kt_all = (g.k + kBK - 1) / kBK;
  it.kt0 = it.split * g.kt_per;
  it.kt1 = it.kt0 + g.kt_per < kt_all ? it.kt0 + g.kt_per : kt_all;
  return it;
}

// Place of column c of row r in a warp's staged 32 x 32 block: the row's eight
// 16-byte chunks are XOR-swizzled by (r & 7), so row-per-lane writes and
// 8-columns-per-lane reads are free of bank conflicts.
__device__ __forceinline__ int stage_idx(int r, int c) { return r * 32 + ((((c >> 2) ^ (r & 7)) << 2) | (c & 3)); }

__device__ __forceinline__ void stage_read8(const float* stage, int r, int c, float (&v)[8]) {
  const float4 x = *reinterpret_cast<const float4*>(stage + stage_idx(r, c));
  const float4 y = *reinterpret_cast<const float4*>(stage + stage_idx(r, c + 4));
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}

// Epi: Epi::Args (kernel parameter, per group), Epi::kGroups (problems per
// launch), kWarps, kStagingBytes (shared memory per epilogue warp, a multiple of 1024),
// Epi(launch, staging, barrier, lane), begin(group, item, row0), fetch(col0)
// (starts what the next block reads), store(accumulator, col0) (a block of 32
// rows: 64 columns from TMEM, or 32 summed ones with PLANES = 2), skip() (after a
// fetch, when another split finishes the tile), spread() (the last tile's blocks
// may use memory of their own), finish(), and
// error_word() (the translation unit's).
template <int CG, int BN, int PLANES, class Epi>
__global__ void __launch_bounds__(threads_of(Epi::kWarps), 1)
    half_gemm_kernel(const __grid_constant__ LaunchOf<Epi> L) {
  using T = Tile<CG, BN, PLANES, Epi>;
  constexpr int BM = CG * kRows;
  constexpr int STAGES = T::kStages;
  constexpr int WARPS = Epi::kWarps;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // 128-byte swizzled tiles need 1024-byte alignment
  unsigned char* tiles = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* staging = tiles + STAGES * T::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + STAGES * T::kStage + T::kStaging);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* epi_bars = acc_empty + 2;  // one per epilogue warp, for the blocks it loads
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(epi_bars + WARPS);

  // the roles run as whole warps, one elected lane issuing, so that what a launch
  // holds for each group stays in uniform registers (by a single lane, with the
  // group's index not a constant, every product took 10 to 17% longer)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  allow_next();
  if (threadIdx.x == 0) {
    for (int i = 0; i < L.groups; ++i) {
      prefetch_tmap(&L.g[i].map_a);
      prefetch_tmap(&L.g[i].map_b);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CG * WARPS);  // one arrival per epilogue warp of the pair
    }
    for (int e = 0; e < WARPS; ++e) mbar_init(&epi_bars[e], 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_cg<CG>(tmem_slot, T::kTmemCols);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();  // the peer's barriers exist before anything reports to them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_previous();
  int* const error_word = Epi::error_word();
  bool ok = true;

  if (warp == 0) {
    // ---------------- TMA producer (each CTA of a pair loads its own rows) ----------------
    const bool issuer = elect_one();
    uint32_t it = 0;
    for (int w = first; w < L.items && ok; w += step) {
      const Item item = item_of<BM, BN>(L, w);
      const auto& g = L.g[item.g];
      const int m0 = item.m0 + (int)rank * kRows, n0 = item.n0 + (int)rank * T::kBRows;
      const int kt1 = item.kt1, z0 = item.batch * PLANES;
      const bool a_mn = g.a_mn != 0, b_mn = g.b_mn != 0;
      const CUtensorMap *map_a = &g.map_a, *map_b = &g.map_b;
      // a K-major B brings its own rows, an MN-major one whole boxes
      const uint32_t stage_bytes = CG * PLANES * (T::kA + (b_mn ? T::kB : T::kBRows * kBK * 2));
      for (int kt = item.kt0; kt < kt1; ++kt, ++it) {
        const int s = it % STAGES;
        const uint32_t round = it / STAGES;
        if (it >= STAGES && !(ok = wait(&empty[s], (round - 1) & 1, error_word))) break;
        const int k0 = kt * kBK;
        if (issuer) {
          if (rank == 0) mbar_arrive_expect_tx(&full[s], stage_bytes);
#pragma unroll
          for (int p = 0; p < PLANES; ++p) {
            unsigned char* sa = tiles + s * T::kStage + p * (T::kA + T::kB);
            unsigned char* sb = sa + T::kA;
            if (!a_mn) {
              tma_load_3d<CG>(sa, map_a, &full[s], k0, m0, z0 + p);
            } else {
#pragma unroll
              for (int c = 0; c < kRows / 64; ++c)
                tma_load_3d<CG>(sa + c * (kBK * 128), map_a, &full[s], m0 + 64 * c, k0, z0 + p);
            }
            if (!b_mn) {
              tma_load_3d<CG>(sb, map_b, &full[s], k0, n0, z0 + p);
            } else {
#pragma unroll
              for (int c = 0; c < T::kBBlocks; ++c)
                tma_load_3d<CG>(sb + c * (kBK * 128), map_b, &full[s], n0 + 64 * c, k0, z0 + p);
            }
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---------------- UMMA issuer (the pair's leader) ----------------
    const bool issuer = elect_one();
    uint32_t it = 0;
    int j = 0;
    for (int w = first; w < L.items && ok; w += step) {
      const Item item = item_of<BM, BN>(L, w);
      const auto& g = L.g[item.g];
      const uint32_t idesc = idesc_f16(BM, BN, L.bf16 != 0, g.a_mn != 0, g.b_mn != 0);
      // K-major: 8-row groups 1024 B apart, 16 values along k = 32 B. MN-major:
      // 64-wide m (n) blocks kBK * 128 B apart, 8-deep k groups 1024 B apart,
      // 16 along k = two groups.
      const uint32_t a_lbo = g.a_mn ? kBK * 128 : 16, a_step = g.a_mn ? 2048 : 32;
      const uint32_t b_lbo = g.b_mn ? kBK * 128 : 16, b_step = g.b_mn ? 2048 : 32;
      // one accumulator per item, or per sum_slices of it
      const int per = PLANES == 2 ? L.sum_slices : item.kt1 - item.kt0;
      for (int kt0 = item.kt0; kt0 < item.kt1 && ok; kt0 += per, ++j) {
        const int b = j & 1, use = j >> 1;
        const int kt1 = kt0 + per < item.kt1 ? kt0 + per : item.kt1;
        if (use > 0 && !(ok = wait(&acc_empty[b], (use - 1) & 1, error_word))) break;
        tc_fence_after();
        const uint32_t acc = tmem + b * T::kAccCols;
        for (int kt = kt0; kt < kt1; ++kt, ++it) {
          const int s = it % STAGES;
          if (!(ok = wait(&full[s], (it / STAGES) & 1, error_word))) break;
          tc_fence_after();
          const uint32_t sa = smem_u32(tiles + s * T::kStage), sb = sa + T::kA;
          auto da = [&](int p, int kk) {
            return smem_desc(sa + p * (T::kA + T::kB) + kk * a_step, a_lbo, 1024, kSwizzle128B);
          };
          auto db = [&](int p, int kk) {
            return smem_desc(sb + p * (T::kA + T::kB) + kk * b_step, b_lbo, 1024, kSwizzle128B);
          };
          if (issuer) {
            if (PLANES == 2) {
              // the small cross terms first: truncation costs nothing while the
              // sum is 2^-11 of its final size
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk) {
                umma_f16<CG>(acc, da(1, kk), db(0, kk), idesc, kt > kt0 || kk > 0);
                umma_f16<CG>(acc, da(0, kk), db(1, kk), idesc, true);
              }
            }
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              umma_f16<CG>(acc, da(0, kk), db(0, kk), idesc, PLANES == 2 || kt > kt0 || kk > 0);
            umma_commit_cg<CG>(&empty[s]);
          }
          __syncwarp();
        }
        if (issuer) umma_commit_cg<CG>(&acc_full[b]);
        __syncwarp();
      }
    }
  } else if (warp >= 2) {
    // ---------------- epilogue ----------------
    // WARPS / 4 warps share a TMEM lane quarter (32 rows) and take turns with its column blocks.
    const int quarter = warp & 3, e = warp - 2, turn = e >> 2;
    // the accumulator may be overwritten once every epilogue warp has read it; an
    // arrival that also ordered the warp's stores waited 2000 to 3500 clocks for
    // them (8280 x 3072 x 768 with silu and pre-activation: 51 us instead of 44)
    auto release = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) mbar_arrive_remote(&acc_empty[b], 0);
        else mbar_arrive(&acc_empty[b]);
      }
    };
    Epi epi(L, staging + e * Epi::kStagingBytes, &epi_bars[e], lane);
    int j = 0;
    for (int w = first; w < L.items && ok; w += step) {
      const Item item = item_of<BM, BN>(L, w);
      const auto& g = L.g[item.g];
      const int row0 = item.m0 + (int)rank * kRows + quarter * 32;
      epi.begin(g, item, row0);
      if constexpr (PLANES == 2) {
        // 32-column blocks turn, turn + WARPS / 4, ..
        constexpr int STEP = 8 * WARPS, NB = BN / STEP;
        const int c_first = 32 * turn;
        float sum[NB][32];
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
          for (int x = 0; x < 32; ++x) sum[q][x] = 0.0f;
        epi.fetch(item.n0 + c_first);  // beside the wait for the accumulator
        for (int kt = item.kt0; kt < item.kt1; kt += L.sum_slices, ++j) {
          const int b = j & 1;
          if (!(ok = wait(&acc_full[b], (j >> 1) & 1, error_word))) break;
          tc_fence_after();
#pragma unroll
          for (int q = 0; q < 2 * NB; ++q) {
            float v[16];
            tmem_load_16(tmem + b * T::kAccCols + ((uint32_t)(quarter * 32) << 16) + c_first + STEP * (q / 2) + 16 * (q % 2), v);
#pragma unroll
            for (int x = 0; x < 16; ++x) sum[q / 2][16 * (q % 2) + x] += v[x];
          }
          release(b);
        }
        if (!ok) break;
        if (g.splits > 1) {
          // leave the sums, thread by thread; the split that arrives last adds
          // up all of them in split order (the same sum whoever is last)
          const int slot = ((g.first_tile + item.tile) * CG + (int)rank) * WARPS + e;
          float4* parts = L.partial + (int64_t)slot * L.most_splits * (NB * 8 * 32) + lane;
          float4* mine = parts + item.split * (NB * 8 * 32);
#pragma unroll
          for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int x = 0; x < 8; ++x)
              __stcg(mine + (q * 8 + x) * 32,
                     make_float4(sum[q][4 * x], sum[q][4 * x + 1], sum[q][4 * x + 2], sum[q][4 * x + 3]));
          __threadfence();
          __syncwarp();
          unsigned before = 0;
          if (lane == 0) before = atomicAdd(L.counters + slot, 1u);
          before = __shfl_sync(0xffffffffu, before, 0);
          if (before + 1 < (unsigned)g.splits) {
            epi.skip();
            continue;
          }
          __threadfence();
          if (lane == 0) L.counters[slot] = 0;
#pragma unroll
          for (int q = 0; q < NB; ++q) {
#pragma unroll
            for (int x = 0; x < 32; ++x) sum[q][x] = 0.0f;
            for (int z = 0; z < g.splits; ++z) {
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const float4 f = __ldcg(parts + z * (NB * 8 * 32) + (q * 8 + x) * 32);
                sum[q][4 * x] += f.x;
                sum[q][4 * x + 1] += f.y;
                sum[q][4 * x + 2] += f.z;
                sum[q][4 * x + 3] += f.w;
              }
            }
          }
        }
        // a CTA's last tile leaves through the ring, which nothing uses any more
        const bool final = w + step >= L.items;
        static_assert(STAGES * T::kStage / WARPS >= 6 * Epi::kStagingBytes, "room of spread()");
        if (final)
          ok = epi.spread(tiles + e * (STAGES * T::kStage / WARPS), item.n0 + c_first, STEP, NB, error_word);
#pragma unroll
        for (int q = 0; q < NB; ++q) {
          if (!(ok = ok && epi.store(sum[q], item.n0 + c_first + STEP * q, q, error_word))) break;
          if (!final && q + 1 < NB) epi.fetch(item.n0 + c_first + STEP * (q + 1));
        }
      } else {
        // 64-column blocks turn, turn + WARPS / 4, ..
        constexpr int STEP = 16 * WARPS;
        const int b = j & 1;
        const uint32_t acc = tmem + b * T::kAccCols + ((uint32_t)(quarter * 32) << 16);
        if (64 * turn < BN) epi.fetch(item.n0 + 64 * turn);  // beside the wait for the accumulator
        if (!(ok = wait(&acc_full[b], (j >> 1) & 1, error_word))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 64 * turn; c0 < BN; c0 += STEP) {
          if (c0 >= STEP) epi.fetch(item.n0 + c0);
          if (!(ok = epi.store(acc + c0, item.n0 + c0, error_word))) break;
        }
        release(b);
        ++j;
      }
    }
    epi.finish();
  }
  // after a timeout, the copies and products still in flight get time to land
  // before the shared memory and TMEM they use are given back
  if (!ok)
    for (int i = 0; i < 1000; ++i) __nanosleep(2000);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();  // neither CTA leaves while its peer may report to it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_cg<CG>(tmem, T::kTmemCols);
  }
}

// ---- host side ----------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// The driver's encoder needs a current context; threads such as autograd's
// backward workers may not have bound the runtime's primary context yet.
inline int bind_context() {
  int dev = 0;
  CG_CUDA(cudaGetDevice(&dev));
  CG_CUDA(cudaSetDevice(dev));
  return kOk;
}

// 3-D tensor map over `planes` matrices of `rows` x `cols` half-precision values
// (row pitch ld, matrix pitch `stride`, in values). mn: 64-wide boxes of kBK
// rows (k along the rows), else kBK-wide boxes of `box_rows` rows.
inline int make_half_map(CUtensorMap* map, const void* ptr, bool bf16, int64_t rows, int64_t cols, int64_t ld,
                         int64_t planes, int64_t stride, bool mn, int box_rows) {
  auto fn = encode_fn();
  CG_REQUIRE(fn != nullptr, "half gemm: cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * 2), (cuuint64_t)(stride * 2)};
  cuuint32_t box[3] = {(cuuint32_t)kBK, (cuuint32_t)(mn ? kBK : box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  CG_REQUIRE(r == CUDA_SUCCESS, "half gemm: cuTensorMapEncodeTiled failed (%d): rows %lld cols %lld ld %lld", (int)r,
             (long long)rows, (long long)cols, (long long)ld);
  return kOk;
}

// 3-D map of a result or residual: blocks of `width` (128 or 64) bytes x 32
// rows, swizzled over that width.
inline int make_block_map(CUtensorMap* map, CUtensorMapDataType type, int size, int width, const void* ptr,
                          int64_t rows, int64_t cols, int64_t ld, int64_t planes, int64_t stride) {
  auto fn = encode_fn();
  CG_REQUIRE(fn != nullptr, "half gemm: cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * size), (cuuint64_t)(stride * size)};
  cuuint32_t box[3] = {(cuuint32_t)(width / size), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, type, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  CG_REQUIRE(r == CUDA_SUCCESS, "half gemm: cuTensorMapEncodeTiled failed (%d): rows %lld cols %lld ld %lld", (int)r,
             (long long)rows, (long long)cols, (long long)ld);
  return kOk;
}

// Fill in a group's tile counts; the caller has set m, n, k, batch, splits,
// kt_per and lower. Returns its items.
template <int CG, int BN, class EpiArgs>
int64_t plan_group(Group<EpiArgs>& g) {
  constexpr int BM = CG * kRows;
  g.m_tiles = (g.m + BM - 1) / BM;
  g.n_tiles = (g.n + BN - 1) / BN;
  int64_t tiles = (int64_t)g.m_tiles * g.n_tiles;
  if (g.lower) {
    tiles = 0;
    for (int i = 0; i < g.m_tiles; ++i) tiles += lower_tiles_of_row(i, BM, BN, g.n_tiles);
  }
  g.tiles = (int)tiles;
  g.by_tiles = divisor(tiles);
  g.by_batch = divisor(g.batch);
  g.by_band = divisor((int64_t)kBand * g.n_tiles);
  g.by_last = divisor(g.m_tiles % kBand ? g.m_tiles % kBand : kBand);
  return tiles * g.batch * g.splits;
}

template <int CG, int BN, int PLANES, class Epi>
int launch_half_gemm(const LaunchOf<Epi>& L, cudaStream_t stream) {
  using T = Tile<CG, BN, PLANES, Epi>;
  auto kernel = half_gemm_kernel<CG, BN, PLANES, Epi>;
  if (int rc = allow_shared<T>(kernel, T::kBytes)) return rc;
  const int slots = sm_count() / CG;
  return launch_chained("half_gemm", kernel, dim3((unsigned)(CG * (L.items < slots ? L.items : slots))),
                        threads_of(Epi::kWarps), T::kBytes, dim3(CG, 1), stream, L);
}

}  // namespace half
}  // namespace cg
