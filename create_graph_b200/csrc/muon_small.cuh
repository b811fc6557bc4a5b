// Newton-Schulz orthogonalisation of small matrices (shorter side up to 128,
// longer side up to 1024) in one kernel: a cluster of CTAs holds one matrix in
// shared memory through all steps.
//
// CTA r of the cluster owns 128 columns of a wide matrix (128 rows of a tall
// one) as a 128 x 128 tile Z of fp16 planes hi + lo scaled by 2^12, and per step
//   G  = Z Z^T (tall: Z^T Z), summed over the cluster through distributed
//        shared memory: each CTA adds up its share of the partial sums in rank
//        order and writes the planes of its share to every CTA;
//   P  = b A + c A A, formed by every CTA for itself, over A's planes (which lack
//        the diagonal, as the tiled products' do: see SplitEpi in muon.cu);
//   Z <- a Z + P Z (tall: a Z + Z P), in place.
// Each product is 24 UMMAs of 128 x 128 x 16 (lo hi, hi lo and hi hi over k =
// 128), issued by one thread from operands that all lie in shared memory: a
// tile of 128-byte swizzled rows is a K-major operand along its columns and an
// MN-major one along its rows, so Z serves both products as it is stored.
// What bounds it is the chain of 3 products and 3 passes over the tile per
// step, not bandwidth or tensor throughput: 37 us for one to 148 matrices of 128 x
// 128 (2.3 us a product), 61 us with clusters of four (the exchange takes 5 us a
// step); as 17 launches over the batch the same steps took 127 and 150 us.
#pragma once

#include "half_gemm.cuh"

namespace cg {
namespace muon {
namespace small {

constexpr int kSide = 128;
constexpr int kMostCluster = 8;
constexpr int kThreads = 512;  // a warp owns 32 rows x 32 columns of the tile
constexpr int kPlane = kSide * kSide * 2;  // bytes of one plane of a tile
constexpr int kRuns = 24;
constexpr int kGroupsOf4 = kSide * kSide / 4 / kThreads;  // per thread

struct Run {
  const void* x;
  float* momentum;
  void* out;
  int64_t ld_x, ld_momentum, ld_out, stride_x, stride_out;
  int rows, cols, count, first;  // first: place of its first matrix in the launch
  int vec_x, vec_out;            // groups of four along the rows
  float keep, rate;              // out <- keep out + rate X (keep = 0: out is not read)
};

struct Args {
  Run run[kRuns];
  int runs, steps;
  float a, b, c, eps;  // b and c as factors of A's planes and of their square in B's
  float scale;         // of X's planes
  float to_a, from_b;  // X's planes' square to A's planes, B's planes to B
  Momentum rule;
};

struct Smem {
  static constexpr int kZ = 0;                       // two planes
  static constexpr int kA = 2 * kPlane;              // two planes (A, then P)
  static constexpr int kPart = 4 * kPlane;           // 128 x 128 fp32
  static constexpr int kDiagonal = kPart + kSide * kSide * 4;  // of A, fp32; its planes hold zeros there
  static constexpr int kBar = kDiagonal + kSide * 4;
  static constexpr int kBytes = kBar + 256 + 1024 /*alignment*/;
};
static_assert(Smem::kBytes <= 227 * 1024, "shared memory budget");

// Byte offset of value (r, c) of a plane: two slices of 64 columns, rows of 128
// bytes, 16-byte groups swizzled by the row.
__device__ __forceinline__ int plane_at(int r, int c) {
  return (c >> 6) * (kPlane / 2) + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4) + (c & 7) * 2;
}
// Index of the 4-value group g of row r of the fp32 block.
__device__ __forceinline__ int part_at(int r, int g) { return r * 32 + (g ^ (r & 7)); }

__device__ inline uint32_t peer_address(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ inline float4 peer_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ inline void peer_store2(uint32_t addr, uint2 v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
__device__ inline void peer_store_double(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ inline void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }

__device__ __forceinline__ void split4(const float (&v)[4], uint2& hi, uint2& lo) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  const float2 fa = __half22float2(a), fb = __half22float2(b);
  const __half2 c = __floats2half2_rn(v[0] - fa.x, v[1] - fa.y), d = __floats2half2_rn(v[2] - fb.x, v[3] - fb.y);
  hi = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  lo = make_uint2(*reinterpret_cast<const uint32_t*>(&c), *reinterpret_cast<const uint32_t*>(&d));
}

// The plane products of a 128 x 128 x 128 product into TMEM columns `acc`. The
// small cross terms come first: the tensor core truncates as it adds, which
// costs nothing while the sum is 2^-11 of its final size (interleaved with hi hi
// they measured up to 1.5 times the error of torch's fp32 products). K-major
// operands advance along the slices' rows, MN-major ones by 16 rows with their
// two 64-wide blocks a slice apart.
__device__ inline void issue_product(uint32_t acc, uint32_t a, bool a_mn, uint32_t b, bool b_mn) {
  const uint32_t idesc = half::idesc_f16(kSide, kSide, false, a_mn, b_mn);
  auto desc = [](uint32_t base, bool mn, int kk) {
    return mn ? smem_desc(base + kk * 2048, kPlane / 2, 1024, kSwizzle128B)
              : smem_desc(base + (kk >> 2) * (kPlane / 2) + (kk & 3) * 32, 16, 1024, kSwizzle128B);
  };
#pragma unroll
  for (int kk = 0; kk < kSide / 16; ++kk) {
    half::umma_f16<1>(acc, desc(a + kPlane, a_mn, kk), desc(b, b_mn, kk), idesc, kk > 0);
    half::umma_f16<1>(acc, desc(a, a_mn, kk), desc(b + kPlane, b_mn, kk), idesc, true);
  }
#pragma unroll
  for (int kk = 0; kk < kSide / 16; ++kk)
    half::umma_f16<1>(acc, desc(a, a_mn, kk), desc(b, b_mn, kk), idesc, true);
}

// The factor of two of a row's 32 plane values: the same for all, or one each.
struct One {
  float alpha;
  __device__ __forceinline__ float2 pair(int) const { return both(alpha); }
};
struct Each {
  float2 f[16];
  __device__ __forceinline__ float2 pair(int i) const { return f[i]; }
};

// alpha planes(row, 32 columns) + beta v over the planes' own place; returns v.
template <bool AUX, bool STORE, class Factor>
__device__ __forceinline__ void blend_row(unsigned char* planes, int row, int col0, const Factor& alpha, float beta,
                                          float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    unsigned char* at = planes + plane_at(row, col0 + 8 * g);
    if (AUX) {
      const uint4 h = *reinterpret_cast<const uint4*>(at), l = *reinterpret_cast<const uint4*>(at + kPlane);
      const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&hw[i]));
        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&lw[i]));
        float* to = v + 8 * g + 2 * i;
        const float2 r = fma2(alpha.pair(4 * g + i), add2(p, q), mul2(both(beta), make_float2(to[0], to[1])));
        to[0] = r.x;
        to[1] = r.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 * g + e] *= beta;
    }
    if (STORE) {
      uint2 h0, l0, h1, l1;
      const float u0[4] = {v[8 * g], v[8 * g + 1], v[8 * g + 2], v[8 * g + 3]};
      const float u1[4] = {v[8 * g + 4], v[8 * g + 5], v[8 * g + 6], v[8 * g + 7]};
      split4(u0, h0, l0);
      split4(u1, h1, l1);
      *reinterpret_cast<uint4*>(at) = make_uint4(h0.x, h0.y, h1.x, h1.y);
      *reinterpret_cast<uint4*>(at + kPlane) = make_uint4(l0.x, l0.y, l1.x, l1.y);
    }
  }
}

// The value at (r, r) of the planes.
__device__ __forceinline__ float plane_value(const unsigned char* planes, int r) {
  const unsigned char* at = planes + plane_at(r, r);
  return __half2float(*reinterpret_cast<const __half*>(at)) + __half2float(*reinterpret_cast<const __half*>(at + kPlane));
}
__device__ __forceinline__ void put_plane_value(unsigned char* planes, int r, float x) {
  unsigned char* at = planes + plane_at(r, r);
  const __half h = __float2half_rn(x);
  *reinterpret_cast<__half*>(at) = h;
  *reinterpret_cast<__half*>(at + kPlane) = __float2half_rn(x - __half2float(h));
}

// 32 values of a row into the fp32 block.
__device__ __forceinline__ void put_row(float4* part, int row, int col0, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    part[part_at(row, col0 / 4 + g)] = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
}

template <class T, bool MOMENTUM>
__global__ void __launch_bounds__(kThreads, 1) newton_schulz_small_kernel(const __grid_constant__ Args p) {
  extern __shared__ unsigned char smem_raw[];
  // at the same offset in every CTA of the cluster
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~uintptr_t(1023));
  unsigned char *Z = smem + Smem::kZ, *A = smem + Smem::kA;
  float4* part = reinterpret_cast<float4*>(smem + Smem::kPart);
  float* diagonal = reinterpret_cast<float*>(smem + Smem::kDiagonal);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Smem::kBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);
  double* sums = reinterpret_cast<double*>(bar + 2);  // one per CTA of the cluster
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int ranks = (int)gridDim.y, rank = (int)blockIdx.y;  // the cluster spans the grid's y

  int i = 0;
  while (i + 1 < p.runs && (int)blockIdx.x >= p.run[i + 1].first) ++i;
  const Run& run = p.run[i];
  const int matrix = (int)blockIdx.x - run.first;
  const int rows = run.rows, cols = run.cols;
  const bool wide = rows <= cols;
  const int row_off = wide ? 0 : rank * kSide, col_off = wide ? rank * kSide : 0;

  if (tid == 0) {
    mbar_init(bar, 1);
    fence_barrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_slot, kSide);
  tc_fence_before();
  half::cluster_sync_all();  // every CTA runs before a peer reaches into it
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  half::allow_next();
  half::wait_previous();

  // ---- the update u of this CTA's tile, in registers; the norm over the cluster
  float u[kGroupsOf4][4];
  double sum = 0.0;
  {
    const T* x = static_cast<const T*>(run.x) + matrix * run.stride_x;
    float* mom = MOMENTUM ? run.momentum : nullptr;
#pragma unroll
    for (int g = 0; g < kGroupsOf4; ++g) {
      const int at = g * kThreads + tid, row = row_off + (at >> 5), col = col_off + (at & 31) * 4;
      u[g][0] = u[g][1] = u[g][2] = u[g][3] = 0.0f;
      if (row < rows && col < cols) {
        if (run.vec_x) {
          load_four(x + row * run.ld_x + col, u[g]);
          if (MOMENTUM) {
            float4* mp = reinterpret_cast<float4*>(mom + row * run.ld_momentum + col);
            float4 m = *mp;
            m = make_float4(p.rule.next(m.x, u[g][0]), p.rule.next(m.y, u[g][1]), p.rule.next(m.z, u[g][2]),
                            p.rule.next(m.w, u[g][3]));
            *mp = m;
            u[g][0] = p.rule.update(m.x, u[g][0]);
            u[g][1] = p.rule.update(m.y, u[g][1]);
            u[g][2] = p.rule.update(m.z, u[g][2]);
            u[g][3] = p.rule.update(m.w, u[g][3]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (col + e < cols) {
              u[g][e] = load_value(x + row * run.ld_x + col + e);
              if (MOMENTUM) {
                float* mp = mom + row * run.ld_momentum + col + e;
                const float m = p.rule.next(*mp, u[g][e]);
                *mp = m;
                u[g][e] = p.rule.update(m, u[g][e]);
              }
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += (double)u[g][e] * u[g][e];
    }
  }
  sum = block_sum<kThreads / 32>(sum);
  // every CTA's tile in every CTA, added up in rank order
  if (tid < ranks) peer_store_double(peer_address(smem_u32(sums + rank), tid), sum);
  half::cluster_sync_all();
  double total = 0.0;
  for (int r = 0; r < ranks; ++r) total += sums[r];
  const PlaneScale scaled = plane_scale(total, p.eps, p.scale);
#pragma unroll
  for (int g = 0; g < kGroupsOf4; ++g) {
    const int at = g * kThreads + tid;
    const float v[4] = {scaled(u[g][0]), scaled(u[g][1]), scaled(u[g][2]), scaled(u[g][3])};
    uint2 h, l;
    split4(v, h, l);
    unsigned char* to = Z + plane_at(at >> 5, (at & 31) * 4);
    *reinterpret_cast<uint2*>(to) = h;
    *reinterpret_cast<uint2*>(to + kPlane) = l;
  }

  // ---- the steps
  const int quarter = warp & 3, col0 = 32 * (warp >> 2);  // TMEM lanes, 32 columns
  const int row = quarter * 32 + lane;
  const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + col0;
  uint32_t phase = 0;
  // one product: what the threads wrote is visible to the tensor core, and the
  // accumulator to the threads after it
  // (meanwhile: what the threads do beside the tensor core)
  auto product = [&](const unsigned char* a, bool a_mn, const unsigned char* b, bool b_mn, auto meanwhile) {
    fence_proxy_async_all();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      if (half::elect_one()) {
        issue_product(tmem, smem_u32(a), a_mn, smem_u32(b), b_mn);
        umma_commit(bar);
      }
      __syncwarp();
    }
    meanwhile();
    half::wait(bar, phase & 1, &g_muon_error);
    ++phase;
    tc_fence_after();
  };
  const auto nothing = [] {};
  const bool on_diagonal = 32 * quarter == col0;  // this warp's block
  for (int t = 0; t < p.steps; ++t) {
    product(Z, !wide, Z, !wide, nothing);
    float v[32];
    tmem_load_32(acc, v);
    if (ranks == 1) {
      blend_row<false, true>(A, row, col0, One{0.0f}, p.to_a, v);
    } else {
      put_row(part, row, col0, v);
      half::cluster_sync_all();
      // this rank's share of the 4096 groups of four, from every CTA, to every CTA
      const int share = (kSide * 32 + ranks - 1) / ranks, g0 = rank * share;
      const int g1 = g0 + share < kSide * 32 ? g0 + share : kSide * 32;
      for (int at = g0 + tid; at < g1; at += kThreads) {
        const int r = at >> 5, g = at & 31;
        const uint32_t from = smem_u32(part + part_at(r, g));
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int q = 0; q < ranks; ++q) {
          const float4 f = peer_load4(peer_address(from, q));
          x[0] += f.x;
          x[1] += f.y;
          x[2] += f.z;
          x[3] += f.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= p.to_a;
        uint2 h, l;
        split4(x, h, l);
        const uint32_t to = smem_u32(A + plane_at(r, 4 * g));
#pragma unroll 4
        for (int q = 0; q < ranks; ++q) {
          const uint32_t peer = peer_address(to, q);
          peer_store2(peer, h);
          peer_store2(peer + kPlane, l);
        }
      }
      half::cluster_sync_all();
    }
    if (on_diagonal) {  // the diagonal apart
      const float d = plane_value(A, row);
      diagonal[row] = d;
      put_plane_value(A, row, d - d);  // 0, or NaN where it is not finite
    }
    Each factor;
    float more;
    product(A, false, A, false, [&] {  // b + c (d_row + d_column), and the diagonal's own term
      const float c = p.c, mine = diagonal[row], alpha = p.b + c * mine;
      more = mine * alpha;
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const float4 d = *reinterpret_cast<const float4*>(diagonal + col0 + 4 * g);
        factor.f[2 * g] = fma2(both(c), make_float2(d.x, d.y), both(alpha));
        factor.f[2 * g + 1] = fma2(both(c), make_float2(d.z, d.w), both(alpha));
      }
    });
    tmem_load_32(acc, v);
    blend_row<true, true>(A, row, col0, factor, p.c, v);
    if (on_diagonal) put_plane_value(A, row, more + plane_value(A, row));
    if (wide) product(A, false, Z, true, nothing);
    else product(Z, false, A, false, nothing);
    tmem_load_32(acc, v);
    if (t + 1 < p.steps) {
      blend_row<true, true>(Z, row, col0, One{p.a}, p.from_b, v);
    } else {
      blend_row<true, false>(Z, row, col0, One{p.a / p.scale}, p.from_b / p.scale, v);
      put_row(part, row, col0, v);
    }
  }
  tc_fence_before();
  __syncthreads();

  // ---- rows out
  {
    T* out = static_cast<T*>(run.out) + matrix * run.stride_out;
    const float keep = run.keep, rate = run.rate;
#pragma unroll 4
    for (int g = 0; g < kGroupsOf4; ++g) {
      const int at = g * kThreads + tid, r = row_off + (at >> 5), col = col_off + (at & 31) * 4;
      if (r >= rows || col >= cols) continue;
      const float4 f = part[part_at(at >> 5, at & 31)];
      float v[4] = {rate * f.x, rate * f.y, rate * f.z, rate * f.w};
      T* to = out + r * run.ld_out + col;
      const bool read = sizeof(T) == 4 && keep != 0.0f;
      if (run.vec_out) {
        float old[4];
        if (read) {
          load_four(to, old);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += keep * old[e];
        }
        store_four(to, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (col + e < cols) {
            if (read) v[e] += keep * load_value(to + e);
            put_value(to + e, v[e]);
          }
        }
      }
    }
  }
  half::cluster_sync_all();  // no CTA leaves while a peer may still write to it
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kSide);
  }
}

// Clusters that hold a matrix of this shape; 0: it does not fit.
inline int cluster_of(int64_t rows, int64_t cols) {
  const int64_t s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
  if (s > kSide || l > kSide * kMostCluster) return 0;
  const int64_t need = (l + kSide - 1) / kSide;
  return need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
}

template <class T, bool MOMENTUM>
int launch(const Args& p, int matrices, int cluster, cudaStream_t stream) {
  auto kernel = newton_schulz_small_kernel<T, MOMENTUM>;
  struct Tag {};
  if (int rc = half::allow_shared<Tag>(kernel, Smem::kBytes)) return rc;
  return half::launch_chained("newton_schulz small", kernel, dim3((unsigned)matrices, (unsigned)cluster), kThreads,
                              Smem::kBytes, dim3(1, (unsigned)cluster), stream, p);
}

}  // namespace small
}  // namespace muon
}  // namespace cg
