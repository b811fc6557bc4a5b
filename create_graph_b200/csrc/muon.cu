// Newton-Schulz orthogonalisation of matrices, and the optimizer step built on
// it (momentum, orthogonalised update, weight decay).
//
//   X0 = G / max(|G|_F, eps)
//   each step: A = X X^T, B = b A + c A A, X <- a X + B X     (rows <= cols)
//              A = X^T X, B = b A + c A A, X <- a X + X B     (rows > cols)
//   step:  m <- m + (1 - mu) (g - m);  u = nesterov ? g + mu (m - g) : m
//          W <- (1 - lr wd) W - lr scale NS(u)
//
// The iteration multiplies the small singular values by a (3.44) each step, so
// rounding an operand to half precision (2^-11) would come back as percents of
// the weak directions of a low-rank gradient: five steps of fp16 products
// measured 6e-3 and of bf16 products 5e-2 relative error on a 32-direction
// gradient with noise. Every matrix is therefore kept as a pair of fp16 planes
// hi + lo, scaled by 2^12 (entries of X, A and B below 16; lo keeps 22
// significant bits down to entries of 2^-14), and each product is made of the
// three plane products lo hi + hi lo + hi hi in fp32 accumulators: fp32-level
// accuracy (1e-6) at a third of the half-precision rate, twice the rate of three
// tf32 products.
// A and B are symmetric: only tiles that reach the lower triangle are formed,
// and their epilogue stores each value at both places.
// Matrices of one shape are one batch; all shapes of a call share each launch.
// What bounds it: many large matrices (the 85M model's 48: 3.2 ms a step alone, 3.7
// back to back under the power limit) the three products, an update launch
// running at 1.35 PFLOP/s of plane products and a gram launch at 1.2 (its tiles
// cross the diagonal); one matrix (3072 x 768: 209 us) the chain of 15 launches,
// each 10 to 15 us of which 3 to 4 are the way from one launch's end to the next
// one's first product.
#include "half_gemm.cuh"
#include "../../include/cg_b200.h"

namespace cg {
namespace muon {

using namespace cg::sm100;

// device error word of this translation unit's kernels
__device__ int g_muon_error = 0;
// a diagonal of nothing (see SplitEpi)
__device__ __align__(16) float g_zeros[32];

constexpr int kGroups = 8;         // shapes per launch
constexpr int kEntries = 24;       // runs of matrices per prepare launch
constexpr int kMostChunk = 8192;   // elements per block of the prepare passes

// What the planes of X, A and B are scaled by (see scales_of).
struct Scales {
  float x, a, b;
};

struct OutRef {
  void* ptr;
  int64_t ld;
};

// ---- prepare: norms, momentum, split planes -----------------------------------
// A run of `count` matrices of one shape at regular strides.
struct Run {
  const void* x;
  float* momentum;
  void* out;
  __half* planes;  // first matrix's hi plane; (rows, pitch) planes, hi then lo per matrix
  int64_t ld_x, ld_momentum, ld_out, stride_x, stride_out;
  int rows, cols, pitch, count;
  int first_chunk, chunks;  // chunks of one matrix
  half::Divisor by_cols;
  int first_matrix;         // its place in the table of outputs
  int vec;                  // groups of four along the rows
};

struct Prepare {
  Run run[kEntries];
  int runs;
  float eps, mu, scale;
  int nesterov;
  int chunk;                // elements per block
  double* partial;
  OutRef* table;
};

__device__ inline float load_value(const float* p) { return *p; }
__device__ inline float load_value(const __half* p) { return __half2float(*p); }
__device__ inline float load_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ inline void load_four(const float* p, float (&v)[4]) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}
__device__ inline void load_four(const __half* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ inline void load_four(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

__device__ inline void put_value(float* p, float v) { *p = v; }
__device__ inline void put_value(__half* p, float v) { *p = __float2half_rn(v); }
__device__ inline void put_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ inline void store_four(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <class H>
__device__ inline void store_four(H* p, const float (&v)[4]) {
  H h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) put_value(h + e, v[e]);
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
}

struct Momentum {
  float mu;
  int nesterov;
  __device__ float next(float m, float g) const { return m + (1.0f - mu) * (g - m); }
  __device__ float update(float m, float g) const { return nesterov ? m + (1.0f - mu) * (g - m) : m; }
};

// Two fp32 values per instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Sum over a block of WARPS warps in a fixed order.
template <int WARPS>
__device__ inline double block_sum(double s) {
  __shared__ double sums[WARPS];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_down_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) s += sums[w];
  return s;
}

// scale / max(norm, eps), what the planes of an update are scaled by, as a power
// of two and the rest: below a norm of 1.2e-35 the quotient alone leaves fp32's
// range (and a matrix of zeros would become NaN), above 2^138 its normal numbers.
struct PlaneScale {
  float power, rest;
  __device__ __forceinline__ float operator()(float v) const { return v * power * rest; }
};
__device__ inline PlaneScale plane_scale(double squares, float eps, float scale) {
  const double norm = sqrt(squares), d = norm > (double)eps ? norm : (double)eps;
  const double power = d < 0x1p-60 ? 0x1p64 : d > 0x1p60 ? 0x1p-64 : 1.0;
  const float rest = isnan(squares) ? __int_as_float(0x7fc00000) : (float)((double)scale / (d * power));
  return {(float)power, rest};
}

}  // namespace muon
}  // namespace cg

#include "muon_small.cuh"

namespace cg {
namespace muon {

// Bound by HBM: 12 bytes per value of the step and pass (42.5 million values: 77 us,
// 6.6 TB/s, in the first pass, 85 us in the second).
// NORM: advance the momentum and leave each chunk's sum of squares (in 64
// bits: squares of gradients may leave the range of 32). Otherwise: read the
// update again, scale it (plane_scale) and write its planes.
// Block = one chunk of kChunk elements of one matrix.
template <class T, bool MOMENTUM, bool NORM>
__global__ void __launch_bounds__(256) prepare_kernel(const __grid_constant__ Prepare p) {
  half::allow_next_if_few();
  half::wait_previous();
  int i = 0;
  while (i + 1 < p.runs && (int)blockIdx.x >= p.run[i + 1].first_chunk) ++i;
  const Run& run = p.run[i];
  const int at = blockIdx.x - run.first_chunk;
  const int matrix = at / run.chunks, chunk = at % run.chunks;
  const T* x = static_cast<const T*>(run.x) + matrix * run.stride_x;
  float* mom = MOMENTUM ? run.momentum : nullptr;
  const Momentum rule = {p.mu, p.nesterov};
  // the chunk's first place; the others follow by 32-bit steps
  const int64_t n = (int64_t)run.rows * run.cols, e0 = (int64_t)chunk * p.chunk;
  const int row0 = (int)(e0 / run.cols), col0 = (int)(e0 - (int64_t)row0 * run.cols);
  const int size = (int)(e0 + p.chunk < n ? p.chunk : n - e0);
  double sum = 0.0;
  PlaneScale scaled = {};
  __half *hi = nullptr, *lo = nullptr;
  if (NORM) {
    if (chunk == 0 && threadIdx.x == 0) {
      const size_t size = MOMENTUM ? 4 : sizeof(T);
      p.table[run.first_matrix + matrix] = {static_cast<char*>(run.out) + matrix * run.stride_out * size, run.ld_out};
    }
  } else {
    double s = 0.0;
    const double* part = p.partial + run.first_chunk + (int64_t)matrix * run.chunks;
    for (int c = threadIdx.x; c < run.chunks; c += 256) s += part[c];
    s = block_sum<8>(s);
    scaled = plane_scale(s, p.eps, p.scale);
    hi = run.planes + (int64_t)matrix * 2 * run.rows * run.pitch;
    lo = hi + (int64_t)run.rows * run.pitch;
  }
  if (run.vec) {
    // two groups of four per thread and turn, their loads ahead of the stores
    constexpr int U = 2;
    for (int base = 4 * threadIdx.x; base < size; base += U * 4 * 256) {
      int row[U], col[U];
      float v[U][4];
      float4 m[U];
#pragma unroll
      for (int g = 0; g < U; ++g) {
        const int e = base + g * 4 * 256;
        if (e < size) {
          const int down = run.by_cols.div(col0 + e);
          row[g] = row0 + down;
          col[g] = col0 + e - down * run.cols;
          load_four(x + (int64_t)row[g] * run.ld_x + col[g], v[g]);
          if (MOMENTUM) m[g] = *reinterpret_cast<const float4*>(mom + (int64_t)row[g] * run.ld_momentum + col[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < U; ++g) {
        if (base + g * 4 * 256 >= size) break;
        if (MOMENTUM) {
          if (NORM) {
            m[g] = make_float4(rule.next(m[g].x, v[g][0]), rule.next(m[g].y, v[g][1]), rule.next(m[g].z, v[g][2]),
                               rule.next(m[g].w, v[g][3]));
            *reinterpret_cast<float4*>(mom + (int64_t)row[g] * run.ld_momentum + col[g]) = m[g];
          }
          v[g][0] = rule.update(m[g].x, v[g][0]);
          v[g][1] = rule.update(m[g].y, v[g][1]);
          v[g][2] = rule.update(m[g].z, v[g][2]);
          v[g][3] = rule.update(m[g].w, v[g][3]);
        }
        if (NORM) {
#pragma unroll
          for (int q = 0; q < 4; ++q) sum += (double)v[g][q] * v[g][q];
        } else {
          __half h[4], l[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float f = scaled(v[g][q]);
            h[q] = __float2half_rn(f);
            l[q] = __float2half_rn(f - __half2float(h[q]));
          }
          const int64_t o = (int64_t)row[g] * run.pitch + col[g];
          *reinterpret_cast<uint2*>(hi + o) = *reinterpret_cast<const uint2*>(h);
          *reinterpret_cast<uint2*>(lo + o) = *reinterpret_cast<const uint2*>(l);
        }
      }
    }
  } else {
#pragma unroll 4
    for (int e = threadIdx.x; e < size; e += 256) {
      const int down = run.by_cols.div(col0 + e), row = row0 + down, col = col0 + e - down * run.cols;
      float v = load_value(x + (int64_t)row * run.ld_x + col);
      if (MOMENTUM) {
        float* mp = mom + (int64_t)row * run.ld_momentum + col;
        float m = *mp;
        if (NORM) *mp = m = rule.next(m, v);
        v = rule.update(m, v);
      }
      if (NORM) {
        sum += (double)v * v;
      } else {
        const float f = scaled(v);
        const __half h = __float2half_rn(f);
        const int64_t o = (int64_t)row * run.pitch + col;
        hi[o] = h;
        lo[o] = __float2half_rn(f - __half2float(h));
      }
    }
  }
  if (NORM) {
    sum = block_sum<8>(sum);
    if (threadIdx.x == 0) p.partial[blockIdx.x] = sum;
  }
}

// ---- epilogues -----------------------------------------------------------------
struct EpiArgs {
  // blocks of 32 x 32 values of the planes added to the result and of the
  // result's planes (plane index 2 batch + {hi, lo})
  CUtensorMap map_aux, map_out;
  int has_aux;
  float alpha, beta;  // alpha aux + beta accumulator
  float diagonal;     // added on the diagonal (of a symmetric result)
  // diagonals of (batch, up(m, 32)): where the result's goes, its planes getting
  // zeros; the one that operands and aux lack (see SplitEpi)
  float* take;
  const float* apart;
  int lower;          // symmetric result
  // final epilogue: out <- keep out + rate value (keep = 0: out is not read)
  const OutRef* table;
  float keep, rate;
};

// A thread owns one row of the warp's 32 x 32 block. The planes that are added
// come by TMA into the warp's staging block (hi, then lo), where each thread
// reads and overwrites its own row, and the result leaves by TMA; with results
// staged in fp32 and stored as 16-byte pieces by the threads the epilogue
// outlasted the products (the 85M step's 1296 update tiles: 550 us).
struct EpiBase {
  using Args = EpiArgs;
  static constexpr int kGroups = muon::kGroups;
  using L = half::Launch<EpiArgs, kGroups>;
  static constexpr int kWarps = 8;
  static constexpr int kStagingBytes = 2 * 32 * 64;
  static constexpr int kBlock = kStagingBytes;
  const EpiArgs* a;
  unsigned char* staging;
  unsigned char* room = nullptr;  // six blocks more, for the last tile
  uint64_t* bar;
  uint32_t loads = 0;
  int lane, m, n, batch, row0;
  bool pending = false;  // a load has been started and not waited for
  bool later = false;    // the same of the last tile's blocks after its first
  __device__ EpiBase(const L&, unsigned char* staging_, uint64_t* bar_, int lane_)
      : staging(staging_), bar(bar_), lane(lane_) {}
  static __device__ int* error_word() { return &g_muon_error; }
  __device__ void begin(const half::Group<EpiArgs>& g, const half::Item& item, int row) {
    a = &g.epi;
    m = g.m;
    n = g.n;
    batch = item.batch;
    row0 = row;
  }
  // nothing to store: out of range, or above the diagonal, where the mirror
  // block below it writes
  __device__ __forceinline__ bool outside(int col0) const {
    return row0 >= m || col0 >= n || (a->lower && row0 + 31 < col0);
  }
  __device__ __forceinline__ void fetch(int col0) {
    if (outside(col0)) return;
    fence_proxy_async_shared();  // what the threads wrote here before
    __syncwarp();
    if (lane == 0) {
      half::tma_store_wait_read();
      if (a->has_aux) {
        mbar_arrive_expect_tx(bar, kStagingBytes);
        half::tma_load_3d<1>(staging, &a->map_aux, bar, col0, row0, 2 * batch);
        half::tma_load_3d<1>(staging + 2048, &a->map_aux, bar, col0, row0, 2 * batch + 1);
      }
    }
    pending = a->has_aux;
    __syncwarp();
  }
  __device__ __forceinline__ bool arrived(int* error) {
    if (!pending) return true;
    pending = false;
    const bool ok = half::wait(bar, loads & 1, error);
    ++loads;
    return ok;
  }
  __device__ __forceinline__ void skip() { arrived(error_word()); }
  // Memory of the tile's block q: the staging block, or in the last tile one of
  // its own, so that no block waits for the one before it to leave (one gram of
  // 12 x 768 x 768: 24.0 us without, 21.6 with).
  __device__ __forceinline__ unsigned char* block(int q) const {
    return room == nullptr || q == 0 ? staging : room + (2 * q - 1) * kBlock;
  }
  // The last tile: start what blocks 1 .. count - 1 read, all at once.
  __device__ __forceinline__ bool spread(unsigned char* room_, int col0, int step, int count, int* error) {
    room = room_;
    const bool ok = arrived(error);
    if (!a->has_aux) return ok;
    int loads_now = 0;
    for (int q = 1; q < count; ++q) loads_now += !outside(col0 + step * q);
    if (loads_now == 0) return ok;
    if (lane == 0) {
      mbar_arrive_expect_tx(bar, loads_now * kBlock);
      for (int q = 1; q < count; ++q) {
        const int col = col0 + step * q;
        if (outside(col)) continue;
        half::tma_load_3d<1>(block(q), &a->map_aux, bar, col, row0, 2 * batch);
        half::tma_load_3d<1>(block(q) + 2048, &a->map_aux, bar, col, row0, 2 * batch + 1);
      }
    }
    later = true;
    __syncwarp();
    return ok;
  }
  // 16-byte group c (8 values) of row r of plane p
  __device__ __forceinline__ static uint4* group(unsigned char* at, int p, int r, int c) {
    return reinterpret_cast<uint4*>(at + p * 2048 + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  }
  // 32 consecutive values of the diagonal kept apart, zeros where there is none
  __device__ __forceinline__ const float* kept(int first) const {
    return a->apart != nullptr ? a->apart + (int64_t)batch * ((m + 31) & ~31) + first : g_zeros;
  }
  // v <- (alpha + beta (d_row + d_column)) aux + beta v, d the diagonal kept apart
  __device__ __forceinline__ bool values(float (&v)[32], int col0, int q, int* error) {
    const float beta = a->beta;
    if (!a->has_aux) {
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] *= beta;
      return true;
    }
    if (q > 0 && later) {
      pending = true;
      later = false;
    }
    const float* d = kept(col0);
    const float alpha = a->alpha + beta * kept(row0)[lane];
    const bool ok = arrived(error);
    unsigned char* at = block(q);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 d0 = reinterpret_cast<const float4*>(d)[2 * c], d1 = reinterpret_cast<const float4*>(d)[2 * c + 1];
      const float2 dw[4] = {{d0.x, d0.y}, {d0.z, d0.w}, {d1.x, d1.y}, {d1.z, d1.w}};
      const uint4 h = *group(at, 0, lane, c), l = *group(at, 1, lane, c);
      const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&hw[i]));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&lw[i]));
        float* to = v + 8 * c + 2 * i;
        const float2 r = fma2(fma2(both(beta), dw[i], both(alpha)), add2(x, y), mul2(both(beta), make_float2(to[0], to[1])));
        to[0] = r.x;
        to[1] = r.y;
      }
    }
    return ok;
  }
};

// Four 8 x 8 matrices of 16-bit values: lane l gives the address of row l & 7 of
// matrix l >> 3. Read transposed, and written as they are held.
__device__ __forceinline__ void load_transposed(const void* row, uint32_t (&v)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(smem_u32(row))
               : "memory");
}
__device__ __forceinline__ void store_matrices(void* row, const uint32_t (&v)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// The result as planes, for the next product.
// The tensor core truncates as it adds. Of A A that would bite on the diagonal,
// one large square and many small terms, all positive, each cut at the square's
// last bit. So the gram's diagonal d is kept apart in fp32: its planes hold N = A -
// diag(d), and with beta the factor of A A
//   (A A)_ij = (N N)_ij + N_ij (d_i + d_j) + [i = j] d_i^2:
// alpha A + beta A A takes alpha + beta (d_i + d_j) for alpha, and d_i (alpha +
// beta d_i) more on the diagonal. Relative errors (torch's fp32 products): 55 x
// 2364 Gaussian 1.0e-6 (1.4e-6), 55 x 600 1.0e-6 (1.9e-6), 55 orthogonal rows of
// 2364 0.5e-6 (0.7e-6), with d in the product and a fitted factor on it 1.6e-6,
// 2.7e-6 and 3.3e-6. It costs the polynomial's epilogue two reads of d a block:
// 12 x 768 x 768 499 -> 507 us, 3 x 257 x 1031 172 -> 175, the 85M step nothing.
struct SplitEpi : EpiBase {
  using EpiBase::EpiBase;
  __device__ __forceinline__ void put(unsigned char* at, int col, int row) {
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) {
      half::tma_store_3d(&a->map_out, at, col, row, 2 * batch);
      half::tma_store_3d(&a->map_out, at + 2048, col, row, 2 * batch + 1);
    }
  }
  __device__ __forceinline__ bool store(float (&v)[32], int col0, int q, int* error) {
    if (outside(col0)) return true;
    const bool ok = values(v, col0, q, error);
    // hi = fp16(v), lo = fp16(v - hi)
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      const float2 f = __half22float2(h);
      const __half2 l = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
      hi[i] = *reinterpret_cast<const uint32_t*>(&h);
      lo[i] = *reinterpret_cast<const uint32_t*>(&l);
    }
    unsigned char* at = block(q);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      *group(at, 0, lane, c) = make_uint4(hi[4 * c], hi[4 * c + 1], hi[4 * c + 2], hi[4 * c + 3]);
      *group(at, 1, lane, c) = make_uint4(lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
    }
    if (a->lower && row0 == col0) {  // this row's place on the diagonal
      __half* h = reinterpret_cast<__half*>(group(at, 0, lane, lane >> 3)) + (lane & 7);
      __half* l = h + 1024;
      float x = __half2float(*h) + __half2float(*l);
      if (a->take != nullptr) {
        a->take[(int64_t)batch * ((m + 31) & ~31) + row0 + lane] = x;  // 0 beyond m
        x -= x;                                                        // 0, or NaN where it is not finite
      } else {
        const float d = kept(row0)[lane];
        x += d * (a->alpha + a->beta * d) + a->diagonal;
      }
      *h = __float2half_rn(x);
      *l = __float2half_rn(x - __half2float(*h));
    }
    put(at, col0, row0);
    if (a->lower && row0 != col0) {  // the mirror block, transposed 8 x 8 values at a time
      uint32_t t[2][4][4];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int g = 0; g < 4; ++g) load_transposed(group(at, p, lane, g), t[p][g]);
      if (room != nullptr && q < 3) {
        at = room + 2 * q * kBlock;
      } else {  // in the staging block, once it has left
        at = staging;
        if (lane == 0) half::tma_store_wait_read();
        __syncwarp();
      }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int g = 0; g < 4; ++g) store_matrices(group(at, p, 8 * g + (lane & 7), lane >> 3), t[p][g]);
      put(at, row0, col0);
    }
    return ok;
  }
  __device__ void finish() {
    if (lane == 0) half::tma_store_wait();
  }
};

// The last step's result in the caller's matrices.
template <class T>
struct FinalEpi : EpiBase {
  T* out;
  int64_t ld;
  bool vec;
  using EpiBase::EpiBase;
  __device__ void begin(const half::Group<EpiArgs>& g, const half::Item& item, int row) {
    EpiBase::begin(g, item, row);
    const OutRef ref = a->table[batch];
    out = static_cast<T*>(ref.ptr);
    ld = ref.ld;
    constexpr int kGroup = 16 / sizeof(T);
    vec = n % 8 == 0 && ld % kGroup == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  }
  // eight values of a row and what is there (old, zeros where keep is 0)
  __device__ __forceinline__ void put8(const float (&v)[8], const float (&old)[8], float* p) const {
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = a->keep * old[e] + a->rate * v[e];
    float4* q = reinterpret_cast<float4*>(p);
    q[0] = make_float4(o[0], o[1], o[2], o[3]);
    q[1] = make_float4(o[4], o[5], o[6], o[7]);
  }
  template <class H>
  __device__ __forceinline__ void put8(const float (&v)[8], const float (&)[8], H* p) const {
    H h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) put_value(h + e, a->rate * v[e]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  }
  // rows of the caller's matrices: fp32 blocks through shared memory
  __device__ __forceinline__ bool store(float (&v)[32], int col0, int q, int* error) {
    if (outside(col0)) return true;
    const bool ok = values(v, col0, q, error);
    float* stage = reinterpret_cast<float*>(block(q));
    __syncwarp();  // every row of the planes has been read
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<float4*>(stage + half::stage_idx(lane, 4 * q)) =
          make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    __syncwarp();
    if (vec) {
      const int c = (lane & 3) * 8, col = col0 + c;
      if (col < n) {
        T* at = out + (int64_t)(row0 + (lane >> 2)) * ld + col;
        // the four rows' weights at once, ahead of the stores
        float old[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) old[i][e] = 0.0f;
        if constexpr (sizeof(T) == 4) {
          if (a->keep != 0.0f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (row0 + (lane >> 2) + 8 * i >= m) break;
              const float4* q = reinterpret_cast<const float4*>(at + (int64_t)8 * i * ld);
              const float4 x = q[0], y = q[1];
              old[i][0] = x.x; old[i][1] = x.y; old[i][2] = x.z; old[i][3] = x.w;
              old[i][4] = y.x; old[i][5] = y.y; old[i][6] = y.z; old[i][7] = y.w;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (row0 + (lane >> 2) + 8 * i >= m) break;
          float x[8];
          half::stage_read8(stage, (lane >> 2) + 8 * i, c, x);
          put8(x, old[i], at + (int64_t)8 * i * ld);
        }
      }
    } else if (col0 + lane < n) {  // odd pitches: one column per lane
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        const int row = row0 + r;
        if (row >= m) break;
        float x = a->rate * stage[half::stage_idx(r, lane)];
        T* p = out + (int64_t)row * ld + col0 + lane;
        if (sizeof(T) == 4 && a->keep != 0.0f) x += a->keep * *reinterpret_cast<const float*>(p);
        put_value(p, x);
      }
    }
    __syncwarp();
    return ok;
  }
  __device__ void finish() {}
};

// ---- host side -------------------------------------------------------------------
struct Shape {
  int64_t rows, cols, count;
  int64_t s, pitch, spitch;
  __half *x0, *x1, *gram, *poly;
  float* diagonal;  // of the gram, (count, up(s, 32))
  int64_t first_matrix;
};

constexpr int64_t kAlign = 256;
static int64_t up(int64_t n, int64_t to) { return ceil_div<int64_t>(n, to) * to; }

static bool empty(const cg_ns_entry& e) { return e.count == 0 || e.rows == 0 || e.cols == 0; }
// Runs of matrices that a cluster holds in shared memory (muon_small.cuh).
static bool is_small(const cg_ns_entry& e) { return small::cluster_of(e.rows, e.cols) > 0; }

// The shapes of up to kGroups different sizes from entry `from` on; *to = the
// first entry that does not fit.
static int gather_shapes(const cg_ns_args& g, int from, Shape* shapes, int* to) {
  int n = 0, i = from;
  for (; i < g.n; ++i) {
    const cg_ns_entry& e = g.entries[i];
    if (empty(e) || is_small(e)) continue;
    int k = 0;
    while (k < n && (shapes[k].rows != e.rows || shapes[k].cols != e.cols)) ++k;
    if (k == n) {
      if (n == kGroups) break;
      shapes[n].rows = e.rows;
      shapes[n].cols = e.cols;
      shapes[n].count = 0;
      ++n;
    }
    shapes[k].count += e.count;
  }
  *to = i;
  return n;
}

static int64_t chunks_of(int64_t rows, int64_t cols, int chunk) { return ceil_div<int64_t>(rows * cols, chunk); }

enum Step { kGram, kPoly, kUpdate };

// Tile of a launch and the k-splits of its products.
struct Plan {
  int cg, bn, splits;
  int64_t slots, floats;  // with splits: counters and partial sums
};

// By time, in nanoseconds measured on launches of one wave and of several: a
// launch takes `once`, and each wave of tiles `slice` per 64-wide k-slice
// (three products) and `wave`; a split adds the partial sums it leaves and
// reads. `coarse` products (see run) keep the epilogue warps less busy, and their
// updates read no planes. Larger tiles feed the tensor cores best, smaller ones
// and splits of k fill the SMs when there are few: the gram of one 3072 x 768
// matrix takes 49 us on 256 x 256 tiles, 27 us on 256 x 128, 31 us on 128 x 64 and
// 17 us there with k split in three; for twelve of them 53, 54, 115 and (too many
// tiles to split) 115 us.
static Plan plan_of(const Shape* shapes, int n, Step step, bool coarse) {
  struct Tile {
    int cg, bn;
    double slice, coarse_slice, wave, coarse_update, once;
  };
  static const Tile choices[] = {{2, 256, 800, 800, 6200, 2200, 5000},
                                 {2, 128, 395, 395, 3700, 1600, 4300},
                                 {1, 128, 658, 522, 2800, 1300, 4500},
                                 {1, 64, 525, 430, 1400, 750, 4200}};
  const int sms = sm_count();
  Plan best = {2, 256, 1, 0, 0};
  double least = 0.0;
  for (const Tile& t : choices) {
    const int bm = t.cg * half::kRows, slots = sms / t.cg;
    const double slice = coarse ? t.coarse_slice : t.slice;
    const double wave = coarse && step == kUpdate ? t.coarse_update : t.wave;
    int64_t tiles = 0, counts[kGroups], slices[kGroups];
    for (int i = 0; i < n; ++i) {
      const Shape& h = shapes[i];
      const int64_t m = step == kUpdate ? h.rows : h.s, w = step == kUpdate ? h.cols : h.s;
      const int64_t k = step == kGram ? (h.rows < h.cols ? h.cols : h.rows) : h.s;
      const int64_t m_tiles = ceil_div<int64_t>(m, bm), n_tiles = ceil_div<int64_t>(w, t.bn);
      counts[i] = m_tiles * n_tiles;
      if (step != kUpdate) {
        counts[i] = 0;
        for (int64_t r = 0; r < m_tiles; ++r) counts[i] += half::lower_tiles_of_row((int)r, bm, t.bn, (int)n_tiles);
      }
      counts[i] *= h.count;
      slices[i] = ceil_div<int64_t>(k, half::kBK);
      tiles += counts[i];
    }
    for (int splits = 1; splits <= 8; ++splits) {
      double items = 0.0, time = 0.0;
      bool any = splits == 1;
      for (int i = 0; i < n; ++i) {
        const int64_t per = ceil_div<int64_t>(slices[i], splits), parts = ceil_div<int64_t>(slices[i], per);
        any = any || (parts == splits && per >= 2);
        items += (double)counts[i] * parts;
        const double join = parts > 1 ? 1300.0 + t.bn / 64 * (300.0 + 250.0 * parts) : 0.0;
        time += (double)counts[i] * parts * (per * slice + wave + join);
      }
      if (!any) continue;
      const double cost = t.once + ceil(items / slots) * time / items;
      if (least == 0.0 || cost < least) {
        least = cost;
        best.cg = t.cg;
        best.bn = t.bn;
        best.splits = splits;
        best.slots = splits > 1 ? tiles * t.cg * EpiBase::kWarps : 0;
        best.floats = splits > 1 ? tiles * splits * bm * t.bn : 0;
      }
    }
  }
  return best;
}

// The planes hold entries below 16 at a scale of 2^12, the published coefficients'
// by far; others may let X, A or B grow, and get the largest power of two that
// keeps them in fp16's range, up to entries of 10^9. The singular values of X start
// at 1 at most and follow s -> |a s + b s^3 + c s^5|, an entry is no larger than
// the largest of them, and the last step's result is fp32.
static Scales scales_of(const cg_ns_args& g, bool coarse) {
  const double a = g.a, b = g.b, c = g.c;
  double x = 1.0, most_x = 1.0, most_a = 1.0, most_b = 0.0;
  auto larger = [](double m, double v) { return !(fabs(v) < m) ? fmin(fabs(v), 1e9) : m; };
  for (int t = 0; t < g.steps; ++t) {
    const double s1 = x * x;
    most_x = larger(most_x, x);
    most_a = larger(most_a, s1);
    // b s + c s^2 (and a) over [0, s1]: its ends and its vertex
    const double free = coarse ? a : 0.0, vertex = c != 0.0 ? -b / (2.0 * c) : 0.0;
    for (double s : {0.0, vertex > 0.0 && vertex < s1 ? vertex : 0.0, s1})
      most_b = larger(most_b, free + s * (b + c * s));
    // a s + b s^3 + c s^5 over [0, x]: its end and where a + 3 b s^2 + 5 c s^4 = 0
    double next = larger(0.0, x * (a + s1 * (b + c * s1)));
    const double root = 9.0 * b * b - 20.0 * a * c;
    if (root >= 0.0) {
      const double q = -0.5 * (3.0 * b + copysign(sqrt(root), b));
      for (double s : {5.0 * c != 0.0 ? q / (5.0 * c) : 0.0, q != 0.0 ? a / q : 0.0})
        if (s > 0.0 && s < s1) next = larger(next, sqrt(s) * (a + s * (b + c * s)));
    }
    x = next;
  }
  auto scale = [](double most) {
    float s = 4096.0f;
    while (most * s > 61440.0) s *= 0.5f;  // most is 1e9 at the most
    return s;
  };
  return {scale(most_x), scale(most_a), scale(most_b)};
}

struct Buffers {
  double* squares;
  OutRef* table;
  float4* partial;
  unsigned* counters;
  int64_t counter_bytes;
  int chunk;  // elements per block of the prepare passes
};

// Lay the set's buffers out from `base`; returns the bytes they take.
static int64_t layout(Shape* shapes, int n, char* base, Buffers* b) {
  int64_t at = 0, matrices = 0, chunks = 0, elements = 0;
  for (int i = 0; i < n; ++i) elements += shapes[i].count * shapes[i].rows * shapes[i].cols;
  // enough blocks to fill the SMs several times where there are few elements
  const int64_t per = up(ceil_div<int64_t>(elements, (int64_t)sm_count() * 8), 1024);
  b->chunk = (int)(per < kMostChunk ? per : kMostChunk);
  auto take = [&](int64_t bytes) {
    char* p = base == nullptr ? nullptr : base + at;
    at += up(bytes, kAlign);
    return p;
  };
  for (int i = 0; i < n; ++i) {
    Shape& h = shapes[i];
    h.s = h.rows < h.cols ? h.rows : h.cols;
    h.pitch = up(h.cols, 8);
    h.spitch = up(h.s, 8);
    h.first_matrix = matrices;
    matrices += h.count;
    chunks += h.count * chunks_of(h.rows, h.cols, b->chunk);
    const int64_t x = h.count * 2 * h.rows * h.pitch * 2, s = h.count * 2 * h.s * h.spitch * 2;
    h.x0 = reinterpret_cast<__half*>(take(x));
    h.x1 = reinterpret_cast<__half*>(take(x));
    h.gram = reinterpret_cast<__half*>(take(s));
    h.poly = reinterpret_cast<__half*>(take(s));
    h.diagonal = reinterpret_cast<float*>(take(h.count * up(h.s, 32) * (int64_t)sizeof(float)));
  }
  b->squares = reinterpret_cast<double*>(take(chunks * (int64_t)sizeof(double)));
  b->table = reinterpret_cast<OutRef*>(take(matrices * (int64_t)sizeof(OutRef)));
  int64_t floats = 0, counters = 0;
  for (int i = 0; i < 6; ++i) {  // a workspace serves exact and coarse products alike
    const Plan p = plan_of(shapes, n, (Step)(i / 2), i % 2 != 0);
    if (p.slots == 0) continue;
    if (p.floats > floats) floats = p.floats;
    if (p.slots > counters) counters = p.slots;
  }
  b->partial = reinterpret_cast<float4*>(take(floats * (int64_t)sizeof(float)));
  b->counters = reinterpret_cast<unsigned*>(take(counters * (int64_t)sizeof(unsigned)));
  b->counter_bytes = counters * (int64_t)sizeof(unsigned);
  return at;
}

static int64_t workspace_bytes(const cg_ns_args& g) {
  int64_t most = 0;
  Shape shapes[kGroups];
  for (int from = 0, to; from < g.n; from = to) {
    const int n = gather_shapes(g, from, shapes, &to);
    Buffers b;
    const int64_t bytes = layout(shapes, n, nullptr, &b);
    if (bytes > most) most = bytes;
  }
  return most;
}

template <class T, bool MOMENTUM>
static int prepare(const cg_ns_args& g, int from, int to, const Shape* shapes, int n, const Buffers& b, float scale,
                   cudaStream_t s) {
  // both passes need every run's place: the first walks all launches, then the second
  for (int pass = 0; pass < 2; ++pass) {
    int64_t filled[kGroups] = {0};
    int64_t chunks_before = 0;
    Prepare p;
    memset(&p, 0, sizeof(p));
    p.eps = g.eps;
    p.scale = scale;
    p.mu = g.momentum;
    p.nesterov = g.nesterov;
    p.table = b.table;
    p.chunk = b.chunk;
    int64_t chunks = 0;
    auto flush = [&]() -> int {
      if (p.runs == 0) return kOk;
      CG_REQUIRE(chunks < (1ll << 31), "newton_schulz: too many elements in one call");
      p.partial = b.squares + chunks_before;
      auto kernel = pass == 0 ? prepare_kernel<T, MOMENTUM, true> : prepare_kernel<T, MOMENTUM, false>;
      if (int rc = half::launch_chained("newton_schulz prepare", kernel, dim3((unsigned)chunks), 256, 0, dim3(1, 1), s, p))
        return rc;
      chunks_before += chunks;
      p.runs = 0;
      chunks = 0;
      return kOk;
    };
    for (int i = from; i < to; ++i) {
      const cg_ns_entry& e = g.entries[i];
      if (empty(e) || is_small(e)) continue;
      int k = 0;
      while (shapes[k].rows != e.rows || shapes[k].cols != e.cols) ++k;
      const Shape& h = shapes[k];
      Run& r = p.run[p.runs];
      r.x = e.x;
      r.momentum = e.momentum;
      r.out = e.out;
      r.planes = h.x0 + filled[k] * 2 * h.rows * h.pitch;
      r.ld_x = e.ld_x;
      r.ld_momentum = e.ld_momentum;
      r.ld_out = e.ld_out;
      r.stride_x = e.stride_x;
      r.stride_out = e.stride_out;
      r.rows = (int)e.rows;
      r.cols = (int)e.cols;
      r.pitch = (int)h.pitch;
      r.count = (int)e.count;
      r.first_chunk = (int)chunks;
      r.chunks = (int)chunks_of(e.rows, e.cols, b.chunk);
      r.by_cols = half::divisor(e.cols);
      r.first_matrix = (int)(h.first_matrix + filled[k]);
      const uintptr_t mask = 4 * sizeof(T) - 1;
      r.vec = e.cols % 4 == 0 && e.ld_x % 4 == 0 && e.stride_x % 4 == 0 &&
              (reinterpret_cast<uintptr_t>(e.x) & mask) == 0 &&
              (!MOMENTUM || (e.ld_momentum % 4 == 0 && (reinterpret_cast<uintptr_t>(e.momentum) & 15) == 0));
      chunks += e.count * r.chunks;
      filled[k] += e.count;
      if (++p.runs == kEntries)
        if (int rc = flush()) return rc;
    }
    if (int rc = flush()) return rc;
  }
  return kOk;
}

// One launch over all shapes: A = X X^T (X^T X), B = b A + c A A, or
// X' = a X + B X (a X + X B).
template <int CG, int BN, class E>
static int product(const cg_ns_args& g, const Shape* shapes, int n, Step step, const Plan& plan, const Buffers& b,
                   const Scales& scales, bool coarse, bool odd, bool last, float keep, const float* rate,
                   cudaStream_t s) {
  half::LaunchOf<E> L;
  memset(&L, 0, sizeof(L));
  L.partial = b.partial;
  L.counters = b.counters;
  L.most_splits = plan.splits;
  // one slice per accumulator where the epilogue adds them up faster than they
  // come (256-wide tiles' sums take as long as a slice)
  L.sum_slices = coarse ? 4 : BN == 256 ? 2 : 1;
  int64_t items = 0, tiles = 0;
  for (int i = 0; i < n; ++i) {
    const Shape& h = shapes[i];
    auto& G = L.g[i];
    const bool wide = h.rows <= h.cols;
    const __half* x = odd ? h.x1 : h.x0;
    __half* next = odd ? h.x0 : h.x1;
    const int64_t xplane = h.rows * h.pitch, splane = h.s * h.spitch, planes = 2 * h.count;
    int rc = kOk;
    auto map_x = [&](CUtensorMap* map, bool mn, int box) {
      if (rc == kOk) rc = half::make_half_map(map, x, false, h.rows, h.cols, h.pitch, planes, xplane, mn, box);
    };
    auto map_s = [&](CUtensorMap* map, const __half* p, int box) {
      if (rc == kOk) rc = half::make_half_map(map, p, false, h.s, h.s, h.spitch, planes, splane, false, box);
    };
    auto blocks_x = [&](CUtensorMap* map, const __half* p) {
      if (rc == kOk)
        rc = half::make_block_map(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, 64, p, h.rows, h.cols, h.pitch, planes,
                                  xplane);
    };
    auto blocks_s = [&](CUtensorMap* map, const __half* p) {
      if (rc == kOk)
        rc = half::make_block_map(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, 64, p, h.s, h.s, h.spitch, planes, splane);
    };
    const int a_box = half::kRows, b_box = BN / CG;
    EpiArgs& e = G.epi;
    if (step == kGram) {
      G.a_mn = G.b_mn = !wide;
      map_x(&G.map_a, !wide, a_box);
      map_x(&G.map_b, !wide, b_box);
      blocks_s(&e.map_out, h.gram);
      G.m = G.n = (int)h.s;
      G.k = (int)(wide ? h.cols : h.rows);
      e.beta = scales.a / (scales.x * scales.x);
      e.take = h.diagonal;
    } else if (step == kPoly) {
      map_s(&G.map_a, h.gram, a_box);
      map_s(&G.map_b, h.gram, b_box);
      blocks_s(&e.map_aux, h.gram);
      blocks_s(&e.map_out, h.poly);
      G.m = G.n = G.k = (int)h.s;
      e.alpha = g.b * (scales.b / scales.a);
      e.beta = g.c * (scales.b / (scales.a * scales.a));
      e.apart = h.diagonal;
      e.diagonal = coarse ? g.a * scales.b : 0.0f;
    } else {
      if (wide) {
        map_s(&G.map_a, h.poly, a_box);
        map_x(&G.map_b, true, b_box);
        G.b_mn = 1;
      } else {
        map_x(&G.map_a, false, a_box);
        map_s(&G.map_b, h.poly, b_box);
      }
      if (!coarse) blocks_x(&e.map_aux, x);
      if (!last) blocks_x(&e.map_out, next);
      G.m = (int)h.rows;
      G.n = (int)h.cols;
      G.k = (int)h.s;
      e.alpha = g.a;
      e.beta = 1.0f / scales.b;
    }
    if (rc) return rc;
    e.has_aux = step == kPoly || (step == kUpdate && !coarse);
    e.lower = G.lower = step != kUpdate;
    if (last) {  // leaves the planes' scale
      e.table = b.table + h.first_matrix;
      e.alpha /= scales.x;
      e.beta /= scales.x;
      e.keep = keep;
      e.rate = rate[i];
    }
    G.batch = (int)h.count;
    const int64_t kts = ceil_div<int64_t>(G.k, half::kBK);
    G.kt_per = (int)ceil_div<int64_t>(kts, plan.splits);
    G.splits = (int)ceil_div<int64_t>(kts, G.kt_per);
    G.first_item = (int)items;
    G.first_tile = (int)tiles;
    const int64_t mine = half::plan_group<CG, BN>(G);
    items += mine;
    // a group may have fewer splits than planned: its tiles keep the planned room
    tiles += mine / G.splits;
    CG_REQUIRE(items < (1ll << 31), "newton_schulz: too many tiles in one call");
  }
  L.groups = n;
  L.items = (int)items;
  return half::launch_half_gemm<CG, BN, 2, E>(L, s);
}

template <class E>
static int product(const cg_ns_args& g, const Shape* shapes, int n, Step step, const Plan* plans, const Buffers& b,
                   const Scales& scales, bool coarse, bool odd, bool last, float keep, const float* rate,
                   cudaStream_t s) {
  const Plan& p = plans[step];
  if (p.cg == 2 && p.bn == 256) return product<2, 256, E>(g, shapes, n, step, p, b, scales, coarse, odd, last, keep, rate, s);
  if (p.cg == 2) return product<2, 128, E>(g, shapes, n, step, p, b, scales, coarse, odd, last, keep, rate, s);
  if (p.bn == 128) return product<1, 128, E>(g, shapes, n, step, p, b, scales, coarse, odd, last, keep, rate, s);
  return product<1, 64, E>(g, shapes, n, step, p, b, scales, coarse, odd, last, keep, rate, s);
}

static float rate_of(const cg_ns_args& g, bool momentum, int64_t rows, int64_t cols) {
  if (!momentum) return 1.0f;
  const double ratio = (double)rows / (double)cols;
  return (float)(-(double)g.lr * (ratio > 1.0 ? sqrt(ratio) : 1.0));
}

// The small matrices of a call. One launch with the largest cluster where all
// fit the SMs at once (the time is that of one matrix, whatever its size), else
// one per cluster size.
template <class T, bool MOMENTUM>
static int run_small(const cg_ns_args& g, cudaStream_t s) {
  int64_t matrices = 0;
  int largest = 0;
  for (int i = 0; i < g.n; ++i) {
    const cg_ns_entry& e = g.entries[i];
    if (empty(e) || !is_small(e)) continue;
    matrices += e.count;
    const int c = small::cluster_of(e.rows, e.cols);
    if (c > largest) largest = c;
  }
  if (matrices == 0) return kOk;
  const bool together = matrices * largest <= sm_count();
  for (int cluster = together ? largest : 1; cluster <= largest; cluster *= 2) {
    small::Args p;
    memset(&p, 0, sizeof(p));
    p.steps = g.steps;
    const Scales scales = scales_of(g, false);
    p.a = g.a;
    p.b = g.b * (scales.b / scales.a);
    p.c = g.c * (scales.b / (scales.a * scales.a));
    p.eps = g.eps;
    p.scale = scales.x;
    p.to_a = scales.a / (scales.x * scales.x);
    p.from_b = 1.0f / scales.b;
    p.rule = {g.momentum, g.nesterov};
    int64_t in_launch = 0;
    auto flush = [&]() -> int {
      if (p.runs == 0) return kOk;
      CG_REQUIRE(in_launch < (1ll << 31), "newton_schulz: too many matrices in one call");
      if (int rc = small::launch<T, MOMENTUM>(p, (int)in_launch, cluster, s)) return rc;
      p.runs = 0;
      in_launch = 0;
      return kOk;
    };
    for (int i = 0; i < g.n; ++i) {
      const cg_ns_entry& e = g.entries[i];
      if (empty(e) || !is_small(e) || (!together && small::cluster_of(e.rows, e.cols) != cluster)) continue;
      small::Run& r = p.run[p.runs];
      r.x = e.x;
      r.momentum = e.momentum;
      r.out = e.out;
      r.ld_x = e.ld_x;
      r.ld_momentum = e.ld_momentum;
      r.ld_out = e.ld_out;
      r.stride_x = e.stride_x;
      r.stride_out = e.stride_out;
      r.rows = (int)e.rows;
      r.cols = (int)e.cols;
      r.count = (int)e.count;
      r.first = (int)in_launch;
      const uintptr_t mask = 4 * sizeof(T) - 1;
      auto fours = [&](const void* p, int64_t ld, int64_t stride, uintptr_t low) {
        return e.cols % 4 == 0 && ld % 4 == 0 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & low) == 0;
      };
      r.vec_x = fours(e.x, e.ld_x, e.stride_x, mask) && (!MOMENTUM || fours(e.momentum, e.ld_momentum, 0, 15));
      r.vec_out = fours(e.out, e.ld_out, e.stride_out, mask);
      r.keep = MOMENTUM ? 1.0f - g.lr * g.weight_decay : 0.0f;
      r.rate = rate_of(g, MOMENTUM, e.rows, e.cols);
      in_launch += e.count;
      if (++p.runs == small::kRuns)
        if (int rc = flush()) return rc;
    }
    if (int rc = flush()) return rc;
  }
  return kOk;
}

static int run(const cg_ns_args& g, bool momentum, void* stream) {
  cudaStream_t s = as_stream(stream);
  int rc;
  if ((rc = half::bind_context())) return rc;
  if (momentum) rc = run_small<float, true>(g, s);
  else if (g.dtype == CG_F32) rc = run_small<float, false>(g, s);
  else if (g.dtype == CG_F16) rc = run_small<__half, false>(g, s);
  else rc = run_small<__nv_bfloat16, false>(g, s);
  if (rc) return rc;
  Shape shapes[kGroups];
  for (int from = 0, to; from < g.n; from = to) {
    const int n = gather_shapes(g, from, shapes, &to);
    if (n == 0) continue;
    // Results that are rounded to half precision, or added to weights a
    // hundredth to a thousandth part at a time, are formed a little less exactly
    // (1e-6 to 6e-6 relative, 1e-5 on strongly decaying spectra, instead of 1e-6
    // and 3e-6; torch's fp32 products 3e-6 and 5e-6): B carries a on its diagonal,
    // so that X <- B X reads no X beside its operand, and accumulators run for four
    // k-slices instead of one or two, so that the products run further ahead of the
    // epilogue: an update product of the 85M step takes 273 us against 350.
    const bool coarse = momentum || g.dtype != CG_F32;
    const Scales scales = scales_of(g, coarse);
    Buffers b;
    layout(shapes, n, static_cast<char*>(g.workspace), &b);
    if (b.counter_bytes) CG_CUDA(cudaMemsetAsync(b.counters, 0, b.counter_bytes, s));
    if (momentum) rc = prepare<float, true>(g, from, to, shapes, n, b, scales.x, s);
    else if (g.dtype == CG_F32) rc = prepare<float, false>(g, from, to, shapes, n, b, scales.x, s);
    else if (g.dtype == CG_F16) rc = prepare<__half, false>(g, from, to, shapes, n, b, scales.x, s);
    else rc = prepare<__nv_bfloat16, false>(g, from, to, shapes, n, b, scales.x, s);
    if (rc) return rc;
    float rate[kGroups];
    for (int i = 0; i < n; ++i) rate[i] = rate_of(g, momentum, shapes[i].rows, shapes[i].cols);
    const float keep = momentum ? 1.0f - g.lr * g.weight_decay : 0.0f;
    Plan plans[3];
    for (int i = 0; i < 3; ++i) plans[i] = plan_of(shapes, n, (Step)i, coarse);
    for (int t = 0; t < g.steps; ++t) {
      const bool odd = t & 1, last = t == g.steps - 1;
      if ((rc = product<SplitEpi>(g, shapes, n, kGram, plans, b, scales, coarse, odd, false, 0.0f, nullptr, s))) return rc;
      if ((rc = product<SplitEpi>(g, shapes, n, kPoly, plans, b, scales, coarse, odd, false, 0.0f, nullptr, s))) return rc;
      if (!last) rc = product<SplitEpi>(g, shapes, n, kUpdate, plans, b, scales, coarse, odd, false, 0.0f, nullptr, s);
      else if (g.dtype == CG_F32) rc = product<FinalEpi<float>>(g, shapes, n, kUpdate, plans, b, scales, coarse, odd, true, keep, rate, s);
      else if (g.dtype == CG_F16) rc = product<FinalEpi<__half>>(g, shapes, n, kUpdate, plans, b, scales, coarse, odd, true, keep, rate, s);
      else rc = product<FinalEpi<__nv_bfloat16>>(g, shapes, n, kUpdate, plans, b, scales, coarse, odd, true, keep, rate, s);
      if (rc) return rc;
    }
  }
  return kOk;
}

static int checked(const cg_ns_args* args, bool momentum, const char* who) {
  CG_REQUIRE(args != nullptr, "%s: args is NULL", who);
  const cg_ns_args& g = *args;
  CG_REQUIRE(g.n >= 0 && (g.n == 0 || g.entries != nullptr), "%s: bad entries", who);
  CG_REQUIRE(g.dtype == CG_F32 || (!momentum && (g.dtype == CG_F16 || g.dtype == CG_BF16)), "%s: bad dtype %d", who,
             g.dtype);
  CG_REQUIRE(g.steps >= 1, "%s: steps = %d, at least one is needed", who, g.steps);
  CG_REQUIRE(g.eps > 0.0f, "%s: eps must be positive", who);
  for (int i = 0; i < g.n; ++i) {
    const cg_ns_entry& e = g.entries[i];
    CG_REQUIRE(e.rows >= 0 && e.cols >= 0 && e.count >= 0, "%s: entry %d has a negative size", who, i);
    if (empty(e)) continue;
    const int64_t most = (1ll << 30);
    CG_REQUIRE(e.rows < most && e.cols < most && e.count < most, "%s: entry %d is too large", who, i);
    CG_REQUIRE(e.x && e.out && (!momentum || e.momentum), "%s: entry %d has a null buffer", who, i);
    CG_REQUIRE(e.ld_x >= e.cols && e.ld_out >= e.cols && (!momentum || e.ld_momentum >= e.cols),
               "%s: entry %d has a row pitch smaller than its row", who, i);
    CG_REQUIRE(!momentum || e.count == 1, "%s: entry %d: one matrix per entry", who, i);
  }
  const int64_t need = workspace_bytes(g);
  CG_REQUIRE(need == 0 || (g.workspace != nullptr && (reinterpret_cast<uintptr_t>(g.workspace) & (kAlign - 1)) == 0 &&
                           g.workspace_bytes >= need),
             "%s: needs %lld workspace bytes on a 256-byte boundary (cg_newton_schulz_workspace_bytes)", who,
             (long long)need);
  return kOk;
}

int device_error(int* out, bool reset) {
  CG_CUDA(cudaMemcpyFromSymbol(out, g_muon_error, sizeof(int)));
  const int zero = 0;
  if (reset) CG_CUDA(cudaMemcpyToSymbol(g_muon_error, &zero, sizeof(int)));
  return kOk;
}

}  // namespace muon
}  // namespace cg

extern "C" {

int64_t cg_newton_schulz_workspace_bytes(const cg_ns_args* args) {
  if (args == nullptr || args->n <= 0 || args->entries == nullptr) return 0;
  return cg::muon::workspace_bytes(*args);
}

int cg_newton_schulz(const cg_ns_args* args, void* stream) {
  if (int rc = cg::muon::checked(args, false, "newton_schulz")) return rc;
  return cg::muon::run(*args, false, stream);
}

int cg_muon_step(const cg_ns_args* args, void* stream) {
  if (int rc = cg::muon::checked(args, true, "muon_step")) return rc;
  return cg::muon::run(*args, true, stream);
}

}  // extern "C"
