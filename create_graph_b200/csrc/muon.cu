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
// hi + lo, scaled by 2^12 (entries of X, A and B stay below 16; lo keeps 22
// significant bits down to entries of 2^-14), and each product is made of the
// three plane products lo hi + hi lo + hi hi in fp32 accumulators: fp32-level
// accuracy (1e-6) at a third of the half-precision rate, four times the rate of
// three tf32 products.
// A and B are symmetric: only tiles that reach the lower triangle are formed,
// and their epilogue stores each value at both places.
// Matrices of one shape are one batch; all shapes of a call share each launch.
#include "half_gemm.cuh"
#include "../../include/cg_b200.h"

namespace cg {
namespace muon {

// device error word of this translation unit's kernels
__device__ int g_muon_error = 0;

constexpr int kGroups = 8;         // shapes per launch
constexpr int kEntries = 24;       // runs of matrices per prepare launch
constexpr int kChunk = 8192;       // elements per block of the prepare passes
constexpr float kScale = 4096.0f;  // of the stored planes

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
  int first_matrix;         // its place in the table of outputs
  int vec;                  // groups of four along the rows
};

struct Prepare {
  Run run[kEntries];
  int runs;
  float eps, mu;
  int nesterov;
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

struct Momentum {
  float mu;
  int nesterov;
  __device__ float next(float m, float g) const { return m + (1.0f - mu) * (g - m); }
  __device__ float update(float m, float g) const { return nesterov ? m + (1.0f - mu) * (g - m) : m; }
};

// Sum over the block in a fixed order.
__device__ inline double block_sum(double s) {
  __shared__ double sums[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_down_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += sums[w];
  return s;
}

// NORM: advance the momentum and leave each chunk's sum of squares (in 64
// bits: squares of gradients may leave the range of 32). Otherwise: read the
// update again, scale it by 2^12 / max(norm, eps) and write its planes.
// Block = one chunk of kChunk elements of one matrix.
template <class T, bool MOMENTUM, bool NORM>
__global__ void __launch_bounds__(256) prepare_kernel(const __grid_constant__ Prepare p) {
  int i = 0;
  while (i + 1 < p.runs && (int)blockIdx.x >= p.run[i + 1].first_chunk) ++i;
  const Run& run = p.run[i];
  const int at = blockIdx.x - run.first_chunk;
  const int matrix = at / run.chunks, chunk = at % run.chunks;
  const T* x = static_cast<const T*>(run.x) + matrix * run.stride_x;
  float* mom = MOMENTUM ? run.momentum : nullptr;
  const Momentum rule = {p.mu, p.nesterov};
  const int64_t n = (int64_t)run.rows * run.cols;
  const int64_t e0 = (int64_t)chunk * kChunk, e1 = e0 + kChunk < n ? e0 + kChunk : n;
  double sum = 0.0;
  float scale = 0.0f;
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
    s = block_sum(s);
    const double norm = sqrt(s);
    scale = (float)(kScale / (norm > (double)p.eps ? norm : (double)p.eps));
    if (isnan(s)) scale = __int_as_float(0x7fc00000);
    hi = run.planes + (int64_t)matrix * 2 * run.rows * run.pitch;
    lo = hi + (int64_t)run.rows * run.pitch;
  }
  if (run.vec) {
#pragma unroll 2
    for (int64_t e = e0 + 4 * threadIdx.x; e < e1; e += 4 * 256) {
      const int row = (int)(e / run.cols), col = (int)(e % run.cols);
      float v[4];
      load_four(x + row * run.ld_x + col, v);
      if (MOMENTUM) {
        float4* mp = reinterpret_cast<float4*>(mom + row * run.ld_momentum + col);
        float4 m = *mp;
        if (NORM) {
          m = make_float4(rule.next(m.x, v[0]), rule.next(m.y, v[1]), rule.next(m.z, v[2]), rule.next(m.w, v[3]));
          *mp = m;
        }
        v[0] = rule.update(m.x, v[0]);
        v[1] = rule.update(m.y, v[1]);
        v[2] = rule.update(m.z, v[2]);
        v[3] = rule.update(m.w, v[3]);
      }
      if (NORM) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sum += (double)v[q] * v[q];
      } else {
        __half h[4], l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float f = v[q] * scale;
          h[q] = __float2half_rn(f);
          l[q] = __float2half_rn(f - __half2float(h[q]));
        }
        const int64_t o = (int64_t)row * run.pitch + col;
        *reinterpret_cast<uint2*>(hi + o) = *reinterpret_cast<const uint2*>(h);
        *reinterpret_cast<uint2*>(lo + o) = *reinterpret_cast<const uint2*>(l);
      }
    }
  } else {
    for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) {
      const int row = (int)(e / run.cols), col = (int)(e % run.cols);
      float v = load_value(x + row * run.ld_x + col);
      if (MOMENTUM) {
        float* mp = mom + row * run.ld_momentum + col;
        float m = *mp;
        if (NORM) *mp = m = rule.next(m, v);
        v = rule.update(m, v);
      }
      if (NORM) {
        sum += (double)v * v;
      } else {
        const float f = v * scale;
        const __half h = __float2half_rn(f);
        const int64_t o = (int64_t)row * run.pitch + col;
        hi[o] = h;
        lo[o] = __float2half_rn(f - __half2float(h));
      }
    }
  }
  if (NORM) {
    sum = block_sum(sum);
    if (threadIdx.x == 0) p.partial[blockIdx.x] = sum;
  }
}

// ---- epilogues -----------------------------------------------------------------
// Eight hi + lo values of an operand, as loaded.
struct Planes8 {
  uint4 hi, lo;
};
__device__ __forceinline__ void join8(const Planes8& p, float (&v)[8]) {
  const uint32_t h[4] = {p.hi.x, p.hi.y, p.hi.z, p.hi.w}, l[4] = {p.lo.x, p.lo.y, p.lo.z, p.lo.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&l[i]));
    v[2 * i] = a.x + b.x;
    v[2 * i + 1] = a.y + b.y;
  }
}
__device__ __forceinline__ void split8(const float (&v)[8], Planes8& p) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 a = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    const float2 f = __half22float2(a);
    const __half2 b = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    h[i] = *reinterpret_cast<const uint32_t*>(&a);
    l[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  p.hi = make_uint4(h[0], h[1], h[2], h[3]);
  p.lo = make_uint4(l[0], l[1], l[2], l[3]);
}

struct EpiArgs {
  __half* out;        // planes of the result (split epilogue)
  const __half* aux;  // planes added to it, or null
  int64_t out_plane, aux_plane;
  int out_pitch, aux_pitch;
  float alpha, beta;  // alpha aux + beta accumulator
  int lower;          // symmetric result
  // final epilogue: out <- keep out + rate value (keep = 0: out is not read)
  const OutRef* table;
  float keep, rate;
};

struct EpiBase {
  using Args = EpiArgs;
  using L = half::Launch<EpiArgs, muon::kGroups>;
  static constexpr int kGroups = muon::kGroups;
  static constexpr int kWarps = 8;
  static constexpr int kStagingBytes = 32 * 32 * 4;
  float* stage;
  const EpiArgs* a;
  Planes8 aux[4];
  int lane, m, n, batch, row0;
  __device__ EpiBase(const L&, unsigned char* staging, uint64_t*, int lane_)
      : stage(reinterpret_cast<float*>(staging)), lane(lane_) {}
  static __device__ int* error_word() { return &g_muon_error; }
  __device__ void begin(const half::Group<EpiArgs>& g, const half::Item& item, int row) {
    a = &g.epi;
    m = g.m;
    n = g.n;
    batch = item.batch;
    row0 = row;
  }
  // lane -> rows (lane >> 2) + 8 i, columns 8 (lane & 3) .. + 7 of the block;
  // planes have pitches of whole groups of eight
  __device__ void fetch(int col0) {
    if (a->aux == nullptr) return;
    const int col = col0 + (lane & 3) * 8;
    const __half* base = a->aux + batch * 2 * a->aux_plane + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + (lane >> 2) + 8 * i;
      if (row < m && col < n) {
        const __half* at = base + (int64_t)row * a->aux_pitch;
        aux[i].hi = *reinterpret_cast<const uint4*>(at);
        aux[i].lo = *reinterpret_cast<const uint4*>(at + a->aux_plane);
      } else {
        aux[i].hi = aux[i].lo = make_uint4(0, 0, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void put_rows(const float (&v)[32]) {  // row `lane` of the block
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<float4*>(stage + half::stage_idx(lane, 4 * q)) =
          make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    __syncwarp();
  }
  __device__ __forceinline__ void put_back8(int r, int c, const float (&v)[8]) {
    *reinterpret_cast<float4*>(stage + half::stage_idx(r, c)) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(stage + half::stage_idx(r, c + 4)) = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void value8(const Planes8& p, float (&v)[8]) const {
    if (a->aux) {
      float x[8];
      join8(p, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = a->alpha * x[e] + a->beta * v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= a->beta;
    }
  }
  __device__ void finish() {}
};

// The result as planes, for the next product.
struct SplitEpi : EpiBase {
  using EpiBase::EpiBase;
  __device__ __forceinline__ void put8(const float (&v)[8], int64_t row, int col) const {
    __half* at = a->out + batch * 2 * a->out_plane + row * a->out_pitch + col;
    Planes8 p;
    split8(v, p);
    *reinterpret_cast<uint4*>(at) = p.hi;
    *reinterpret_cast<uint4*>(at + a->out_plane) = p.lo;
  }
  __device__ void store(const float (&acc)[32], int col0) {
    if (a->lower && row0 + 31 < col0) return;  // above the diagonal: its mirror block writes it
    put_rows(acc);
    const bool diagonal = a->lower && row0 == col0, mirror = a->lower && !diagonal;
    const int c = (lane & 3) * 8, col = col0 + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + 8 * i, row = row0 + r;
      float v[8];
      if (diagonal) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = stage[half::stage_idx(max(r, c + e), min(r, c + e))];
      } else {
        half::stage_read8(stage, r, c, v);
      }
      value8(aux[i], v);
      if (mirror) put_back8(r, c, v);
      if (row < m && col < n) put8(v, row, col);
    }
    if (mirror) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = (lane >> 2) + 8 * i;  // row of the mirrored block
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = stage[half::stage_idx(c + e, t)];
        if (col0 + t < n && row0 + c < m) put8(v, col0 + t, row0 + c);
      }
    }
    __syncwarp();
  }
};

// The last step's result in the caller's matrices.
__device__ inline void put_value(float* p, float v) { *p = v; }
__device__ inline void put_value(__half* p, float v) { *p = __float2half_rn(v); }
__device__ inline void put_value(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

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
  __device__ __forceinline__ void put8(const float (&v)[8], float* p) const {
    float4* q = reinterpret_cast<float4*>(p);
    const float rate = a->rate, keep = a->keep;
    if (keep != 0.0f) {
      const float4 x = q[0], y = q[1];
      q[0] = make_float4(keep * x.x + rate * v[0], keep * x.y + rate * v[1], keep * x.z + rate * v[2],
                         keep * x.w + rate * v[3]);
      q[1] = make_float4(keep * y.x + rate * v[4], keep * y.y + rate * v[5], keep * y.z + rate * v[6],
                         keep * y.w + rate * v[7]);
    } else {
      q[0] = make_float4(rate * v[0], rate * v[1], rate * v[2], rate * v[3]);
      q[1] = make_float4(rate * v[4], rate * v[5], rate * v[6], rate * v[7]);
    }
  }
  template <class H>
  __device__ __forceinline__ void put8(const float (&v)[8], H* p) const {
    H h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) put_value(h + e, a->rate * v[e]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  }
  __device__ void store(const float (&acc)[32], int col0) {
    put_rows(acc);
    const int c = (lane & 3) * 8, col = col0 + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 2) + 8 * i, row = row0 + r;
      float v[8];
      half::stage_read8(stage, r, c, v);
      value8(aux[i], v);
      if (vec) {
        if (row < m && col < n) put8(v, out + row * ld + col);
      } else {
        put_back8(r, c, v);
      }
    }
    __syncwarp();
    const int cs = col0 + lane;
    if (!vec && cs < n) {  // odd pitches: one column per lane
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        const int row = row0 + r;
        if (row >= m) break;
        float v = a->rate * stage[half::stage_idx(r, lane)];
        T* p = out + row * ld + cs;
        if (sizeof(T) == 4 && a->keep != 0.0f) v += a->keep * *reinterpret_cast<const float*>(p);
        put_value(p, v);
      }
    }
    __syncwarp();
  }
};

// ---- host side -------------------------------------------------------------------
struct Shape {
  int64_t rows, cols, count;
  int64_t s, pitch, spitch;
  __half *x0, *x1, *gram, *poly;
  int64_t first_matrix;
};

constexpr int64_t kAlign = 256;
static int64_t up(int64_t n, int64_t to) { return ceil_div<int64_t>(n, to) * to; }

static bool empty(const cg_ns_entry& e) { return e.count == 0 || e.rows == 0 || e.cols == 0; }

// The shapes of up to kGroups different sizes from entry `from` on; *to = the
// first entry that does not fit.
static int gather_shapes(const cg_ns_args& g, int from, Shape* shapes, int* to) {
  int n = 0, i = from;
  for (; i < g.n; ++i) {
    const cg_ns_entry& e = g.entries[i];
    if (empty(e)) continue;
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

static int64_t chunks_of(int64_t rows, int64_t cols) { return ceil_div<int64_t>(rows * cols, kChunk); }

// Lay the set's buffers out from `base`; returns the bytes they take.
static int64_t layout(Shape* shapes, int n, char* base, double** partial, OutRef** table) {
  int64_t at = 0, matrices = 0, chunks = 0;
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
    chunks += h.count * chunks_of(h.rows, h.cols);
    const int64_t x = h.count * 2 * h.rows * h.pitch * 2, s = h.count * 2 * h.s * h.spitch * 2;
    h.x0 = reinterpret_cast<__half*>(take(x));
    h.x1 = reinterpret_cast<__half*>(take(x));
    h.gram = reinterpret_cast<__half*>(take(s));
    h.poly = reinterpret_cast<__half*>(take(s));
  }
  *partial = reinterpret_cast<double*>(take(chunks * (int64_t)sizeof(double)));
  *table = reinterpret_cast<OutRef*>(take(matrices * (int64_t)sizeof(OutRef)));
  return at;
}

static int64_t workspace_bytes(const cg_ns_args& g) {
  int64_t most = 0;
  Shape shapes[kGroups];
  for (int from = 0, to; from < g.n; from = to) {
    const int n = gather_shapes(g, from, shapes, &to);
    double* partial;
    OutRef* table;
    const int64_t bytes = layout(shapes, n, nullptr, &partial, &table);
    if (bytes > most) most = bytes;
  }
  return most;
}

template <class T, bool MOMENTUM>
static int prepare(const cg_ns_args& g, int from, int to, const Shape* shapes, int n, double* partial, OutRef* table,
                   cudaStream_t s) {
  // both passes need every run's place: the first walks all launches, then the second
  for (int pass = 0; pass < 2; ++pass) {
    int64_t filled[kGroups] = {0};
    int64_t chunks_before = 0;
    Prepare p;
    memset(&p, 0, sizeof(p));
    p.eps = g.eps;
    p.mu = g.momentum;
    p.nesterov = g.nesterov;
    p.table = table;
    int64_t chunks = 0;
    auto flush = [&]() -> int {
      if (p.runs == 0) return kOk;
      CG_REQUIRE(chunks < (1ll << 31), "newton_schulz: too many elements in one call");
      p.partial = partial + chunks_before;
      if (pass == 0) prepare_kernel<T, MOMENTUM, true><<<(unsigned)chunks, 256, 0, s>>>(p);
      else prepare_kernel<T, MOMENTUM, false><<<(unsigned)chunks, 256, 0, s>>>(p);
      CG_LAUNCHED("newton_schulz prepare");
      chunks_before += chunks;
      p.runs = 0;
      chunks = 0;
      return kOk;
    };
    for (int i = from; i < to; ++i) {
      const cg_ns_entry& e = g.entries[i];
      if (empty(e)) continue;
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
      r.chunks = (int)chunks_of(e.rows, e.cols);
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

enum Step { kGram, kPoly, kUpdate };

// One launch over all shapes: A = X X^T (X^T X), B = b A + c A A, or
// X' = a X + B X (a X + X B).
template <int CG, int BN, class E>
static int product(const cg_ns_args& g, const Shape* shapes, int n, Step step, bool odd, const OutRef* table,
                   float keep, const float* rate, cudaStream_t s) {
  half::LaunchOf<E> L;
  memset(&L, 0, sizeof(L));
  int64_t items = 0;
  for (int i = 0; i < n; ++i) {
    const Shape& h = shapes[i];
    auto& G = L.g[i];
    const bool wide = h.rows <= h.cols;
    const __half* x = odd ? h.x1 : h.x0;
    const int64_t xplane = h.rows * h.pitch, splane = h.s * h.spitch, planes = 2 * h.count;
    int rc = kOk;
    auto map_x = [&](CUtensorMap* map, bool mn, int box) {
      if (rc == kOk) rc = half::make_half_map(map, x, false, h.rows, h.cols, h.pitch, planes, xplane, mn, box);
    };
    auto map_s = [&](CUtensorMap* map, const __half* p, int box) {
      if (rc == kOk) rc = half::make_half_map(map, p, false, h.s, h.s, h.spitch, planes, splane, false, box);
    };
    const int a_box = half::kRows, b_box = BN / CG;
    EpiArgs& e = G.epi;
    if (step == kGram) {
      G.a_mn = G.b_mn = !wide;
      map_x(&G.map_a, !wide, a_box);
      map_x(&G.map_b, !wide, b_box);
      G.m = G.n = (int)h.s;
      G.k = (int)(wide ? h.cols : h.rows);
      e.out = h.gram;
      e.beta = 1.0f / kScale;
    } else if (step == kPoly) {
      map_s(&G.map_a, h.gram, a_box);
      map_s(&G.map_b, h.gram, b_box);
      G.m = G.n = G.k = (int)h.s;
      e.out = h.poly;
      e.aux = h.gram;
      e.alpha = g.b;
      e.beta = g.c / kScale;
    } else {
      if (wide) {
        map_s(&G.map_a, h.poly, a_box);
        map_x(&G.map_b, true, b_box);
        G.b_mn = 1;
      } else {
        map_x(&G.map_a, false, a_box);
        map_s(&G.map_b, h.poly, b_box);
      }
      G.m = (int)h.rows;
      G.n = (int)h.cols;
      G.k = (int)h.s;
      e.out = odd ? h.x0 : h.x1;
      e.aux = x;
      e.alpha = g.a;
      e.beta = 1.0f / kScale;
    }
    if (rc) return rc;
    const bool square = step != kUpdate;
    e.lower = G.lower = square;
    e.out_plane = square ? splane : xplane;
    e.out_pitch = (int)(square ? h.spitch : h.pitch);
    e.aux_plane = step == kUpdate ? xplane : splane;
    e.aux_pitch = (int)(step == kUpdate ? h.pitch : h.spitch);
    if (table != nullptr) {  // the last product leaves the planes' scale
      e.table = table + h.first_matrix;
      e.alpha /= kScale;
      e.beta /= kScale;
      e.keep = keep;
      e.rate = rate[i];
    }
    G.batch = (int)h.count;
    G.splits = 1;
    G.kt_per = (int)ceil_div<int64_t>(G.k, half::kBK);
    G.first_item = (int)items;
    items += half::plan_group<CG, BN>(G);
    CG_REQUIRE(items < (1ll << 31), "newton_schulz: too many tiles in one call");
  }
  L.groups = n;
  L.items = (int)items;
  return half::launch_half_gemm<CG, BN, 2, E>(L, s);
}

// Tile of a launch: the larger tiles feed the tensor cores best, the smaller
// ones fill the SMs when there are few.
template <class E>
static int product(const cg_ns_args& g, const Shape* shapes, int n, Step step, bool odd, const OutRef* table,
                   float keep, const float* rate, cudaStream_t s) {
  struct Choice {
    int bm, bn, slots;
    double clocks;
  };
  const int sms = sm_count();
  const Choice choices[] = {{256, 256, sms / 2, 1600}, {256, 128, sms / 2, 900}, {128, 128, sms, 950}, {128, 64, sms, 650}};
  int best = 0;
  double least = 0.0;
  for (int c = 0; c < 4; ++c) {
    double tiles = 0.0, slices = 0.0;
    for (int i = 0; i < n; ++i) {
      const Shape& h = shapes[i];
      const int64_t m = step == kUpdate ? h.rows : h.s, w = step == kUpdate ? h.cols : h.s;
      const int64_t k = step == kGram ? (h.rows < h.cols ? h.cols : h.rows) : h.s;
      double t = (double)ceil_div<int64_t>(m, choices[c].bm) * ceil_div<int64_t>(w, choices[c].bn);
      if (step != kUpdate) {
        t = 0.0;
        for (int64_t r = 0; r < ceil_div<int64_t>(m, choices[c].bm); ++r)
          t += half::lower_tiles_of_row((int)r, choices[c].bm, choices[c].bn, (int)ceil_div<int64_t>(w, choices[c].bn));
      }
      tiles += t * h.count;
      slices += t * h.count * (ceil_div<int64_t>(k, half::kBK) + 2);
    }
    const double waves = ceil(tiles / choices[c].slots);
    const double cost = waves * (slices / tiles) * choices[c].clocks;
    if (c == 0 || cost < least) {
      least = cost;
      best = c;
    }
  }
  switch (best) {
    case 0: return product<2, 256, E>(g, shapes, n, step, odd, table, keep, rate, s);
    case 1: return product<2, 128, E>(g, shapes, n, step, odd, table, keep, rate, s);
    case 2: return product<1, 128, E>(g, shapes, n, step, odd, table, keep, rate, s);
    default: return product<1, 64, E>(g, shapes, n, step, odd, table, keep, rate, s);
  }
}

static int run(const cg_ns_args& g, bool momentum, void* stream) {
  cudaStream_t s = as_stream(stream);
  int rc;
  if ((rc = half::bind_context())) return rc;
  Shape shapes[kGroups];
  for (int from = 0, to; from < g.n; from = to) {
    const int n = gather_shapes(g, from, shapes, &to);
    if (n == 0) continue;
    double* partial;
    OutRef* table;
    layout(shapes, n, static_cast<char*>(g.workspace), &partial, &table);
    if (momentum) rc = prepare<float, true>(g, from, to, shapes, n, partial, table, s);
    else if (g.dtype == CG_F32) rc = prepare<float, false>(g, from, to, shapes, n, partial, table, s);
    else if (g.dtype == CG_F16) rc = prepare<__half, false>(g, from, to, shapes, n, partial, table, s);
    else rc = prepare<__nv_bfloat16, false>(g, from, to, shapes, n, partial, table, s);
    if (rc) return rc;
    float rate[kGroups];
    for (int i = 0; i < n; ++i) {
      const double ratio = (double)shapes[i].rows / (double)shapes[i].cols;
      rate[i] = momentum ? (float)(-(double)g.lr * (ratio > 1.0 ? sqrt(ratio) : 1.0)) : 1.0f;
    }
    const float keep = momentum ? 1.0f - g.lr * g.weight_decay : 0.0f;
    for (int t = 0; t < g.steps; ++t) {
      const bool odd = t & 1, last = t == g.steps - 1;
      if ((rc = product<SplitEpi>(g, shapes, n, kGram, odd, nullptr, 0.0f, nullptr, s))) return rc;
      if ((rc = product<SplitEpi>(g, shapes, n, kPoly, odd, nullptr, 0.0f, nullptr, s))) return rc;
      if (!last) rc = product<SplitEpi>(g, shapes, n, kUpdate, odd, nullptr, 0.0f, nullptr, s);
      else if (g.dtype == CG_F32) rc = product<FinalEpi<float>>(g, shapes, n, kUpdate, odd, table, keep, rate, s);
      else if (g.dtype == CG_F16) rc = product<FinalEpi<__half>>(g, shapes, n, kUpdate, odd, table, keep, rate, s);
      else rc = product<FinalEpi<__nv_bfloat16>>(g, shapes, n, kUpdate, odd, table, keep, rate, s);
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
