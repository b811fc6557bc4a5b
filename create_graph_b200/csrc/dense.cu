// Half-precision dense layer: y = f(x W^T + b) + r in one product with a fused
// epilogue, and the elementwise passes of its first and second derivatives.
//
//   z = x W^T + b,  y = f(z) + r,  f one of identity, relu, silu, gelu (erf)
//   gz = gy f'(z);  dx = gz W;  dW = gz^T x;  db = sum over rows of gz;  dr = gy
//   second order, given cotangents h of gz and hb of db:
//     d gy = (h + hb) f'(z),  d z = (h + hb) gy f''(z)
//
// Products accumulate in fp32 (half_gemm.cuh); the activation, bias and
// residual are applied to the fp32 accumulator, which is rounded to the
// half-precision output once. z is kept in the layer's own type for the
// backward: its rounding (2^-9 relative in bf16) is of the size of the rounding
// of y itself.
#include <math.h>

#include "half_gemm.cuh"
#include "../../include/cg_b200.h"

namespace cg {
namespace dense {

using namespace cg::sm100;
using half::tma_store_wait;
using half::tma_store_wait_read;

// device error word of this translation unit's kernels
__device__ int g_dense_error = 0;

// ---- half-precision values ---------------------------------------------------
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float2 unpack2(uint32_t u, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(w[i], T());
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <class T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
}

// ---- activations ---------------------------------------------------------------
// The hardware's approximate 2^x and reciprocal (about 1e-6 relative together,
// far below the 2^-9 or 2^-11 of the output's rounding; results below 2^-126
// are flushed to zero) keep the epilogue warps ahead of the tensor cores; 2^x
// overflowing to infinity gives 0, the limit. The normal distribution function
// Phi is Abramowitz and Stegun's formula 7.1.26 for erfc (absolute error below
// 1.5e-7), taken on the side where it is small: with CUDA's erff the gelu
// epilogue alone outlasted the products (65536 x 3072 x 768: 509 us against
// 298 us without an activation).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.44269504f;
constexpr float kInvSqrt2Pi = 0.39894228f;

__device__ __forceinline__ float sigmoid(float z) { return rcp_approx(1.0f + exp2_approx(-kLog2e * z)); }

// ---- epilogue --------------------------------------------------------------------
struct EpiArgs {
  // blocks of 32 rows x 128 bytes of y, z, the residual and the fp32 partial
  // tiles (aligned problems)
  CUtensorMap map_y, map_z, map_res, map_partial;
  void* y;
  int64_t ld_y;
  const void* bias;      // (n,) or null
  const void* residual;  // (m, n) or null
  int64_t ld_res;
  void* z;               // (m, n): pre-activation out, or null
  int64_t ld_z;
  float* partial;        // split-K: raw fp32 tiles, (splits, m, n)
  int act;
};

// The larger of two values, NaN if either is (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Beyond +-43 silu, gelu and their derivatives are at their limits.
constexpr float kFar = 43.0f;
// z held to [-most, most]; NaN stays NaN.
__device__ __forceinline__ float hold_nan(float z, float most) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(max_nan(z, -most)), "f"(most));
  return r;
}

// Eight values held to [-43, 43].
__device__ __forceinline__ uint32_t hold_two(uint32_t u, __half) {
  const __half2 far = __float2half2_rn(kFar);
  const __half2 r = __hmin2_nan(__hmax2_nan(*reinterpret_cast<const __half2*>(&u), __hneg2(far)), far);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hold_two(uint32_t u, __nv_bfloat16) {
  const __nv_bfloat162 far = __float2bfloat162_rn(kFar);
  const __nv_bfloat162 r = __hmin2_nan(__hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&u), __hneg2(far)), far);
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <class T>
__device__ __forceinline__ uint4 hold_group(uint4 v) {
  return make_uint4(hold_two(v.x, T()), hold_two(v.y, T()), hold_two(v.z, T()), hold_two(v.w, T()));
}

// Two fp32 values per instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.ftz.f32x2 c, a, b;\n\tmov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.ftz.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// 1 / d for two values of at most 2^62 with one reciprocal: the special
// function unit (16 results per clock and SM) bounds these epilogues, two
// per element of a 128 x 256 tile are 4096 clocks.
__device__ __forceinline__ float2 rcp2(float2 d) {
  const float r = rcp_approx(d.x * d.y);
  return make_float2(r * d.y, r * d.x);
}

// silu of two values. z is held at -43 and above, where silu is -9e-18, so that
// 2^-x stays below 2^62 for the pair's reciprocal; below it, down to -infinity,
// silu is smaller still and 0 in the limit. A NaN stays in z and does not enter
// the reciprocal, which is the other value's too.
__device__ __forceinline__ float2 silu2(float2 z) {
  z = make_float2(max_nan(z.x, -kFar), max_nan(z.y, -kFar));
  const float2 x = mul2(z, both(-kLog2e));
  const float2 e = make_float2(exp2_approx(fminf(x.x, 62.0f)), exp2_approx(fminf(x.y, 62.0f)));
  return mul2(z, rcp2(make_float2(1.0f + e.x, 1.0f + e.y)));
}
// gelu of two values: max(z, 0) - |z| (1 - Phi(|z|)). The tail 1 - Phi goes
// through one reciprocal and no exponential: its 32nd root's reciprocal grows
// like exp(z^2 / 64) and is a polynomial of degree 7 to 5e-7 (minimax relative
// error on [0, 6.5], fitted to the normal distribution's logarithm), so the tail
// is right to 2e-5 there, far below the rounding to 2^-9 or 2^-11, and to 1e-2
// at 8, where gelu is 5e-15; at -12 and beyond it is held at 2^-107. A NaN goes
// through the positive part alone: in the tail it would reach the other value
// of the pair through the shared reciprocal.
__device__ __forceinline__ float2 gelu2(float2 z) {
  const float2 a = make_float2(fmaxf(-fabsf(z.x), -12.0f), fmaxf(-fabsf(z.y), -12.0f));
  float2 p = fma2(a, both(-1.763030895e-07f), both(-2.591498287e-06f));
  p = fma2(a, p, both(-3.504646520e-05f));
  p = fma2(a, p, both(-1.234932133e-04f));
  p = fma2(a, p, both(-1.482319436e-03f));
  p = fma2(a, p, both(1.043934096e-02f));
  p = fma2(a, p, both(-2.549119666e-02f));
  p = fma2(a, p, both(1.021896601f));
  p = mul2(p, p);
  p = mul2(p, p);
  p = mul2(p, p);
  p = mul2(p, p);           // at most 2^54
  const float2 r = rcp2(p);  // the tail's square root
  return fma2(mul2(a, r), r, make_float2(max_nan(z.x, 0.0f), max_nan(z.y, 0.0f)));
}

// f' of two values within [-43, 43] (hold_nan, hold_group): at the bounds f' is 0
// to 1e-17 or 1, its limits at the infinities, so a pre-activation that left the
// range of its type and was kept as -infinity (fp16 below -65504) has the gradient
// 0 that goes with its output 0. silu's 1 - s is off by an ulp, times z: 5e-6 at
// the most. One reciprocal each: these passes wait for memory, not for the special
// function unit, and neither value depends on the other.
__device__ __forceinline__ float2 rcp_each(float2 d) { return make_float2(rcp_approx(d.x), rcp_approx(d.y)); }
__device__ __forceinline__ float2 silu_grad2(float2 z) {
  const float2 x = mul2(z, both(-kLog2e));
  const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
  const float2 s = rcp_each(fma2(e, both(1.0f), both(1.0f)));
  // s (1 + z (1 - s)) = s + (z s - z s s)
  const float2 zs = mul2(z, s);
  return fma2(fma2(zs, make_float2(-s.x, -s.y), zs), both(1.0f), s);
}
__device__ __forceinline__ float2 gelu_grad2(float2 z) {
  constexpr float kP = 0.3275911f * 0.70710678f;
  const float2 t = rcp_each(make_float2(fmaf(fabsf(z.x), kP, 1.0f), fmaf(fabsf(z.y), kP, 1.0f)));
  const float2 u = mul2(mul2(z, z), both(-0.5f * kLog2e));
  const float2 e = make_float2(exp2_approx(u.x), exp2_approx(u.y));
  float2 p = fma2(t, both(0.5307027145f), both(-0.7265760135f));
  p = fma2(t, p, both(0.7107068705f));
  p = fma2(t, p, both(-0.142248368f));
  p = fma2(t, p, both(0.127414796f));
  // Phi(z) = 1/2 + sign(z) (1/2 - tail)
  const float2 h = fma2(mul2(p, t), make_float2(-e.x, -e.y), both(0.5f));
  const float2 signed_h = make_float2(copysignf(h.x, z.x), copysignf(h.y, z.y));
  return fma2(fma2(mul2(z, both(kInvSqrt2Pi)), e, both(0.5f)), both(1.0f), signed_h);
}
// f' of one value within the same bounds.
__device__ __forceinline__ float act_grad(float z, int kind) {
  if (kind == CG_ACT_SILU) return silu_grad2(both(z)).x;
  if (kind == CG_ACT_GELU) return gelu_grad2(both(z)).x;
  if (kind == CG_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  return 1.0f;
}
// f'' of one value within the same bounds, where its square stays in fp32.
__device__ __forceinline__ float act_grad2(float z, int kind) {
  if (kind == CG_ACT_SILU) {
    const float s = sigmoid(z);
    return s * (1.0f - s) * (2.0f + z * (1.0f - 2.0f * s));
  }
  if (kind == CG_ACT_GELU) return kInvSqrt2Pi * exp2_approx(z * z * (-0.5f * kLog2e)) * (2.0f - z * z);
  return 0.0f;
}
// g <- g f'(z), z within [-43, 43]; the branch on the kind is outside the loop.
template <int N>
__device__ __forceinline__ void act_grad_all(float (&g)[N], const float (&z)[N], int kind) {
  if (kind == CG_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] = z[e] > 0.0f ? g[e] : 0.0f * g[e];
  } else if (N % 2 == 0 && (kind == CG_ACT_SILU || kind == CG_ACT_GELU)) {
#pragma unroll
    for (int e = 0; e + 1 < N; e += 2) {
      const float2 x = make_float2(z[e], z[e + 1]);
      const float2 d = kind == CG_ACT_SILU ? silu_grad2(x) : gelu_grad2(x);
      g[e] *= d.x;
      g[e + 1] *= d.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) g[e] *= act_grad(z[e], kind);
  }
}

// f of one value, as act_all's.
__device__ __forceinline__ float act(float z, int kind) {
  if (kind == CG_ACT_SILU) return silu2(both(z)).x;
  if (kind == CG_ACT_GELU) return gelu2(both(z)).x;
  if (kind == CG_ACT_RELU) return z < 0.0f ? 0.0f : z;
  return z;
}
// f applied to a thread's values; the branch on the kind is outside the loop.
template <int N>
__device__ __forceinline__ void act_all(float (&v)[N], int kind) {
  if (kind == CG_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 y = silu2(make_float2(v[e], v[e + 1]));
      v[e] = y.x;
      v[e + 1] = y.y;
    }
  } else if (kind == CG_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 y = gelu2(make_float2(v[e], v[e + 1]));
      v[e] = y.x;
      v[e + 1] = y.y;
    }
  } else if (kind == CG_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = act(v[e], CG_ACT_RELU);
  }
}

struct EpiBase {
  using Args = EpiArgs;
  static constexpr int kGroups = 2;  // dx and dW of a backward share a launch
  using L = half::Launch<EpiArgs, kGroups>;
  const EpiArgs* p;
  unsigned char* staging;
  uint64_t* bar;
  int lane, m, n, split, row0;
  __device__ EpiBase(const L&, unsigned char* staging_, uint64_t* bar_, int lane_)
      : staging(staging_), bar(bar_), lane(lane_) {}
  static __device__ int* error_word() { return &g_dense_error; }
  __device__ void begin(const half::Group<EpiArgs>& g, const half::Item& item, int row) {
    p = &g.epi;
    m = g.m;
    n = g.n;
    split = item.split;
    row0 = row;
  }
};

// Aligned problems (n and every pitch a multiple of 8, 16-byte aligned bases).
// A thread owns one row of the warp's 32 x 64 block: bias, activation and
// residual are applied in registers, the rounded row goes to a 128-byte
// swizzled block in shared memory and TMA writes the block. The residual comes
// by TMA into the same block beforehand (each thread reads and overwrites its
// own row); the pre-activation follows through the same block, read from TMEM
// once more. Sixteen warps, one block each of a 256-wide tile, hide one
// another's latencies (65536 x 3072 x 768 with gelu: 287 us, eight warps 323 us,
// before the activation's and the barriers' later steps: 255 to 270 us).
// Against staging fp32 blocks and storing 64-byte row segments from the
// threads this halves the shared-memory traffic that competes with the
// operands: 65536 x 3072 x 768 with no activation takes 230 us (298 us before,
// 203 us without any stores), with a residual 275, with gelu, residual and
// pre-activation 340 to 370 (three 400 MB streams: 200 us at the copy rate; the
// activation's arithmetic, the block's second use for the pre-activation and the
// power limit are what is left).
template <class T>
struct BlockEpi : EpiBase {
  static constexpr int kWarps = 16;
  static constexpr int kStagingBytes = 4096;
  using EpiBase::EpiBase;
  uint32_t loads = 0;

  __device__ __forceinline__ bool outside(int col0) const { return row0 >= m || col0 >= n; }
  // 16-byte group c of this thread's row of the block
  __device__ __forceinline__ uint4* group(int c) const {
    return reinterpret_cast<uint4*>(staging + lane * 128 + ((c ^ (lane & 7)) << 4));
  }
  // the block is free once the last store has read it
  __device__ __forceinline__ void fetch(int col0) {
    if (outside(col0)) return;
    if (lane == 0) {
      tma_store_wait_read();
      if (p->residual != nullptr && p->partial == nullptr) {
        mbar_arrive_expect_tx(bar, 4096);
        half::tma_load_3d<1>(staging, &p->map_res, bar, col0, row0, 0);
      }
    }
    __syncwarp();
  }
  __device__ __forceinline__ void put(const CUtensorMap* map, int col, int z) {
    fence_proxy_async_shared();
    __syncwarp();
    if (lane == 0) half::tma_store_3d(map, staging, col, row0, z);
  }
  __device__ __forceinline__ void reuse() {
    if (lane == 0) tma_store_wait_read();
    __syncwarp();
  }
  // 32 pre-activations of this thread's row
  __device__ __forceinline__ void load(uint32_t acc, int col0, float (&v)[32]) const {
    uint4 b[4];  // on their way beside the accumulator's
    if (p->bias) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        b[c] = col0 + 8 * c < n ? __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p->bias) + col0 + 8 * c))
                                : make_uint4(0, 0, 0, 0);
    }
    tmem_load_32(acc, v);
    if (p->bias == nullptr) return;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float f[8];
      unpack8<T>(b[c], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[8 * c + e] += f[e];
    }
  }
  __device__ __forceinline__ bool store(uint32_t acc, int col0, int* error) {
    if (outside(col0)) return true;
    if (p->partial != nullptr) {
#pragma unroll 1
      for (int h = 0; h < 2 && col0 + 32 * h < n; ++h) {
        float v[32];
        tmem_load_32(acc + 32 * h, v);
        if (h == 1) reuse();
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *group(c) = make_uint4(__float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]),
                                 __float_as_uint(v[4 * c + 2]), __float_as_uint(v[4 * c + 3]));
        put(&p->map_partial, col0 + 32 * h, split);
      }
      return true;
    }
    bool ok = true;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[32];
      load(acc + 32 * h, col0 + 32 * h, v);
      act_all(v, p->act);
      if (p->residual && h == 0) {
        ok = half::wait(bar, loads & 1, error);
        ++loads;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float o[8] = {v[8 * c],     v[8 * c + 1], v[8 * c + 2], v[8 * c + 3],
                      v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]};
        uint4* at = group(4 * h + c);
        if (p->residual) {
          float r[8];
          unpack8<T>(*at, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] += r[e];
        }
        *at = pack8<T>(o);
      }
    }
    put(&p->map_y, col0, 0);
    if (p->z) {
      reuse();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[32];
        load(acc + 32 * h, col0 + 32 * h, v);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float o[8] = {v[8 * c],     v[8 * c + 1], v[8 * c + 2], v[8 * c + 3],
                              v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]};
          *group(4 * h + c) = pack8<T>(o);
        }
      }
      put(&p->map_z, col0, 0);
    }
    return ok;
  }
  __device__ void finish() {
    if (lane == 0) tma_store_wait();
  }
};

// Any pitch and alignment: bias and activation are applied a row per thread, then
// the block is transposed through shared memory and stored one column per lane
// (z the same way before the activation); the residual of a 32 x 32 block is read
// before the accumulator is waited for. 4099 x 1031 x 515 fp16 with gelu, residual
// and z: 42 us (47 with the activation applied value by value behind the
// transpose), its gradients dx + dW 40 us (47), against 8 us of bytes: the
// two-byte stores, 64 bytes a warp and across sectors, are what is left.
template <class T>
struct PlainEpi : EpiBase {
  static constexpr int kWarps = 16;
  static constexpr int kStagingBytes = 32 * 32 * 4;
  using EpiBase::EpiBase;
  T res[32];
  __device__ __forceinline__ void fetch32(int col0) {
    if (p->residual == nullptr || p->partial != nullptr) return;
    const int col = col0 + lane;
    const T* at = static_cast<const T*>(p->residual) + (int64_t)row0 * p->ld_res + col;
#pragma unroll
    for (int r = 0; r < 32; ++r)
      if (col < n && row0 + r < m) res[r] = at[r * p->ld_res];
  }
  __device__ void fetch(int col0) { fetch32(col0); }
  static __device__ __forceinline__ void finish1(const EpiArgs& a, float v, float residual, int64_t row, int col) {
    if (a.z) static_cast<T*>(a.z)[row * a.ld_z + col] = from_float<T>(v);
    static_cast<T*>(a.y)[row * a.ld_y + col] = from_float<T>(act(v, a.act) + residual);
  }
  // a thread's row of the block goes to shared memory, a lane's column comes back
  __device__ __forceinline__ void put(const float (&v)[32]) const {
    float* stage = reinterpret_cast<float*>(staging);
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<float4*>(stage + half::stage_idx(lane, 4 * q)) =
          make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    __syncwarp();
  }
  template <class Out>
  __device__ __forceinline__ void columns(Out* at, int64_t ld, bool add) const {
    const float* stage = reinterpret_cast<const float*>(staging);
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      if (row0 + r >= m) break;
      float x = stage[half::stage_idx(r, lane)];
      if (add) x += to_float(res[r]);
      if constexpr (sizeof(Out) == 4) at[r * ld] = x;
      else at[r * ld] = from_float<T>(x);
    }
  }
  __device__ bool store(uint32_t acc, int col0, int*) {
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      const int col = col0 + 32 * h + lane;
      const bool mine = col < n;
      if (h == 1) fetch32(col0 + 32);
      float v[32];
      tmem_load_32(acc + 32 * h, v);
      if (p->partial != nullptr) {
        put(v);
        if (mine) columns(p->partial + ((int64_t)split * m + row0) * n + col, n, false);
        continue;
      }
      if (p->bias) {
        const float b = mine ? to_float(static_cast<const T*>(p->bias)[col]) : 0.0f;
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] += __shfl_sync(0xffffffffu, b, c);
      }
      if (p->z) {
        put(v);
        if (mine) columns(static_cast<T*>(p->z) + (int64_t)row0 * p->ld_z + col, p->ld_z, false);
      }
      act_all(v, p->act);
      put(v);
      if (mine) columns(static_cast<T*>(p->y) + (int64_t)row0 * p->ld_y + col, p->ld_y, p->residual != nullptr);
    }
    return true;
  }
  __device__ void finish() {}
};

// Joins the k-splits in split order (the same sum every run) and finishes the
// elements as the epilogue does; VEC: groups of eight columns.
template <class T, bool VEC>
__global__ void join_splits_kernel(const __grid_constant__ EpiArgs a, int splits, int m, int n) {
  half::allow_next_if_few();
  half::wait_previous();
  const int64_t mn = (int64_t)m * n, stride = (int64_t)gridDim.x * blockDim.x;
  const int64_t first = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (VEC) {
    const int n8 = n / 8;
    for (int64_t i = first; i < mn / 8; i += stride) {
      const int64_t row = i / n8;
      const int col = (int)(i % n8) * 8;
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0}, x[8];
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const float4* p = reinterpret_cast<const float4*>(a.partial + s * mn + i * 8);
        const float4 f = __ldg(p), g = __ldg(p + 1);
        v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
        v[4] += g.x; v[5] += g.y; v[6] += g.z; v[7] += g.w;
      }
      if (a.bias) {
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.bias) + col)), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += x[e];
      }
      if (a.z) *reinterpret_cast<uint4*>(static_cast<T*>(a.z) + row * a.ld_z + col) = pack8<T>(v);
      act_all(v, a.act);
      if (a.residual) {
        unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.residual) + row * a.ld_res + col), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += x[e];
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.ld_y + col) = pack8<T>(v);
    }
  } else {
    for (int64_t i = first; i < mn; i += stride) {
      float v = 0.0f;
      for (int s = 0; s < splits; ++s) v += a.partial[s * mn + i];
      const int64_t row = i / n;
      const int col = (int)(i % n);
      if (a.bias) v += to_float(static_cast<const T*>(a.bias)[col]);
      PlainEpi<T>::finish1(
          a, v, a.residual ? to_float(static_cast<const T*>(a.residual)[row * a.ld_res + col]) : 0.0f, row, col);
    }
  }
}

// ---- elementwise passes of the derivatives -----------------------------------------
// Bound by HBM: three streams of rows x cols values (65536 x 3072 bf16: 1.2 GB with
// silu in 199 us, 6.1 TB/s, 93% of the measured copy rate, with gelu in 212 us;
// 8280 x 3072 32 and 34 us).
// gz = gy f'(z) and the column sums of gz (the bias gradient) in one pass over
// gy and z: block (x, y) owns 32 x V columns and the rows of chunk y; its eight
// warps walk the rows, each lane adding up V columns in fp32, and the warps'
// sums meet in shared memory in warp order. V = 8 where the columns are whole
// groups, read value by value if the rows are not ALIGNED, so that neither gz nor
// the sums depend on where they lie; else 1. Four
// blocks an SM with two rows of a warp in flight: with five or six the registers
// spill (229 and 267 us with silu), with three or two too little is in flight (205
// and 245), one row at a time waits (236).
template <bool ALIGNED, class T>
__device__ __forceinline__ uint4 load_group(const T* p) {
  if (ALIGNED) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool ALIGNED, class T>
__device__ __forceinline__ void store_group(T* p, uint4 v) {
  if (ALIGNED) {
    *reinterpret_cast<uint4*>(p) = v;
    return;
  }
  unsigned short* h = reinterpret_cast<unsigned short*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = (unsigned short)w[i];
    h[2 * i + 1] = (unsigned short)(w[i] >> 16);
  }
}
template <class T, int V, bool ALIGNED>
__global__ void __launch_bounds__(256, V == 8 && ALIGNED ? 4 : 1) act_grad_kernel(const T* __restrict__ gy, int64_t ld_gy,
                                                       const T* __restrict__ z, int64_t ld_z, T* __restrict__ gz,
                                                       int64_t ld_gz, int rows, int cols, int kind, int rows_per,
                                                       float* __restrict__ partial, T* __restrict__ db) {
  half::allow_next_if_few();
  half::wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + lane) * V;
  const int r0 = blockIdx.y * rows_per, r1 = min(rows, r0 + rows_per);
  float sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = 0.0f;
  if constexpr (V == 8) {
    // two rows' loads on their way before the first is used
    if (col < cols) {
      for (int64_t r = r0 + warp; r < r1; r += 16) {
        uint4 ga[2], za[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (r + 8 * i >= r1) break;
          ga[i] = load_group<ALIGNED>(gy + (r + 8 * i) * ld_gy + col);
          if (gz) za[i] = load_group<ALIGNED>(z + (r + 8 * i) * ld_z + col);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (r + 8 * i >= r1) break;
          float g[8], x[8];
          unpack8<T>(ga[i], g);
          if (gz) {
            unpack8<T>(hold_group<T>(za[i]), x);
            act_grad_all(g, x, kind);
            store_group<ALIGNED>(gz + (r + 8 * i) * ld_gz + col, pack8<T>(g));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += g[e];
        }
      }
    }
  } else if (col < cols) {
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      float g[1] = {to_float(gy[r * ld_gy + col])};
      if (gz) {
        const float x[1] = {hold_nan(to_float(z[r * ld_z + col]), kFar)};
        act_grad_all(g, x, kind);
        gz[r * ld_gz + col] = from_float<T>(g[0]);
      }
      sum[0] += g[0];
    }
  }
  if (partial == nullptr && db == nullptr) return;
  __shared__ float sums[8][32 * V];
#pragma unroll
  for (int e = 0; e < V; ++e) sums[warp][lane * V + e] = sum[e];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * V; c += 256) {
    const int at = blockIdx.x * 32 * V + c;
    if (at >= cols) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][c];
    if (db) db[at] = from_float<T>(s);  // the only chunk
    else partial[(int64_t)blockIdx.y * cols + at] = s;
  }
}

// db[c] = sum of the chunks' sums in chunk order, rounded once.
template <class T>
__global__ void join_columns_kernel(const float* __restrict__ partial, int chunks, int cols, T* __restrict__ db) {
  half::allow_next_if_few();
  half::wait_previous();
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  float s = 0.0f;
#pragma unroll 8
  for (int i = 0; i < chunks; ++i) s += partial[(int64_t)i * cols + c];
  db[c] = from_float<T>(s);
}

// Second order: t = h + hb; dgy = t f'(z), dz = t gy f''(z). Value by value: 8280 x
// 3072 in 136 us, 1.9 TB/s, bound by its two-byte accesses and their indices.
template <class T>
__global__ void act_grad2_kernel(const T* __restrict__ h, const T* __restrict__ hb, const T* __restrict__ gy,
                                 const T* __restrict__ z, T* __restrict__ dgy, T* __restrict__ dz, int64_t rows,
                                 int cols, int kind) {
  const int64_t n = rows * cols, stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += stride) {
    const float t = (h ? to_float(h[i]) : 0.0f) + (hb ? to_float(hb[i % cols]) : 0.0f);
    const float x = hold_nan(to_float(z[i]), kFar);
    dgy[i] = from_float<T>(t * act_grad(x, kind));
    dz[i] = from_float<T>(t * to_float(gy[i]) * act_grad2(x, kind));
  }
}

// Rows of one or two matrices onto 16-byte boundaries: a thread writes 8 values.
struct Padded {
  const uint16_t* src;
  uint16_t* dst;
  int64_t ld_src, ld_dst, rows;
  int cols;
};
__global__ void __launch_bounds__(256) pad_rows_kernel(Padded a, Padded b) {
  half::allow_next_if_few();
  half::wait_previous();
  const int64_t first = (a.ld_dst / 8) * a.rows, all = first + (b.ld_dst / 8) * b.rows;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < all; i += stride) {
    const Padded& p = i < first ? a : b;
    const int64_t at = i < first ? i : i - first, per = p.ld_dst / 8, row = at / per;
    const int col = (int)(at - row * per) * 8;
    const uint16_t* src = p.src + row * p.ld_src + col;
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = col + 2 * e < p.cols ? src[2 * e] : 0, y = col + 2 * e + 1 < p.cols ? src[2 * e + 1] : 0;
      v[e] = x | y << 16;
    }
    *reinterpret_cast<uint4*>(p.dst + row * p.ld_dst + col) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// ---- host side ---------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool known_act(int act) {
  return act == CG_ACT_NONE || act == CG_ACT_SILU || act == CG_ACT_RELU || act == CG_ACT_GELU;
}

struct Plan {
  int cg, bn;
  int splits[2], kt_per[2];
};

// Tile of a launch and k-splits of its one or two products, by the time of the
// slot (SM or SM pair) that gets most: a tile takes `slice` per 64-wide k-slice
// and `wave` beside it, in nanoseconds measured on launches of one wave and of
// several, and a launch `once`. 256 x 256 tiles of an SM pair feed the tensor
// cores best (4096^3: 97 us, 108 us with 256 x 128, 125 with 128 x 128, 223 with
// 128 x 64), the smaller ones fill the SMs when there are few (512^3: 7.7, 6.0,
// 5.8 and 5.1 us); a split pays when k is long (3072 x 768 x 8280: 40 us in two
// parts, 55 us whole).
static Plan search_plan(const cg_linear_args* g, int count) {
  const int64_t sms = sm_count();
  struct Shape {
    int cg, bn;
    double slice, wave, once;
  };
  static const Shape shapes[] = {
      {2, 256, 320, 1450, 4200}, {2, 192, 278, 950, 4000}, {2, 128, 215, 810, 4000}, {1, 128, 205, 1400, 2900}, {1, 64, 195, 900, 2700}};
  const int kMost = 24;
  int64_t kts[2] = {1, 1};
  for (int i = 0; i < count; ++i) kts[i] = ceil_div<int64_t>(g[i].k, half::kBK);
  Plan best = {};
  double least = 0.0;
  for (const Shape& s : shapes) {
    const int64_t slots = sms / s.cg;
    int64_t tiles[2] = {0, 0};
    int most[2] = {1, 1};
    for (int i = 0; i < count; ++i) {
      tiles[i] = ceil_div<int64_t>(g[i].m, s.cg * half::kRows) * ceil_div<int64_t>(g[i].n, s.bn);
      // more parts than fill the slots twice only add to the join
      int64_t n = 2 * slots / tiles[i];
      if (n > kts[i] / 4) n = kts[i] / 4;
      most[i] = n < 1 ? 1 : n > kMost ? kMost : (int)n;
    }
    for (int s0 = 1; s0 <= most[0]; ++s0)
      for (int s1 = 1; s1 <= most[1]; ++s1) {
        const int split[2] = {s0, s1};
        int64_t per[2] = {1, 1}, items[2] = {0, 0};
        double time[2] = {0.0, 0.0}, join = 0.0;
        bool same = true;
        for (int i = 0; i < count; ++i) {
          per[i] = ceil_div<int64_t>(kts[i], split[i]);
          same = same && ceil_div<int64_t>(kts[i], per[i]) == split[i];
          items[i] = tiles[i] * split[i];
          time[i] = (double)per[i] * s.slice + s.wave;
          // the join's launch on both sides, the partial tiles written and read at about 4 TB/s
          if (split[i] > 1) join += 4500.0 + (double)split[i] * g[i].m * g[i].n * 8.0 / 4000.0;
        }
        if (!same) continue;
        // slot k gets items k, k + slots, ..: at most three different loads
        const int64_t total = items[0] + items[1], edges[3] = {0, items[0] % slots, total % slots};
        double cost = 0.0;
        for (int64_t k : edges) {
          const int64_t first = items[0] / slots + (k < items[0] % slots), all = total / slots + (k < total % slots);
          const double load = (double)first * time[0] + (double)(all - first) * time[1];
          if (load > cost) cost = load;
        }
        cost += join + s.once;
        if (least == 0.0 || cost < least) {
          least = cost;
          best.cg = s.cg;
          best.bn = s.bn;
          for (int i = 0; i < 2; ++i) {
            best.splits[i] = split[i];
            best.kt_per[i] = (int)per[i];
          }
        }
      }
  }
  return best;
}

// The search takes tens of microseconds for two products that may both split, so
// each host thread keeps the plans of the last sizes it met.
static Plan plan_of(const cg_linear_args* g, int count) {
  struct Entry {
    int64_t key[7];
    Plan plan;
  };
  constexpr int kEntries = 256;
  static thread_local Entry table[kEntries];
  const int64_t key[7] = {g[0].m, g[0].n, g[0].k, count > 1 ? g[1].m : 0, count > 1 ? g[1].n : 0,
                          count > 1 ? g[1].k : 0, sm_count()};
  uint64_t h = 1469598103934665603ull;
  for (int64_t v : key) h = (h ^ (uint64_t)v) * 1099511628211ull;
  Entry& e = table[(h >> 32) % kEntries];
  if (memcmp(e.key, key, sizeof(key)) != 0) {
    e.plan = search_plan(g, count);
    memcpy(e.key, key, sizeof(key));
  }
  return e.plan;
}

static int64_t partial_bytes(const cg_linear_args& g, int splits) {
  return splits > 1 ? ceil_div<int64_t>((int64_t)splits * g.m * g.n * (int64_t)sizeof(float), 256) * 256 : 0;
}

// Partial tiles of a launch's products, one after the other.
static int64_t workspace_bytes(const cg_linear_args* g, int count) {
  const Plan p = plan_of(g, count);
  int64_t n = 0;
  for (int i = 0; i < count; ++i) n += partial_bytes(g[i], p.splits[i]);
  return n;
}

// 16-byte groups of eight columns everywhere.
static bool aligned_problem(const cg_linear_args& g) {
  return g.n % 8 == 0 && g.ld_y % 8 == 0 && aligned16(g.y) && (g.bias == nullptr || aligned16(g.bias)) &&
         (g.residual == nullptr || (aligned16(g.residual) && g.ld_residual % 8 == 0)) &&
         (g.z == nullptr || (aligned16(g.z) && g.ld_z % 8 == 0));
}

template <int CG, int BN, class E>
static int launch(const cg_linear_args* g, int count, const Plan& p, const EpiArgs* ea, bool bf16, cudaStream_t s) {
  half::LaunchOf<E> L;
  memset(&L, 0, sizeof(L));
  L.groups = count;
  L.bf16 = bf16;
  int64_t items = 0;
  for (int i = 0; i < count; ++i) {
    const cg_linear_args& q = g[i];
    auto& G = L.g[i];
    int rc;
    if ((rc = half::make_half_map(&G.map_a, q.a, bf16, q.a_mn_major ? q.k : q.m, q.a_mn_major ? q.m : q.k, q.lda, 1,
                                  q.lda * (q.a_mn_major ? q.k : q.m), q.a_mn_major != 0, half::kRows)))
      return rc;
    if ((rc = half::make_half_map(&G.map_b, q.b, bf16, q.b_mn_major ? q.k : q.n, q.b_mn_major ? q.n : q.k, q.ldb, 1,
                                  q.ldb * (q.b_mn_major ? q.k : q.n), q.b_mn_major != 0, BN / CG)))
      return rc;
    G.m = (int)q.m;
    G.n = (int)q.n;
    G.k = (int)q.k;
    G.batch = 1;
    G.a_mn = q.a_mn_major;
    G.b_mn = q.b_mn_major;
    G.splits = p.splits[i];
    G.kt_per = p.kt_per[i];
    G.epi = ea[i];
    G.first_item = (int)items;
    items += half::plan_group<CG, BN>(G);
    CG_REQUIRE(items < (1ll << 31), "linear_half: too many tiles");
  }
  L.items = (int)items;
  return half::launch_half_gemm<CG, BN, 1, E>(L, s);
}

template <class E>
static int launch_plan(const cg_linear_args* g, int count, const Plan& p, const EpiArgs* ea, bool bf16,
                       cudaStream_t s) {
  if (p.cg == 2 && p.bn == 256) return launch<2, 256, E>(g, count, p, ea, bf16, s);
  if (p.cg == 2 && p.bn == 192) return launch<2, 192, E>(g, count, p, ea, bf16, s);
  if (p.cg == 2) return launch<2, 128, E>(g, count, p, ea, bf16, s);
  if (p.bn == 128) return launch<1, 128, E>(g, count, p, ea, bf16, s);
  return launch<1, 64, E>(g, count, p, ea, bf16, s);
}

// One or two products (all checked) in one launch, and the joins of those that
// split k.
template <class T>
static int run_typed(const cg_linear_args* g, int count, void* workspace, int64_t bytes, bool bf16, cudaStream_t s) {
  int rc;
  if ((rc = half::bind_context())) return rc;
  const Plan p = plan_of(g, count);
  EpiArgs ea[2];
  memset(ea, 0, sizeof(ea));
  bool vec = true;
  int64_t used = 0;
  for (int i = 0; i < count; ++i) {
    const cg_linear_args& q = g[i];
    ea[i].y = q.y;
    ea[i].ld_y = q.ld_y;
    ea[i].bias = q.bias;
    ea[i].residual = q.residual;
    ea[i].ld_res = q.ld_residual;
    ea[i].z = q.z;
    ea[i].ld_z = q.ld_z;
    ea[i].act = q.act;
    vec = vec && aligned_problem(q);
    if (p.splits[i] > 1) ea[i].partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + used);
    used += partial_bytes(q, p.splits[i]);
  }
  CG_REQUIRE(used == 0 || (workspace != nullptr && aligned16(workspace) && bytes >= used),
             "linear_half: this shape splits K and needs %lld workspace bytes on a 16-byte boundary "
             "(cg_linear_half_workspace_bytes)",
             (long long)used);
  if (vec) {
    const auto type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    for (int i = 0; i < count; ++i) {
      const cg_linear_args& q = g[i];
      auto block_map = [&](CUtensorMap* map, const void* ptr, int64_t ld) {
        return ptr ? half::make_block_map(map, type, 2, 128, ptr, q.m, q.n, ld, 1, q.m * ld) : kOk;
      };
      if (ea[i].partial)
        rc = half::make_block_map(&ea[i].map_partial, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, 128, ea[i].partial, q.m, q.n,
                                  q.n, p.splits[i], q.m * q.n);
      else if ((rc = block_map(&ea[i].map_y, q.y, q.ld_y)) == kOk && (rc = block_map(&ea[i].map_z, q.z, q.ld_z)) == kOk)
        rc = block_map(&ea[i].map_res, q.residual, q.ld_residual);
      if (rc) return rc;
    }
    rc = launch_plan<BlockEpi<T>>(g, count, p, ea, bf16, s);
  } else {
    rc = launch_plan<PlainEpi<T>>(g, count, p, ea, bf16, s);
  }
  if (rc) return rc;
  for (int i = 0; i < count; ++i) {
    if (p.splits[i] == 1) continue;
    const int64_t blocks = ceil_div<int64_t>(ceil_div<int64_t>(g[i].m * g[i].n, vec ? 8 : 1), 256);
    const int64_t most = (int64_t)sm_count() * 8;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    auto kernel = vec ? join_splits_kernel<T, true> : join_splits_kernel<T, false>;
    if ((rc = half::launch_chained("linear_half split join", kernel, dim3(grid), 256, 0, dim3(1, 1), s, ea[i],
                                   p.splits[i], (int)g[i].m, (int)g[i].n)))
      return rc;
  }
  return kOk;
}

static int checked(const cg_linear_args& g) {
  CG_REQUIRE(g.dtype == CG_F16 || g.dtype == CG_BF16, "linear_half: dtype %d is neither CG_F16 nor CG_BF16", g.dtype);
  CG_REQUIRE(known_act(g.act), "linear_half: bad act %d", g.act);
  CG_REQUIRE(g.m >= 1 && g.n >= 1 && g.k >= 1, "linear_half: sizes must be at least 1");
  const int64_t most = (1ll << 31) - 512;  // tile coordinates are 32-bit
  CG_REQUIRE(g.m < most && g.n < most && g.k < most, "linear_half: size too large");
  CG_REQUIRE(g.a && g.b && g.y, "linear_half: a, b and y must be non-null");
  CG_REQUIRE(aligned16(g.a) && aligned16(g.b), "linear_half: a and b must be 16-byte aligned");
  CG_REQUIRE(g.lda % 8 == 0 && g.ldb % 8 == 0, "linear_half: lda and ldb must be multiples of 8 values");
  CG_REQUIRE(g.lda >= (g.a_mn_major ? g.m : g.k) && g.ldb >= (g.b_mn_major ? g.n : g.k) && g.ld_y >= g.n &&
                 (g.residual == nullptr || g.ld_residual >= g.n) && (g.z == nullptr || g.ld_z >= g.n),
             "linear_half: row pitch smaller than the row");
  return kOk;
}

static int run_products(const cg_linear_args* g, int count, void* workspace, int64_t bytes, void* stream) {
  for (int i = 0; i < count; ++i)
    if (int rc = checked(g[i])) return rc;
  if (g->dtype == CG_F16) return run_typed<__half>(g, count, workspace, bytes, false, as_stream(stream));
  return run_typed<__nv_bfloat16>(g, count, workspace, bytes, true, as_stream(stream));
}

static int run(const cg_linear_args* args, void* stream) {
  CG_REQUIRE(args != nullptr, "linear_half: args is NULL");
  if (args->m == 0 || args->n == 0) return kOk;
  return run_products(args, 1, args->workspace, args->workspace_bytes, stream);
}

// Row chunks of act_grad, each of at least 32 rows: as many blocks as the SMs
// hold at once (V = 8: four an SM), for single columns enough to fill them
// several times; up to 128 rows are one chunk, whose sums need no join.
static int chunk_rows(int64_t rows, int64_t cols, int v) {
  if (rows <= 128) return 128;
  const int64_t strips = ceil_div<int64_t>(cols, 32 * v);
  int64_t chunks = v == 8 ? (int64_t)sm_count() * 4 / strips : ceil_div<int64_t>((int64_t)sm_count() * 8, strips);
  if (chunks < 1) chunks = 1;
  int64_t per = ceil_div<int64_t>(rows, chunks);
  per = ceil_div<int64_t>(per < 32 ? 32 : per, 8) * 8;
  const int64_t least = ceil_div<int64_t>(rows, 65535);  // gridDim.y
  return (int)(per < least ? least : per);
}

template <class T>
static int act_grad_typed(const cg_act_grad_args& g, cudaStream_t s) {
  const bool vec = g.cols % 8 == 0;
  const bool aligned = aligned16(g.gy) && g.ld_gy % 8 == 0 &&
                       (g.gz == nullptr || (aligned16(g.z) && aligned16(g.gz) && g.ld_z % 8 == 0 && g.ld_gz % 8 == 0));
  const int per = chunk_rows(g.rows, g.cols, vec ? 8 : 1);
  const int chunks = (int)ceil_div<int64_t>(g.rows, per);
  const dim3 grid((unsigned)ceil_div<int64_t>(g.cols, vec ? 256 : 32), (unsigned)chunks);
  const bool direct = chunks == 1;
  float* partial = g.db && !direct ? g.scratch : nullptr;
  T* db = g.db && direct ? (T*)g.db : nullptr;
  auto kernel = !vec ? act_grad_kernel<T, 1, false>
                : aligned ? act_grad_kernel<T, 8, true> : act_grad_kernel<T, 8, false>;
  if (int rc = half::launch_chained("act_grad_half", kernel, grid, 256, 0, dim3(1, 1), s, (const T*)g.gy, g.ld_gy,
                                    (const T*)g.z, g.ld_z, (T*)g.gz, g.ld_gz, (int)g.rows, (int)g.cols, g.act, per,
                                    partial, db))
    return rc;
  if (partial == nullptr) return kOk;
  return half::launch_chained("act_grad_half column join", join_columns_kernel<T>,
                              dim3((unsigned)ceil_div<int64_t>(g.cols, 128)), 128, 0, dim3(1, 1), s,
                              (const float*)partial, chunks, (int)g.cols, (T*)g.db);
}

static int64_t act_grad_scratch(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  int64_t most = 0;
  for (int v : {1, 8}) {
    const int64_t chunks = ceil_div<int64_t>(rows, chunk_rows(rows, cols, v));
    if (chunks > most) most = chunks;
  }
  return most * cols * (int64_t)sizeof(float);
}

static int act_grad_run(const cg_act_grad_args* args, void* stream) {
  CG_REQUIRE(args != nullptr, "act_grad_half: args is NULL");
  const cg_act_grad_args& g = *args;
  CG_REQUIRE(g.dtype == CG_F16 || g.dtype == CG_BF16, "act_grad_half: dtype %d is neither CG_F16 nor CG_BF16",
             g.dtype);
  CG_REQUIRE(known_act(g.act), "act_grad_half: bad act %d", g.act);
  CG_REQUIRE(g.rows >= 0 && g.cols >= 0 && g.rows < (1ll << 31) - 512 && g.cols < (1ll << 31) - 512,
             "act_grad_half: bad size");
  if (g.rows == 0 || g.cols == 0) {
    // a sum over no rows
    if (g.db && g.cols > 0) CG_CUDA(cudaMemsetAsync(g.db, 0, (size_t)g.cols * 2, as_stream(stream)));
    return kOk;
  }
  CG_REQUIRE(g.gy != nullptr && (g.gz == nullptr || g.z != nullptr), "act_grad_half: null input");
  CG_REQUIRE(g.gz != nullptr || g.db != nullptr, "act_grad_half: no output asked for");
  CG_REQUIRE(g.ld_gy >= g.cols && (g.gz == nullptr || (g.ld_z >= g.cols && g.ld_gz >= g.cols)),
             "act_grad_half: row pitch smaller than the row");
  CG_REQUIRE(g.db == nullptr || (g.scratch != nullptr && g.scratch_bytes >= act_grad_scratch(g.rows, g.cols)),
             "act_grad_half: the column sums need %lld scratch bytes (cg_act_grad_half_scratch_bytes)",
             (long long)act_grad_scratch(g.rows, g.cols));
  if (g.dtype == CG_F16) return act_grad_typed<__half>(g, as_stream(stream));
  return act_grad_typed<__nv_bfloat16>(g, as_stream(stream));
}

// The products of a backward: dx = gz W (W read along n) and dW = gz^T x.
static cg_linear_args dx_product(const cg_linear_backward_args& g) {
  cg_linear_args p;
  memset(&p, 0, sizeof(p));
  p.m = g.m;
  p.n = g.k;
  p.k = g.n;
  p.a = g.act == CG_ACT_NONE ? g.gy : g.gz;
  p.lda = g.act == CG_ACT_NONE ? g.ld_gy : g.ld_gz;
  p.b = g.w;
  p.ldb = g.ld_w;
  p.b_mn_major = !g.w_mn_major;
  p.y = g.dx;
  p.ld_y = g.k;
  p.dtype = g.dtype;
  return p;
}
static cg_linear_args dw_product(const cg_linear_backward_args& g) {
  cg_linear_args p = dx_product(g);
  p.m = g.n;
  p.k = g.m;
  p.a_mn_major = 1;
  p.b = g.x;
  p.ldb = g.ld_x;
  p.b_mn_major = !g.x_mn_major;
  p.y = g.dw;
  return p;
}

static int products(const cg_linear_backward_args& g, cg_linear_args* p) {
  int n = 0;
  if (g.dx) p[n++] = dx_product(g);
  if (g.dw) p[n++] = dw_product(g);
  return n;
}

// One region serves the column sums and then the products.
static int64_t backward_workspace(const cg_linear_backward_args& g) {
  if (g.m <= 0 || g.n <= 0 || g.k <= 0) return 0;
  int64_t most = g.db ? act_grad_scratch(g.m, g.n) : 0;
  cg_linear_args p[2];
  const int count = products(g, p);
  const int64_t n = count ? workspace_bytes(p, count) : 0;
  return n > most ? n : most;
}

static int backward_run(const cg_linear_backward_args* args, void* stream) {
  CG_REQUIRE(args != nullptr, "linear_half_backward: args is NULL");
  const cg_linear_backward_args& g = *args;
  CG_REQUIRE(known_act(g.act), "linear_half_backward: bad act %d", g.act);
  CG_REQUIRE(g.m >= 1 && g.n >= 1 && g.k >= 1, "linear_half_backward: sizes must be at least 1");
  CG_REQUIRE(g.workspace_bytes >= backward_workspace(g) &&
                 (backward_workspace(g) == 0 || (g.workspace != nullptr && aligned16(g.workspace))),
             "linear_half_backward: needs %lld workspace bytes on a 16-byte boundary "
             "(cg_linear_half_backward_workspace_bytes)",
             (long long)backward_workspace(g));
  int rc;
  const bool plain = g.act == CG_ACT_NONE;
  if (!plain || g.db) {
    cg_act_grad_args a;
    memset(&a, 0, sizeof(a));
    a.rows = g.m;
    a.cols = g.n;
    a.gy = g.gy;
    a.ld_gy = g.ld_gy;
    a.act = g.act;
    a.dtype = g.dtype;
    if (!plain) {
      CG_REQUIRE(g.z != nullptr && g.gz != nullptr, "linear_half_backward: an activation needs z and gz");
      a.z = g.z;
      a.ld_z = g.ld_z;
      a.gz = g.gz;
      a.ld_gz = g.ld_gz;
    }
    a.db = g.db;
    a.scratch = static_cast<float*>(g.workspace);
    a.scratch_bytes = g.workspace_bytes;
    if ((rc = act_grad_run(&a, stream))) return rc;
  }
  cg_linear_args p[2];
  const int count = products(g, p);
  return count ? run_products(p, count, g.workspace, g.workspace_bytes, stream) : kOk;
}

template <class T>
static int act_grad2_typed(const void* h, const void* hb, const void* gy, const void* z, void* dgy, void* dz,
                           int64_t rows, int64_t cols, int act, cudaStream_t s) {
  const int64_t blocks = ceil_div<int64_t>(rows * cols, 256), most = (int64_t)sm_count() * 16;
  act_grad2_kernel<T><<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>(
      (const T*)h, (const T*)hb, (const T*)gy, (const T*)z, (T*)dgy, (T*)dz, rows, (int)cols, act);
  CG_LAUNCHED("act_grad2_half");
  return kOk;
}

int device_error(int* out, bool reset) {
  CG_CUDA(cudaMemcpyFromSymbol(out, g_dense_error, sizeof(int)));
  const int zero = 0;
  if (reset) CG_CUDA(cudaMemcpyToSymbol(g_dense_error, &zero, sizeof(int)));
  return kOk;
}

}  // namespace dense
}  // namespace cg

extern "C" {

int cg_linear_half(const cg_linear_args* args, void* stream) { return cg::dense::run(args, stream); }

int64_t cg_linear_half_workspace_bytes(const cg_linear_args* args) {
  if (args == nullptr || args->m <= 0 || args->n <= 0 || args->k <= 0) return 0;
  return cg::dense::workspace_bytes(args, 1);
}

int cg_pad_rows_half(const void* src, int64_t ld_src, int64_t rows, int64_t cols, void* dst, int64_t ld_dst,
                     const void* src2, int64_t ld_src2, int64_t rows2, int64_t cols2, void* dst2, int64_t ld_dst2,
                     void* stream) {
  using namespace cg;
  auto padded = [](const void* from, int64_t ld_from, int64_t r, int64_t c, void* to, int64_t ld_to) {
    return dense::Padded{static_cast<const uint16_t*>(from), static_cast<uint16_t*>(to), ld_from, ld_to, r, (int)c};
  };
  auto fine = [](const void* from, int64_t ld_from, int64_t r, int64_t c, const void* to, int64_t ld_to) {
    return r >= 0 && c >= 0 && c < (1ll << 31) &&
           (r == 0 || (from != nullptr && to != nullptr && dense::aligned16(to) && ld_to % 8 == 0 && ld_from >= c &&
                       ld_to >= c));
  };
  CG_REQUIRE(fine(src, ld_src, rows, cols, dst, ld_dst) && fine(src2, ld_src2, rows2, cols2, dst2, ld_dst2),
             "pad_rows_half: bad size, pitch or alignment");
  const int64_t work = ld_dst / 8 * rows + (rows2 > 0 ? ld_dst2 / 8 * rows2 : 0);
  if (work == 0) return kOk;
  const int64_t blocks = ceil_div<int64_t>(work, 256), most = (int64_t)sm_count() * 8;
  return cg::half::launch_chained("pad_rows_half", dense::pad_rows_kernel, dim3((unsigned)(blocks < most ? blocks : most)),
                              256, 0, dim3(1, 1), as_stream(stream), padded(src, ld_src, rows, cols, dst, ld_dst),
                              rows2 > 0 ? padded(src2, ld_src2, rows2, cols2, dst2, ld_dst2)
                                        : dense::Padded{nullptr, nullptr, 0, 8, 0, 0});
}

int cg_linear_half_backward(const cg_linear_backward_args* args, void* stream) {
  return cg::dense::backward_run(args, stream);
}

int64_t cg_linear_half_backward_workspace_bytes(const cg_linear_backward_args* args) {
  return args == nullptr ? 0 : cg::dense::backward_workspace(*args);
}

int cg_act_grad_half(const cg_act_grad_args* args, void* stream) { return cg::dense::act_grad_run(args, stream); }

int64_t cg_act_grad_half_scratch_bytes(int64_t rows, int64_t cols) { return cg::dense::act_grad_scratch(rows, cols); }

int cg_act_grad2_half(const void* h, const void* hb, const void* gy, const void* z, void* dgy, void* dz, int64_t rows,
                      int64_t cols, int act, int dtype, void* stream) {
  using namespace cg;
  CG_REQUIRE(dtype == CG_F16 || dtype == CG_BF16, "act_grad2_half: dtype %d is neither CG_F16 nor CG_BF16", dtype);
  CG_REQUIRE(dense::known_act(act), "act_grad2_half: bad act %d", act);
  CG_REQUIRE(rows >= 0 && cols >= 0 && cols < (1ll << 31), "act_grad2_half: bad size");
  if (rows == 0 || cols == 0) return kOk;
  CG_REQUIRE((h || hb) && gy && z && dgy && dz, "act_grad2_half: null buffer");
  if (dtype == CG_F16)
    return dense::act_grad2_typed<__half>(h, hb, gy, z, dgy, dz, rows, cols, act, as_stream(stream));
  return dense::act_grad2_typed<__nv_bfloat16>(h, hb, gy, z, dgy, dz, rows, cols, act, as_stream(stream));
}

}  // extern "C"
