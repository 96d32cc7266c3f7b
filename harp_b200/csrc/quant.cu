// Rows in 8 bits: the quantisers that feed the int8 GEMM (gemm_s8_sm100.cu).
//
//   quant_rows          y = x
//   swiglu_quant        y = silu(g) * u of a row [g | u]
//   rmsnorm_mod_quant   h = residual + gate[b] * x (h = x without a residual),
//                       y = h * rsqrt(mean(h^2) + eps) * w * (1 + scale[b]) + shift[b]
//   then for each row   s = max(max|y| / 127, 2^-126),  q = y / s rounded half to even
//   dequant_rows        q * s, the inverse
//
// All of it is 32-bit arithmetic on registers; the only roundings to fewer bits
// are q itself and the stored h (in x's type, as the residual stream is kept).
// The norm and y use h before that rounding.  1 / 127 and 1 / s are rounded once
// and multiplied, so an error of about 2^-23 in y / s can move a value that lies
// that close to a rounding boundary, nothing else.  The floor of s keeps 1 / s
// finite, so a row of zeros (or of values below 2^-127) gives q = 0.  A row that
// holds a NaN or an infinity has s = NaN and q = 0: what is computed from it is
// NaN, as it is in bf16.
//
// Bound by memory: each value is read once and held in registers between the
// row's reductions and the rounding.  Measured on one B200, bf16, on three sets of inputs
// in turn, of which L2 (126 MB) still holds a part, and in brackets after 512 MB were
// written: quant_rows of 17408 x 1152 9.8 us (16.4), swiglu_quant of 17408 x 4608 66.7 us
// (71.7), rmsnorm_mod_quant of 17408 x 1152 with residual, gate and modulation 20.3 us
// (31.7), dequant_rows of 17408 x 1152 10.9 us (16.4); a copy of the same bytes at 6.5 TB/s
// takes 9.2, 61.3, 21.5 and 9.2.  One to a few hundred rows take 1.3 to 2.1 us back to back.
// Widths that are not multiples of 8 read 2 or 1 values at a time: 17408 x 1154 21.4 us
// (28.7), 17408 x 1155 31.2 us (38.9), bound by instructions.
#include "common.cuh"
#include "dependent_launch.cuh"
#include "gemm_sm100.h"
#include "per_device.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

namespace harp {

namespace {

using bf16 = __nv_bfloat16;

constexpr float kMinScale = 1.17549435e-38f;  // 2^-126
constexpr int kMaxWarps = 16;
constexpr size_t kVecSmem = 96 * 1024;  // of a sample's vectors in norm_sample_kernel

enum QuantMode : int { kRows = 0, kSwiglu = 1, kNorm = 2, kNormRes = 3 };

struct QuantArgs {
  const void* x;
  long ldx;
  const void* res;
  long ldr;
  void* h;
  long ldh;
  const void* w;
  const void* gate;
  const void* scale;
  const void* shift;
  long ld_gate, ld_scale, ld_shift;
  int8_t* q;
  long ldq;
  float* s;
  long R;
  int D;
  long rows_per_batch;
  float eps;
  int device;  // that of every tensor here
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f(float v, bf16* p) { *p = __float2bfloat16(v); }

// V consecutive values (1, 2 or 8) as they are stored, aligned to their size or to
// 16 bytes, and as fp32.
template <int BYTES>
struct Words {
  uint4 v[BYTES / 16];
};
template <>
struct Words<2> { uint16_t v[1]; };
template <>
struct Words<4> { uint32_t v[1]; };
template <>
struct Words<8> { uint2 v[1]; };
template <int V, typename T>
using Raw = Words<V * (int)sizeof(T)>;

template <int V, typename T>
__device__ __forceinline__ Raw<V, T> load_raw(const T* p) {
  Raw<V, T> r;
  using E = std::remove_reference_t<decltype(r.v[0])>;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r.v) / sizeof(E)); ++i) r.v[i] = reinterpret_cast<const E*>(p)[i];
  return r;
}
// (volatile: a load in assembly stays behind dependency_wait() only so)
__device__ __forceinline__ uint16_t ld_first(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.cs.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_first(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.cs.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_first(const uint2* p) {
  uint2 v;
  asm volatile("ld.global.cs.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_first(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
// Values of a row, which nothing reads again: first to leave the caches, so that
// they do not push out what is being written (norm of 17408 x 1152 with a residual:
// 25.9 us, 30.6 without, when this was added).
template <int V, typename T>
__device__ __forceinline__ Raw<V, T> load_once(const T* p) {
  Raw<V, T> r;
  using E = std::remove_reference_t<decltype(r.v[0])>;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r.v) / sizeof(E)); ++i) r.v[i] = ld_first(reinterpret_cast<const E*>(p) + i);
  return r;
}
template <int V, typename T>
__device__ __forceinline__ Raw<V, T> zero_raw() {
  Raw<V, T> r;
  memset(&r, 0, sizeof(r));
  return r;
}
template <int V, typename T>
__device__ __forceinline__ void to_f32(const Raw<V, T>& r, float* f) {
  if constexpr (sizeof(T) == 2 && V == 1) {
    f[0] = __uint_as_float((uint32_t)r.v[0] << 16);
  } else {
    uint32_t u[sizeof(r) / 4];
    memcpy(u, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r) / 4); ++i) {
      if constexpr (sizeof(T) == 2) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      } else {
        f[i] = __uint_as_float(u[i]);
      }
    }
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_v(T* p, const float* f) {
  if constexpr (V == 1) {
    from_f(f[0], p);
  } else if constexpr (V == 2) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(f[0], f[1]);
    else *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// Pairs: one instruction for two fp32 operations (sm_100), which is what keeps
// these kernels bound by memory and not by instruction issue.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// max(|a|, |b|, m), keeping a NaN.
__device__ __forceinline__ float amax2(float a, float b, float m) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(m));
  return r;
}
template <int L>
__device__ __forceinline__ float amax_all(const float (&y)[L]) {
  float m = 0.f, m2 = 0.f;
#pragma unroll
  for (int i = 0; i + 3 < L; i += 4) {
    m = amax2(y[i], y[i + 1], m);
    m2 = amax2(y[i + 2], y[i + 3], m2);
  }
#pragma unroll
  for (int i = L / 4 * 4; i < L; ++i) m = amax2(y[i], 0.f, m);
  return amax2(m, m2, 0.f);
}
template <int L>
__device__ __forceinline__ float square_sum(const float (&y)[L]) {
  uint64_t s = pair(0.f, 0.f), s2 = s;
#pragma unroll
  for (int i = 0; i + 3 < L; i += 4) {
    const uint64_t u = pair(y[i], y[i + 1]), v = pair(y[i + 2], y[i + 3]);
    s = fma2(u, u, s);
    s2 = fma2(v, v, s2);
  }
  float a, b;
  unpair(add2(s, s2), a, b);
  a += b;
#pragma unroll
  for (int i = L / 4 * 4; i < L; ++i) a = fmaf(y[i], y[i], a);
  return a;
}

__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// The row's scale and its reciprocal (0 for a row with NaN or infinity).
__device__ __forceinline__ void row_scale(float amax, float& s, float& inv) {
  s = fmaxf(__fmul_rn(amax, 1.0f / 127.0f), kMinScale);
  inv = __frcp_rn(s);
  if (!(amax < INFINITY)) {
    s = __uint_as_float(0x7FFFFFFFu);
    inv = 0.f;
  }
}
// y / s to the nearest integer, ties to even, as the low byte of the sum: |y * inv| < 127.5
// by the scale's construction.
constexpr float kRound = 12582912.f;  // 1.5 * 2^23
template <int V>
__device__ __forceinline__ void store_q(int8_t* p, const float* y, float inv) {
  if constexpr (V == 1) {
    *p = inv != 0.f ? (int8_t)(__float_as_uint(__fadd_rn(__fmul_rn(y[0], inv), kRound)) & 0xFFu) : (int8_t)0;
  } else if constexpr (V == 2) {
    const uint32_t b0 = __float_as_uint(__fadd_rn(__fmul_rn(y[0], inv), kRound));
    const uint32_t b1 = __float_as_uint(__fadd_rn(__fmul_rn(y[1], inv), kRound));
    *reinterpret_cast<uint16_t*>(p) = inv != 0.f ? (uint16_t)__byte_perm(b0, b1, 0x0040) : (uint16_t)0;
  } else {
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float lo, hi;
      // (as two scalar products: ptxas joins the packed product and sum into one rounding)
      unpair(add2(pair(__fmul_rn(y[2 * j], inv), __fmul_rn(y[2 * j + 1], inv)), pair(kRound, kRound)), lo, hi);
      b[2 * j] = __float_as_uint(lo);
      b[2 * j + 1] = __float_as_uint(hi);
    }
    uint2 o;
    o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    *reinterpret_cast<uint2*>(p) = inv != 0.f ? o : make_uint2(0u, 0u);
  }
}

// Sum, or NaN-keeping maximum, over the lanes of a row (8, 16 or 32 of a warp).
// Non-negative floats and NaN order as their bits do.
template <bool MAX>
__device__ __forceinline__ float lane_reduce(float v, int lanes) {
  if (MAX && lanes == 32) return __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v)));
  for (int o = lanes / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if constexpr (MAX) v = __uint_as_float(max(__float_as_uint(v), __float_as_uint(u)));
    else v += u;
  }
  return v;
}
// The same over a row that is `warps` warps (the block, if more than one).
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, int lanes, int warps, float* smem) {
  v = lane_reduce<MAX>(v, lanes);
  if (warps == 1) return v;
  if (threadIdx.x % 32 == 0) smem[threadIdx.x / 32] = v;
  __syncthreads();
  v = threadIdx.x % 32 < warps ? smem[threadIdx.x % 32] : 0.f;
  return lane_reduce<MAX>(v, 32);
}

// A row's values in registers: its `per_row` threads (8, 16 or 32 lanes of a warp,
// or the block) hold N groups of V values each, group k of thread t at column
// (k * per_row + t) * V.  V = 8 needs D % 8 == 0 and 16-byte aligned rows, V = 2 an even
// D and rows aligned to two values.  All of a
// thread's loads are issued before the first is used.
template <int MODE, typename T, int V, int N>
__global__ void __launch_bounds__(32 * kMaxWarps) quant_rows_kernel(const QuantArgs a, int lanes, int warps) {
  constexpr bool NORM = MODE >= kNorm, TWO = MODE == kSwiglu || MODE == kNormRes;
  __shared__ float red[2][32];
  dependency_wait();
  const int per_row = lanes * warps;
  const int t = warps == 1 ? threadIdx.x % lanes : threadIdx.x;
  const long at = warps == 1 ? (long)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes : (long)blockIdx.x;
  // groups past the end go along with the last row (shuffles need the whole warp) and store nothing
  const long row = min(at, a.R - 1);
  const bool live = at < a.R;
  using R_ = Raw<V, T>;
  R_ x[N], x2[TWO ? N : 1];
  {
    const T* px = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const T* p2 = MODE == kSwiglu ? px + a.D : reinterpret_cast<const T*>(a.res) + row * a.ldr;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = (k * per_row + t) * V;
      x[k] = e < a.D ? load_once<V, T>(px + e) : zero_raw<V, T>();
      if constexpr (TWO) x2[k] = e < a.D ? load_once<V, T>(p2 + e) : zero_raw<V, T>();
    }
  }
  R_ vw[NORM ? N : 1], vscale[NORM ? N : 1], vshift[NORM ? N : 1], vgate[MODE == kNormRes ? N : 1];
  if constexpr (NORM) {
    const long b = row / a.rows_per_batch;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = (k * per_row + t) * V;
      const bool in = e < a.D;
      vw[k] = in && a.w != nullptr ? load_raw<V, T>(reinterpret_cast<const T*>(a.w) + e) : zero_raw<V, T>();
      vscale[k] = in && a.scale != nullptr
                      ? load_raw<V, T>(reinterpret_cast<const T*>(a.scale) + b * a.ld_scale + e)
                      : zero_raw<V, T>();
      vshift[k] = in && a.shift != nullptr
                      ? load_raw<V, T>(reinterpret_cast<const T*>(a.shift) + b * a.ld_shift + e)
                      : zero_raw<V, T>();
      if constexpr (MODE == kNormRes)
        vgate[k] = in && a.gate != nullptr ? load_raw<V, T>(reinterpret_cast<const T*>(a.gate) + b * a.ld_gate + e)
                                           : zero_raw<V, T>();
    }
  }
  float y[N * V];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float* const yk = y + k * V;
    to_f32<V, T>(x[k], yk);
    if constexpr (TWO) {
      float f[V];
      to_f32<V, T>(x2[k], f);
      if constexpr (MODE == kSwiglu) {
#pragma unroll
        for (int j = 0; j < V; ++j) yk[j] = silu_mul(yk[j], f[j]);
      } else {
        float g[V];
        to_f32<V, T>(vgate[k], g);
#pragma unroll
        for (int j = 0; j < V; ++j) yk[j] = fmaf(a.gate != nullptr ? g[j] : 1.f, yk[j], f[j]);
        const int e = (k * per_row + t) * V;
        if (live && e < a.D) store_v<V, T>(reinterpret_cast<T*>(a.h) + row * a.ldh + e, yk);
      }
    }
  }
  if constexpr (NORM) {
    const float ss = row_reduce<false>(square_sum(y), lanes, warps, red[0]);
    const float rstd = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float w[V], sc[V], sh[V];
      to_f32<V, T>(vw[k], w);
      to_f32<V, T>(vscale[k], sc);
      to_f32<V, T>(vshift[k], sh);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float mul = (a.w != nullptr ? w[j] : 1.f) * (1.f + sc[j]);
        y[k * V + j] = fmaf(y[k * V + j] * rstd, mul, sh[j]);
      }
    }
  }
  const float m = row_reduce<true>(amax_all(y), lanes, warps, red[1]);
  float s, inv;
  row_scale(m, s, inv);
  if (live && t == 0) a.s[row] = s;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int e = (k * per_row + t) * V;
    if (live && e < a.D) store_q<V>(a.q + row * a.ldq + e, y + k * V, inv);
  }
}

// Many rows of a norm.  A block belongs to one sample (blockIdx.y) and keeps that
// sample's w * (1 + scale), shift and gate in shared memory as fp32; its row groups
// (a warp each, or the whole block for a wide row) go over the sample's rows with
// the next row's loads under the reductions of this one.
template <int MODE, typename T, int V, int N, bool MULTI>
__global__ void __launch_bounds__(MULTI ? 32 * kMaxWarps : 128, MULTI ? 1 : N > 5 && V == 8 ? 2 : MODE == kNormRes ? 3 : 4)
    norm_sample_kernel(const QuantArgs a, int warps) {
  constexpr bool TWO = MODE == kNormRes;
  constexpr int H = V == 8 ? 4 : V;  // a vector lies in V / H planes, so that wide reads meet no bank twice
  extern __shared__ __align__(16) float vec[];
  __shared__ float red[2][32];
  dependency_wait();
  const int slots = (a.D + V - 1) / V;
  float* const s_mul = vec;  // each [V / H][slots][H]
  float* const s_shift = s_mul + slots * V;
  float* const s_gate = s_shift + slots * V;
  const long b = blockIdx.y;
  const int per_row = MULTI ? 32 * warps : 32;
  const int t = MULTI ? threadIdx.x : threadIdx.x % 32;
  const int nw = MULTI ? warps : 1;
  const long stride = (long)gridDim.x * (MULTI ? 1 : 4);
  auto in = [&](int k) { return (V == 8 && k < N - 1) || (k * per_row + t) * V < a.D; };  // V = 8: N is exact
  auto vector = [&](const float* v, int k, float* f) {
    const int slot = min(k * per_row + t, slots - 1);
#pragma unroll
    for (int h = 0; h < V / H; ++h) {
      if constexpr (H == 4) {
        const float4 q4 = *reinterpret_cast<const float4*>(v + (h * slots + slot) * 4);
        f[4 * h] = q4.x; f[4 * h + 1] = q4.y; f[4 * h + 2] = q4.z; f[4 * h + 3] = q4.w;
      } else if constexpr (H == 2) {
        const float2 q2 = *reinterpret_cast<const float2*>(v + slot * 2);
        f[0] = q2.x; f[1] = q2.y;
      } else {
        f[0] = v[slot];
      }
    }
  };
  using R_ = Raw<V, T>;
  R_ x[N], x2[TWO ? N : 1];
  auto load_row = [&](long row) {
    const T* px = reinterpret_cast<const T*>(a.x) + row * a.ldx + t * V;
    const T* p2 = reinterpret_cast<const T*>(a.res) + row * a.ldr + t * V;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      x[k] = in(k) ? load_once<V, T>(px + k * per_row * V) : zero_raw<V, T>();
      if constexpr (TWO) x2[k] = in(k) ? load_once<V, T>(p2 + k * per_row * V) : zero_raw<V, T>();
    }
  };
  long r = (long)blockIdx.x * (MULTI ? 1 : 4) + (MULTI ? 0 : threadIdx.x / 32);
  if (r < a.rows_per_batch) load_row(b * a.rows_per_batch + r);
  // the sample's vectors, while the first rows are on their way
#pragma unroll 2
  for (int slot = threadIdx.x; slot < slots; slot += blockDim.x) {
    const int e = slot * V;
    R_ w, sc, sh, g;
    if (a.w != nullptr) w = load_raw<V, T>(reinterpret_cast<const T*>(a.w) + e);
    if (a.scale != nullptr) sc = load_raw<V, T>(reinterpret_cast<const T*>(a.scale) + b * a.ld_scale + e);
    if (a.shift != nullptr) sh = load_raw<V, T>(reinterpret_cast<const T*>(a.shift) + b * a.ld_shift + e);
    if (TWO && a.gate != nullptr) g = load_raw<V, T>(reinterpret_cast<const T*>(a.gate) + b * a.ld_gate + e);
    float f[V], m[V];
    auto put = [&](float* v, const float* f) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[(j / H * slots + slot) * H + j % H] = f[j];
    };
#pragma unroll
    for (int j = 0; j < V; ++j) m[j] = 1.f;
    if (a.w != nullptr) to_f32<V, T>(w, m);
    if (a.scale != nullptr) {
      to_f32<V, T>(sc, f);
#pragma unroll
      for (int j = 0; j < V; ++j) m[j] *= 1.f + f[j];
    }
    put(s_mul, m);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = 0.f;
    if (a.shift != nullptr) to_f32<V, T>(sh, f);
    put(s_shift, f);
    if constexpr (TWO) {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = 1.f;
      if (a.gate != nullptr) to_f32<V, T>(g, f);
      put(s_gate, f);
    }
  }
  __syncthreads();
  for (; r < a.rows_per_batch; r += stride) {
    const long row = b * a.rows_per_batch + r;
    float y[N * V];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float* const yk = y + k * V;
      to_f32<V, T>(x[k], yk);
      if constexpr (TWO) {
        float f[V], g[V];
        to_f32<V, T>(x2[k], f);
        vector(s_gate, k, g);
        if constexpr (V > 1) {
#pragma unroll
          for (int j = 0; j < V; j += 2)
            unpair(fma2(pair(g[j], g[j + 1]), pair(yk[j], yk[j + 1]), pair(f[j], f[j + 1])), yk[j], yk[j + 1]);
        } else {
          yk[0] = fmaf(g[0], yk[0], f[0]);
        }
        if (!in(k)) {  // the clamped slot's gate may be NaN or infinite
#pragma unroll
          for (int j = 0; j < V; ++j) yk[j] = 0.f;
        }
      }
    }
    if (r + stride < a.rows_per_batch) load_row(row + stride);
    if constexpr (TWO) {
      T* const h = reinterpret_cast<T*>(a.h) + row * a.ldh + t * V;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (in(k)) store_v<V, T>(h + k * per_row * V, y + k * V);
    }
    const float ss = row_reduce<false>(square_sum(y), 32, nw, red[0]);
    const float rstd = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float* const yk = y + k * V;
      float mul[V], sh[V];
      vector(s_mul, k, mul);
      vector(s_shift, k, sh);
      if constexpr (V > 1) {
#pragma unroll
        for (int j = 0; j < V; j += 2)
          unpair(fma2(mul2(pair(yk[j], yk[j + 1]), pair(rstd, rstd)), pair(mul[j], mul[j + 1]), pair(sh[j], sh[j + 1])),
                 yk[j], yk[j + 1]);
      } else {
        yk[0] = fmaf(yk[0] * rstd, mul[0], sh[0]);
      }
      if (!in(k)) {
#pragma unroll
        for (int j = 0; j < V; ++j) yk[j] = 0.f;
      }
    }
    const float m = row_reduce<true>(amax_all(y), 32, nw, red[1]);
    float s, inv;
    row_scale(m, s, inv);
    if (t == 0) a.s[row] = s;
    int8_t* const q = a.q + row * a.ldq + t * V;
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (in(k)) store_q<V>(q + k * per_row * V, y + k * V, inv);
  }
}

// Rows too wide for the registers of one block: the block goes over the row
// once for each reduction and once for the rounding.
template <int MODE, typename T>
__device__ __forceinline__ float wide_h(const QuantArgs& a, long row, long b, int e, bool store) {
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx + e;
  float f = to_f(*x);
  if constexpr (MODE == kSwiglu) f = silu_mul(f, to_f(x[a.D]));
  if constexpr (MODE == kNormRes) {
    const float g = a.gate != nullptr ? to_f(reinterpret_cast<const T*>(a.gate)[b * a.ld_gate + e]) : 1.f;
    f = fmaf(g, f, to_f(reinterpret_cast<const T*>(a.res)[row * a.ldr + e]));
    if (store) from_f(f, reinterpret_cast<T*>(a.h) + row * a.ldh + e);
  }
  return f;
}
template <int MODE, typename T>
__device__ __forceinline__ float wide_y(const QuantArgs& a, long row, long b, int e, float rstd) {
  float f = wide_h<MODE, T>(a, row, b, e, false);
  if constexpr (MODE >= kNorm) {
    float mul = a.w != nullptr ? to_f(reinterpret_cast<const T*>(a.w)[e]) : 1.f;
    if (a.scale != nullptr) mul *= 1.f + to_f(reinterpret_cast<const T*>(a.scale)[b * a.ld_scale + e]);
    f = fmaf(f * rstd, mul, a.shift != nullptr ? to_f(reinterpret_cast<const T*>(a.shift)[b * a.ld_shift + e]) : 0.f);
  }
  return f;
}
template <int MODE, typename T>
__global__ void __launch_bounds__(512) quant_wide_kernel(const QuantArgs a) {
  __shared__ float red[2][32];
  dependency_wait();
  const int warps = blockDim.x / 32;
  const long row = blockIdx.x;
  const long b = MODE >= kNorm ? row / a.rows_per_batch : 0;
  float rstd = 1.f;
  if constexpr (MODE >= kNorm) {
    float ss = 0.f;
    for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
      const float f = wide_h<MODE, T>(a, row, b, e, true);
      ss += f * f;
    }
    ss = row_reduce<false>(ss, 32, warps, red[0]);
    rstd = rsqrtf(ss / (float)a.D + a.eps);
  }
  float m = 0.f;
  for (int e = threadIdx.x; e < a.D; e += blockDim.x) m = amax2(wide_y<MODE, T>(a, row, b, e, rstd), 0.f, m);
  m = row_reduce<true>(m, 32, warps, red[1]);
  float s, inv;
  row_scale(m, s, inv);
  if (threadIdx.x == 0) a.s[row] = s;
  for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
    const float y[1] = {wide_y<MODE, T>(a, row, b, e, rstd)};
    store_q<1>(a.q + row * a.ldq + e, y, inv);
  }
}

// q * s.  Rows of whole 16-byte groups: a thread turns 16 values of one row into
// 32 (or 64) bytes; else neighbouring lanes take neighbouring values, V each.
template <typename T>
__global__ void __launch_bounds__(256) dequant_vec_kernel(const int8_t* q, long ldq, const float* s, long groups,
                                                          int per_row, T* out) {
  dependency_wait();
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= groups) return;
  const long row = groups <= 0x7FFFFFFFL ? (long)((unsigned)i / (unsigned)per_row) : i / per_row;
  const int e = (int)(i - row * per_row) * 16;
  const uint4 v = *reinterpret_cast<const uint4*>(q + row * ldq + e);
  const float sc = s[row];
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)(int8_t)(w[2 * g + j / 4] >> (8 * (j % 4))) * sc;
    store_v<8, T>(out + i * 16 + g * 8, f);
  }
}
template <typename T, int V>
__global__ void __launch_bounds__(256) dequant_rows_kernel(const int8_t* q, long ldq, const float* s, long R, int D,
                                                           T* out) {
  dependency_wait();
  const long row = (long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= R) return;
  const float sc = s[row];
  const int step = blockDim.x * V;
  for (int e0 = threadIdx.x * V; e0 < D; e0 += 4 * step) {
    uint16_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int8_t* p = q + row * ldq + e0 + j * step;
      v[j] = e0 + j * step >= D ? 0 : V == 2 ? *reinterpret_cast<const uint16_t*>(p) : (uint16_t)(uint8_t)*p;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float f[2] = {(float)(int8_t)v[j] * sc, (float)(int8_t)(v[j] >> 8) * sc};
      if (e0 + j * step < D) store_v<V, T>(out + row * D + e0 + j * step, f);
    }
  }
}

template <typename T>
void launch_dequant(const int8_t* q, long ldq, const float* s, long R, int D, T* out, cudaStream_t stream) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(q) | (R > 1 ? (uintptr_t)ldq : 0);
  const bool vec = D % 16 == 0 && bits % 16 == 0;
  const int V = D % 2 == 0 && bits % 2 == 0 ? 2 : 1;
  // lanes a row, the rest of 256 threads over rows: the most that leave few of a lane's four slots idle
  int lanes = 32, slots = 1 << 30;
  for (int l = 256; l >= 32; l /= 2) {
    const int n = (D + 4 * l * V - 1) / (4 * l * V) * 4 * l;
    if (n < slots) { slots = n; lanes = l; }
  }
  const long blocks = vec ? (R * (D / 16) + 255) / 256 : (R + 256 / lanes - 1) / (256 / lanes);
  TORCH_CHECK(blocks <= 0x7FFFFFFFL, "dequant_rows: too many rows");
  const dim3 block(lanes, 256 / lanes);
  if (vec) launch_dependent(dequant_vec_kernel<T>, (unsigned)blocks, 256, 0, stream, 1, q, ldq, s, R * (D / 16), D / 16, out);
  else if (V == 2) launch_dependent(dequant_rows_kernel<T, 2>, (unsigned)blocks, block, 0, stream, 1, q, ldq, s, R, D, out);
  else launch_dependent(dequant_rows_kernel<T, 1>, (unsigned)blocks, block, 0, stream, 1, q, ldq, s, R, D, out);
  count_launch();
}

template <int MODE, typename T, int V, int N>
void launch_few(const QuantArgs& a, int lanes, int warps, cudaStream_t stream) {
  const int threads = warps == 1 ? 128 : 32 * warps;
  const int per_block = warps == 1 ? threads / lanes : 1;
  const long blocks = (a.R + per_block - 1) / per_block;
  TORCH_CHECK(blocks <= 0x7FFFFFFFL, "harp quant: too many rows");
  launch_dependent(quant_rows_kernel<MODE, T, V, N>, (unsigned)blocks, threads, 0, stream, 1, a, lanes, warps);
}

template <int MODE, typename T, int V, int N, bool MULTI>
void launch_sample(const QuantArgs& a, int warps, size_t smem, cudaStream_t stream) {
  auto kern = norm_sample_kernel<MODE, T, V, N, MULTI>;
  const int threads = MULTI ? 32 * warps : 128, per_block = MULTI ? 1 : 4;
  static PerDevice<bool> configured;
  configured.get(a.device, [&] {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kVecSmem));
    return true;
  });
  int n = 0;
  C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem));
  const long samples = a.R / a.rows_per_batch;
  const long most = (a.rows_per_batch + per_block - 1) / per_block;
  const long blocks = std::max<long>(1, std::min<long>(most, (long)std::max(1, n) * num_sms() / samples));
  launch_dependent(kern, dim3((unsigned)blocks, (unsigned)samples), threads, smem, stream, 1, a, warps);
}

// The warps and groups a thread (at most `most`) with the fewest idle slots, of equals the fewest warps.
struct RowShape {
  int warps, n;
};
RowShape fewest_warps(int groups, int most) {
  RowShape best = {0, 0};
  for (int n = most; n >= 1; --n) {
    const int w = (groups + 32 * n - 1) / (32 * n);
    if (w > kMaxWarps) break;
    const int exact = (groups + 32 * w - 1) / (32 * w);
    if (best.warps == 0 || 50 * w * exact < 49 * best.warps * best.n) best = {w, exact};
  }
  return best;
}

// One of the instantiations of a kernel by V and N; `n` groups a thread at most.
#define HARP_QUANT_BY_N(V_, n, CALL)            \
  do {                                          \
    if constexpr (V_ == 8) {                    \
      switch (n) {                              \
        case 1: CALL(8, 1); break;              \
        case 2: CALL(8, 2); break;              \
        case 3: CALL(8, 3); break;              \
        case 4: CALL(8, 4); break;              \
        default: CALL(8, 5); break;             \
      }                                         \
    } else if ((n) <= 4) {                      \
      CALL(V_, 4);                              \
    } else if ((n) <= 8) {                      \
      CALL(V_, 8);                              \
    } else {                                    \
      CALL(V_, 16);                             \
    }                                           \
  } while (0)

template <int MODE, typename T, int V>
void launch(const QuantArgs& a, cudaStream_t stream) {
  const int groups = (a.D + V - 1) / V;
  const int lanes = V == 8 && groups <= 8 ? 8 : V == 8 && groups <= 16 ? 16 : 32;
  RowShape many;
  if (V == 8) {
    many = fewest_warps(groups, 5);
  } else {
    // one warp for up to 16 groups a lane (a 333 wide bf16 row: 6.1 us, 8.5 on two warps), else 8
    // groups a lane (1155 wide: 69 us with a residual, 118 with 16)
    const int most = groups <= 512 ? 16 : groups <= 256 * kMaxWarps ? 8 : 16;
    const int w = (groups + 32 * most - 1) / (32 * most);
    many = {w <= kMaxWarps ? w : 0, (groups + 32 * w - 1) / (32 * w)};
  }
  if (many.warps == 0) {
    TORCH_CHECK(a.R <= 0x7FFFFFFFL, "harp quant: too many rows");
    launch_dependent(quant_wide_kernel<MODE, T>, (unsigned)a.R, 512, 0, stream, 1, a);
  } else if (a.R * many.warps <= 8L * num_sms()) {
    // Few rows: latency counts, so as many warps as the row has groups for.
    auto with = [&](int n) { return std::max(1, (groups + 32 * n - 1) / (32 * n)); };
    const int n = (groups + 32 * kMaxWarps - 1) / (32 * kMaxWarps);
#define HARP_FEW(V_, N_) launch_few<MODE, T, V_, N_>(a, N_ == 1 ? lanes : 32, with(N_), stream)
    HARP_QUANT_BY_N(V, n, HARP_FEW);
#undef HARP_FEW
  } else {
    bool by_sample = false;
    if constexpr (MODE >= kNorm) {
      const size_t smem = (size_t)groups * V * 4 * (MODE == kNormRes ? 3 : 2);
      by_sample = smem <= kVecSmem && a.R / a.rows_per_batch <= 65535 && a.rows_per_batch >= 8;
      // A warp holds a row of up to 2560 values (its loads twice in fp32 with a residual: 1280). Wider
      // rows take the block, at a barrier for each reduction: a weighted norm of 17408 x 2304 bf16 took
      // 24.9 us on three warps a row, 19.2 on one; with a residual 4352 x 2560 17.9 and 14.2.
      if constexpr (V == 8 && !(MODE == kNormRes && sizeof(T) == 4)) {
        if (by_sample && groups > 160 && groups <= 320) {
          switch ((groups + 31) / 32) {
            case 6: launch_sample<MODE, T, 8, 6, false>(a, 1, smem, stream); break;
            case 7: launch_sample<MODE, T, 8, 7, false>(a, 1, smem, stream); break;
            case 8: launch_sample<MODE, T, 8, 8, false>(a, 1, smem, stream); break;
            case 9: launch_sample<MODE, T, 8, 9, false>(a, 1, smem, stream); break;
            default: launch_sample<MODE, T, 8, 10, false>(a, 1, smem, stream); break;
          }
          count_launch();
          return;
        }
      }
      if (by_sample) {
#define HARP_SAMPLE(V_, N_)                                                                 \
  (many.warps == 1 ? launch_sample<MODE, T, V_, N_, false>(a, many.warps, smem, stream)     \
                   : launch_sample<MODE, T, V_, N_, true>(a, many.warps, smem, stream))
        HARP_QUANT_BY_N(V, many.n, HARP_SAMPLE);
#undef HARP_SAMPLE
      }
    }
    if (!by_sample) {
#define HARP_MANY(V_, N_) launch_few<MODE, T, V_, N_>(a, N_ == 1 ? lanes : 32, many.warps, stream)
      HARP_QUANT_BY_N(V, many.n, HARP_MANY);
#undef HARP_MANY
    }
  }
  count_launch();
}

// width: 8, 2 or 1 values an access
template <int MODE>
void launch_mode(const QuantArgs& a, at::ScalarType t, int width, cudaStream_t stream) {
  if (t == at::kBFloat16) {
    if (width == 8) launch<MODE, bf16, 8>(a, stream);
    else if (width == 2) launch<MODE, bf16, 2>(a, stream);
    else launch<MODE, bf16, 1>(a, stream);
  } else {
    if (width == 8) launch<MODE, float, 8>(a, stream);
    else if (width == 2) launch<MODE, float, 2>(a, stream);
    else launch<MODE, float, 1>(a, stream);
  }
}

// Numbers in messages go through std::to_string: with a statically linked libstdc++ (as some
// toolchains give the library) a stream's number formatting meets another copy's locale.
std::string num(int64_t v) { return std::to_string(v); }

bool is_act_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }

void check_rows(const at::Tensor& x, const char* op, const char* name) {
  TORCH_CHECK(x.is_cuda(), op, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(is_act_type(x.scalar_type()), op, ": ", name, " must be bf16 or fp32, got ", c10::toString(x.scalar_type()));
  TORCH_CHECK(x.dim() == 2, op, ": ", name, " must be 2-D, got ", num(x.dim()), " dimensions");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= (1 << 30), op, ": ", name, " must have 1 to 2^30 columns");
  TORCH_CHECK(x.stride(1) == 1 || x.size(1) == 1, op, ": ", name, " needs a unit inner stride");
}

// The bits that keep a tensor's rows from alignment: its address and row stride in bytes.
uintptr_t low_bits(const at::Tensor& t) {
  uintptr_t b = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.dim() == 2 && t.size(0) > 1) b |= (uintptr_t)(t.stride(0) * t.element_size());
  return b;
}
int width_of(uintptr_t bits, int64_t D, int esize) {
  return D % 8 == 0 && bits % 16 == 0 ? 8 : D % 2 == 0 && bits % (2 * esize) == 0 ? 2 : 1;
}

// q [R, D] with rows on 16-byte boundaries (what TMA can address), s [R]
std::tuple<at::Tensor, at::Tensor> new_rows8(const at::Tensor& x, int64_t R, int64_t D) {
  const int64_t ld = (D + 15) / 16 * 16;
  at::Tensor q(at::detail::empty_strided_cuda({R, D}, {ld, 1}, at::kChar, x.device()));
  at::Tensor s(at::detail::empty_cuda({R}, at::kFloat, x.device(), c10::nullopt));
  return {q, s};
}

void set_out(QuantArgs& a, const at::Tensor& q, const at::Tensor& s) {
  a.q = reinterpret_cast<int8_t*>(q.data_ptr());
  a.ldq = q.stride(0);
  a.s = s.data_ptr<float>();
  a.R = q.size(0);
  a.D = (int)q.size(1);
  a.device = q.get_device();
}

std::tuple<at::Tensor, at::Tensor> rows_or_swiglu(const at::Tensor& x, int64_t D, bool swiglu) {
  const at::cuda::CUDAGuard guard(x.device());
  auto [q, s] = new_rows8(x, x.size(0), D);
  if (x.size(0) == 0) return {q, s};
  QuantArgs a = {};
  set_out(a, q, s);
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  const int width = width_of(low_bits(x), D, (int)x.element_size());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (swiglu) launch_mode<kSwiglu>(a, x.scalar_type(), width, stream);
  else launch_mode<kRows>(a, x.scalar_type(), width, stream);
  return {q, s};
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> quant_rows(const at::Tensor& x) {
  check_rows(x, "quant_rows", "x");
  return rows_or_swiglu(x, x.size(1), false);
}

std::tuple<at::Tensor, at::Tensor> swiglu_quant(const at::Tensor& gu) {
  check_rows(gu, "swiglu_quant", "gu");
  TORCH_CHECK(gu.size(1) % 2 == 0, "swiglu_quant: gu must have an even number of columns [g | u], got ", num(gu.size(1)));
  return rows_or_swiglu(gu, gu.size(1) / 2, true);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> rmsnorm_mod_quant(
    const at::Tensor& x, const c10::optional<at::Tensor>& w, const c10::optional<at::Tensor>& scale,
    const c10::optional<at::Tensor>& shift, int64_t rows_per_batch, double eps,
    const c10::optional<at::Tensor>& residual, const c10::optional<at::Tensor>& gate) {
  const char* op = "rmsnorm_mod_quant";
  check_rows(x, op, "x");
  const int64_t R = x.size(0), D = x.size(1);
  TORCH_CHECK(!gate.has_value() || residual.has_value(), op, ": gate needs a residual");
  const bool per_sample = scale.has_value() || shift.has_value() || gate.has_value();
  TORCH_CHECK(!per_sample || (rows_per_batch > 0 && R % rows_per_batch == 0), op, ": ",
              num(R), " rows are not whole samples of ", num(rows_per_batch));
  const at::cuda::CUDAGuard guard(x.device());
  QuantArgs a = {};
  uintptr_t bits = low_bits(x);
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  a.eps = (float)eps;
  a.rows_per_batch = per_sample ? rows_per_batch : std::max<int64_t>(R, 1);
  if (w.has_value()) {
    TORCH_CHECK(w->is_cuda() && w->device() == x.device() && w->scalar_type() == x.scalar_type() && w->dim() == 1 &&
                    w->size(0) == D && (D == 1 || w->stride(0) == 1),
                op, ": w must be a dense vector of ", num(D), " values of x's type on x's device");
    a.w = w->data_ptr();
    bits |= low_bits(*w);
  }
  auto vectors = [&](const c10::optional<at::Tensor>& v, const char* name, const void*& p, long& ld) {
    if (!v.has_value()) return;
    TORCH_CHECK(v->is_cuda() && v->device() == x.device() && v->scalar_type() == x.scalar_type() && v->dim() == 2 &&
                    v->size(1) == D && v->size(0) * rows_per_batch == R && (D == 1 || v->stride(1) == 1),
                op, ": ", name, " must be [", num(R / rows_per_batch), ", ", num(D),
                "] of x's type on x's device with a unit inner stride");
    p = v->data_ptr();
    ld = v->stride(0);
    bits |= low_bits(*v);
  };
  vectors(scale, "scale", a.scale, a.ld_scale);
  vectors(shift, "shift", a.shift, a.ld_shift);
  vectors(gate, "gate", a.gate, a.ld_gate);
  at::Tensor h;  // undefined (None) without a residual: h is x itself
  if (residual.has_value()) {
    TORCH_CHECK(residual->is_cuda() && residual->device() == x.device() &&
                    residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes() &&
                    (D == 1 || residual->stride(1) == 1),
                op, ": residual must have x's shape, type and device and a unit inner stride");
    a.res = residual->data_ptr();
    a.ldr = residual->stride(0);
    h = at::Tensor(at::detail::empty_cuda({R, D}, x.scalar_type(), x.device(), c10::nullopt));
    a.h = h.data_ptr();
    a.ldh = D;
    bits |= low_bits(*residual);
  }
  auto [q, s] = new_rows8(x, R, D);
  if (R == 0) return {q, s, h};
  set_out(a, q, s);
  const int width = width_of(bits, D, (int)x.element_size());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (residual.has_value()) launch_mode<kNormRes>(a, x.scalar_type(), width, stream);
  else launch_mode<kNorm>(a, x.scalar_type(), width, stream);
  return {q, s, h};
}

at::Tensor dequant_rows(const at::Tensor& q, const at::Tensor& s, bool f32) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kChar && q.dim() == 2, "dequant_rows: q must be a 2-D int8 CUDA tensor");
  TORCH_CHECK(q.size(1) <= (1 << 30) && (q.stride(1) == 1 || q.size(1) <= 1), "dequant_rows: q needs a unit inner stride");
  TORCH_CHECK(s.is_cuda() && s.device() == q.device() && s.scalar_type() == at::kFloat && s.dim() == 1 &&
                  s.size(0) == q.size(0) && (s.size(0) <= 1 || s.stride(0) == 1),
              "dequant_rows: s must be a dense fp32 vector with a scale for each row, on q's device");
  const at::cuda::CUDAGuard guard(q.device());
  const long R = q.size(0), D = q.size(1);
  at::Tensor out(at::detail::empty_cuda({R, D}, f32 ? at::kFloat : at::kBFloat16, q.device(), c10::nullopt));
  if (R == 0 || D == 0) return out;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int8_t* qp = reinterpret_cast<const int8_t*>(q.data_ptr());
  if (f32) launch_dequant<float>(qp, q.stride(0), s.data_ptr<float>(), R, (int)D, out.data_ptr<float>(), stream);
  else launch_dequant<bf16>(qp, q.stride(0), s.data_ptr<float>(), R, (int)D, reinterpret_cast<bf16*>(out.data_ptr()), stream);
  return out;
}

}  // namespace harp
