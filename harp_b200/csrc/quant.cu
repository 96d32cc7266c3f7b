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
// row's reductions and the rounding.
#include "common.cuh"
#include "gemm_sm100.h"

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
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f(float v, bf16* p) { *p = __float2bfloat16(v); }

// V consecutive values as fp32 (V = 8: 16-byte aligned).
template <int V, typename T>
__device__ __forceinline__ void load_v(const T* p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_f(*p);
  } else if constexpr (sizeof(T) == 2) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = __uint_as_float(u[j] << 16);
      f[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
    }
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_v(T* p, const float (&f)[V]) {
  if constexpr (V == 1) {
    from_f(f[0], p);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// |v| joins a running maximum that keeps a NaN.
__device__ __forceinline__ float amax_nan(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}
// Non-negative floats and NaN order as their bits do.
__device__ __forceinline__ float warp_amax(float m) {
  return __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m)));
}
__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
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
__device__ __forceinline__ uint32_t round_byte(float y, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(y, inv), 12582912.f));
}
template <int V>
__device__ __forceinline__ void store_q(int8_t* p, const float (&y)[V], float inv) {
  if constexpr (V == 1) {
    *p = inv != 0.f ? (int8_t)(round_byte(y[0], inv) & 0xFFu) : (int8_t)0;
  } else {
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = round_byte(y[j], inv);
    uint2 o;
    o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    *reinterpret_cast<uint2*>(p) = inv != 0.f ? o : make_uint2(0u, 0u);
  }
}

// h of V values at column e of a row (and, with a residual, its store).
template <int MODE, int V, typename T>
__device__ __forceinline__ void load_h(const QuantArgs& a, long row, long b, int e, float (&f)[V], bool store) {
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx + e;
  load_v<V, T>(x, f);
  if constexpr (MODE == kSwiglu) {
    float u[V];
    load_v<V, T>(x + a.D, u);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = silu_mul(f[j], u[j]);
  } else if constexpr (MODE == kNormRes) {
    float r[V];
    load_v<V, T>(reinterpret_cast<const T*>(a.res) + row * a.ldr + e, r);
    if (a.gate != nullptr) {
      float g[V];
      load_v<V, T>(reinterpret_cast<const T*>(a.gate) + b * a.ld_gate + e, g);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = __fadd_rn(r[j], __fmul_rn(g[j], f[j]));
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] += r[j];
    }
    if (store) store_v<V, T>(reinterpret_cast<T*>(a.h) + row * a.ldh + e, f);
  }
}
// y of V values whose h is in f.
template <int V, typename T>
__device__ __forceinline__ void modulate(const QuantArgs& a, long b, int e, float rstd, float (&f)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] *= rstd;
  float t[V];
  if (a.w != nullptr) {
    load_v<V, T>(reinterpret_cast<const T*>(a.w) + e, t);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] *= t[j];
  }
  if (a.scale != nullptr) {
    load_v<V, T>(reinterpret_cast<const T*>(a.scale) + b * a.ld_scale + e, t);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] *= 1.f + t[j];
  }
  if (a.shift != nullptr) {
    load_v<V, T>(reinterpret_cast<const T*>(a.shift) + b * a.ld_shift + e, t);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] += t[j];
  }
}

// Sum (or NaN-keeping maximum) over the threads of a row: a warp, or the block.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, int warps, float* smem) {
  v = MAX ? warp_amax(v) : warp_sum_f(v);
  if (warps == 1) return v;
  if (threadIdx.x % 32 == 0) smem[threadIdx.x / 32] = v;
  __syncthreads();
  v = threadIdx.x % 32 < warps ? smem[threadIdx.x % 32] : 0.f;
  return MAX ? warp_amax(v) : warp_sum_f(v);
}

// One row for each `warps` warps, the row's values in registers: thread t holds
// N groups of V values, group k at column (k * 32 * warps + t) * V.  warps == 1:
// each warp of the block has a row of its own and nothing is shared; otherwise
// the block is one row.  V = 8 needs D % 8 == 0 and 16-byte aligned rows.
template <int MODE, typename T, int V, int N>
__global__ void __launch_bounds__(32 * kMaxWarps) quant_rows_kernel(const QuantArgs a, int warps) {
  __shared__ float red[2][32];
  const int per_row = 32 * warps;
  const long row = warps == 1 ? (long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : (long)blockIdx.x;
  if (row >= a.R) return;  // warps == 1: whole warps, no barrier follows
  const int t = warps == 1 ? threadIdx.x % 32 : threadIdx.x;
  const long b = MODE >= kNorm ? row / a.rows_per_batch : 0;
  float y[N][V];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int e = (k * per_row + t) * V;
    if (e < a.D) {
      load_h<MODE, V, T>(a, row, b, e, y[k], true);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) y[k][j] = 0.f;
    }
  }
  if constexpr (MODE >= kNorm) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) ss += y[k][j] * y[k][j];
    ss = row_reduce<false>(ss, warps, red[0]);
    const float rstd = rsqrtf(ss / (float)a.D + a.eps);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = (k * per_row + t) * V;
      if (e < a.D) modulate<V, T>(a, b, e, rstd, y[k]);
    }
  }
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) m = amax_nan(m, y[k][j]);
  m = row_reduce<true>(m, warps, red[1]);
  float s, inv;
  row_scale(m, s, inv);
  if (t == 0) a.s[row] = s;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int e = (k * per_row + t) * V;
    if (e < a.D) store_q<V>(a.q + row * a.ldq + e, y[k], inv);
  }
}

// Rows too wide for the registers of one block: the block goes over the row
// once for each reduction and once for the rounding.
template <int MODE, typename T>
__global__ void __launch_bounds__(512) quant_wide_kernel(const QuantArgs a) {
  __shared__ float red[2][32];
  const int warps = blockDim.x / 32;
  const long row = blockIdx.x;
  const long b = MODE >= kNorm ? row / a.rows_per_batch : 0;
  float rstd = 1.f;
  if constexpr (MODE >= kNorm) {
    float ss = 0.f;
    for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
      float f[1];
      load_h<MODE, 1, T>(a, row, b, e, f, true);
      ss += f[0] * f[0];
    }
    ss = row_reduce<false>(ss, warps, red[0]);
    rstd = rsqrtf(ss / (float)a.D + a.eps);
  }
  float m = 0.f;
  for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
    float f[1];
    load_h<MODE, 1, T>(a, row, b, e, f, false);
    if constexpr (MODE >= kNorm) modulate<1, T>(a, b, e, rstd, f);
    m = amax_nan(m, f[0]);
  }
  m = row_reduce<true>(m, warps, red[1]);
  float s, inv;
  row_scale(m, s, inv);
  if (threadIdx.x == 0) a.s[row] = s;
  for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
    float f[1];
    load_h<MODE, 1, T>(a, row, b, e, f, false);
    if constexpr (MODE >= kNorm) modulate<1, T>(a, b, e, rstd, f);
    store_q<1>(a.q + row * a.ldq + e, f, inv);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequant_rows_kernel(const int8_t* __restrict__ q, long ldq,
                                                           const float* __restrict__ s, long R, int D,
                                                           T* __restrict__ out, long ldo) {
  for (long row = blockIdx.x; row < R; row += gridDim.x) {
    const float sc = s[row];
    for (int e = threadIdx.x; e < D; e += blockDim.x) from_f((float)q[row * ldq + e] * sc, out + row * ldo + e);
  }
}

template <int MODE, typename T, int V, int N>
void launch_n(const QuantArgs& a, int warps, cudaStream_t stream) {
  const int rows_per_block = warps == 1 ? 4 : 1;
  const long grid = (a.R + rows_per_block - 1) / rows_per_block;
  TORCH_CHECK(grid <= 0x7FFFFFFFL, "harp quant: too many rows");
  quant_rows_kernel<MODE, T, V, N><<<(unsigned)grid, 32 * warps * rows_per_block, 0, stream>>>(a, warps);
}

template <int MODE, typename T>
void launch(const QuantArgs& a, bool vec, cudaStream_t stream) {
  // Groups of V values for each thread: the fewest warps that hold the row with
  // the fewest idle slots.
  const int V = vec ? 8 : 1, most = vec ? 5 : 16;
  const int groups = (a.D + V - 1) / V;
  int warps = 0, n = 0;
  double best = 0.0;
  for (int w = 1; w <= kMaxWarps; ++w) {
    const int need = (groups + 32 * w - 1) / (32 * w);
    if (need > most) continue;
    const double used = (double)groups / (32.0 * w * need);
    if (used > best * 1.02) { best = used; warps = w; n = need; }
  }
  if (warps == 0) {
    TORCH_CHECK(a.R <= 0x7FFFFFFFL, "harp quant: too many rows");
    quant_wide_kernel<MODE, T><<<(unsigned)a.R, 512, 0, stream>>>(a);
  } else if (vec) {
    switch (n) {
      case 1: launch_n<MODE, T, 8, 1>(a, warps, stream); break;
      case 2: launch_n<MODE, T, 8, 2>(a, warps, stream); break;
      case 3: launch_n<MODE, T, 8, 3>(a, warps, stream); break;
      case 4: launch_n<MODE, T, 8, 4>(a, warps, stream); break;
      default: launch_n<MODE, T, 8, 5>(a, warps, stream); break;
    }
  } else if (n <= 4) {
    launch_n<MODE, T, 1, 4>(a, warps, stream);
  } else if (n <= 8) {
    launch_n<MODE, T, 1, 8>(a, warps, stream);
  } else {
    launch_n<MODE, T, 1, 16>(a, warps, stream);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
}

template <int MODE>
void launch_mode(const QuantArgs& a, at::ScalarType t, bool vec, cudaStream_t stream) {
  if (t == at::kBFloat16) launch<MODE, bf16>(a, vec, stream);
  else launch<MODE, float>(a, vec, stream);
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

// 16-byte accesses are possible on every row of t.
bool vec_ok(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 &&
         (t.dim() < 2 || t.size(0) <= 1 || (t.stride(0) * t.element_size()) % 16 == 0);
}

// q [R, D] with rows on 16-byte boundaries (what TMA can address), s [R]
std::tuple<at::Tensor, at::Tensor> new_rows8(const at::Tensor& x, int64_t R, int64_t D) {
  const int64_t ld = (D + 15) / 16 * 16;
  at::Tensor q(at::detail::empty_cuda({R, ld}, at::kChar, x.device(), c10::nullopt));
  at::Tensor s(at::detail::empty_cuda({R}, at::kFloat, x.device(), c10::nullopt));
  return {ld == D ? q : q.narrow(1, 0, D), s};
}

void set_out(QuantArgs& a, const at::Tensor& q, const at::Tensor& s) {
  a.q = reinterpret_cast<int8_t*>(q.data_ptr());
  a.ldq = q.stride(0);
  a.s = s.data_ptr<float>();
  a.R = q.size(0);
  a.D = (int)q.size(1);
}

std::tuple<at::Tensor, at::Tensor> rows_or_swiglu(const at::Tensor& x, int64_t D, bool swiglu) {
  const at::cuda::CUDAGuard guard(x.device());
  auto [q, s] = new_rows8(x, x.size(0), D);
  if (x.size(0) == 0) return {q, s};
  QuantArgs a = {};
  set_out(a, q, s);
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  const bool vec = D % 8 == 0 && vec_ok(x);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (swiglu) launch_mode<kSwiglu>(a, x.scalar_type(), vec, stream);
  else launch_mode<kRows>(a, x.scalar_type(), vec, stream);
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
  bool vec = D % 8 == 0 && vec_ok(x);
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  a.eps = (float)eps;
  a.rows_per_batch = per_sample ? rows_per_batch : std::max<int64_t>(R, 1);
  if (w.has_value()) {
    TORCH_CHECK(w->is_cuda() && w->device() == x.device() && w->scalar_type() == x.scalar_type() && w->dim() == 1 &&
                    w->size(0) == D && (D == 1 || w->stride(0) == 1),
                op, ": w must be a dense vector of ", num(D), " values of x's type on x's device");
    a.w = w->data_ptr();
    vec = vec && vec_ok(*w);
  }
  auto vectors = [&](const c10::optional<at::Tensor>& v, const char* name, const void*& p, long& ld) {
    if (!v.has_value()) return;
    TORCH_CHECK(v->is_cuda() && v->device() == x.device() && v->scalar_type() == x.scalar_type() && v->dim() == 2 &&
                    v->size(1) == D && v->size(0) * rows_per_batch == R && (D == 1 || v->stride(1) == 1),
                op, ": ", name, " must be [", num(R / rows_per_batch), ", ", num(D),
                "] of x's type on x's device with a unit inner stride");
    p = v->data_ptr();
    ld = v->stride(0);
    vec = vec && vec_ok(*v);
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
    vec = vec && vec_ok(*residual);
  }
  auto [q, s] = new_rows8(x, R, D);
  if (R == 0) return {q, s, h};
  set_out(a, q, s);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (residual.has_value()) launch_mode<kNormRes>(a, x.scalar_type(), vec, stream);
  else launch_mode<kNorm>(a, x.scalar_type(), vec, stream);
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
  const unsigned grid = (unsigned)std::min<long>(R, 1L << 20);
  const int8_t* qp = reinterpret_cast<const int8_t*>(q.data_ptr());
  if (f32)
    dequant_rows_kernel<float><<<grid, 256, 0, stream>>>(qp, q.stride(0), s.data_ptr<float>(), R, (int)D, out.data_ptr<float>(), D);
  else
    dequant_rows_kernel<bf16><<<grid, 256, 0, stream>>>(qp, q.stride(0), s.data_ptr<float>(), R, (int)D,
                                                        reinterpret_cast<bf16*>(out.data_ptr()), D);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
  return out;
}

}  // namespace harp
