// rmsnorm.cu — RMS norm of a residual stream, with the residual's addition and
// 8-bit codes for the product that follows (linear.cu):
//
//   h = round(x + residual)             kept in the stream's type T (f32, f16, bf16)
//   rstd = 1 / sqrt(mean(h^2) + eps)    FP32 sums
//   y = round(h * rstd * gamma)
//   t = h * gamma, top = 127 (s8) or 448 (e4m3):
//   code = round_to_even(t * top / max|t|), scale = max|t| * rstd / top
//
// so code * scale stands for y. It stands beside LayerNormalization
// (glue.cu, src/OnnxSharp/Ops/AttnOps.cs:199-358) and DynamicQuantizeLinear
// (dqmm_i8.cu); the reference has neither the RMS form nor codes per row.
//
// The codes do not contain rstd: it cancels, so the row's maximum comes out of
// the same reduction as its sum of squares, and a code is a function of exact
// products alone. FP32 gives t * (top / max|t|) to about 4 * 2^-24 relative;
// only where that lies so close to a border between two codes that the error
// could decide (one element in some thousands) it is settled in FP64.
//
// One pass over the data: a row stays in the registers of its warp (short
// rows) or CTA. Bandwidth bounds it from a few hundred rows on, launch latency
// below.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "runtime.h"

namespace osc {
namespace {

constexpr float kTiny = 8.27180612553028e-25f;  // 2^-80: below it FP32 products of 24-bit factors lose bits
constexpr int kMaxThreads = 1024;
constexpr int kRegFloats = 16;                            // elements of a row a thread keeps
constexpr int kMaxRegCols = kMaxThreads * kRegFloats;     // longer rows are read again

struct NormArgs {
  const void* x;
  const void* residual;
  void* sum;
  const void* gamma;
  void* y;
  uint8_t* q;
  float* scales;
  long long x_ld, res_ld, sum_ld, y_ld, q_ld, rows;
  int cols;
  int q_dtype;
  float eps;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements as one access.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

// What a row's codes are made from, the same in all of its threads.
struct RowCode {
  float ratio;  // top / peak in FP32
  double peak;  // max|t|, exact
  float top;
  bool live;    // false: the codes are 0
};

// The code of t = h * g as its byte. r is t * top / peak to about 5 ulp; where
// a border between codes is nearer than that, FP64 decides.
__device__ __forceinline__ uint8_t code_s8(float t, float h, float g, const RowCode& c) {
  const float r = t * c.ratio;
  float n = rintf(r);
  if (fabsf(fabsf(r - n) - 0.5f) < 1e-4f)
    n = static_cast<float>(rint(static_cast<double>(h) * static_cast<double>(g) * static_cast<double>(c.top) / c.peak));
  return static_cast<uint8_t>(static_cast<int8_t>(static_cast<int>(n)));
}
__device__ __forceinline__ uint8_t code_e4m3(float t, float h, float g, const RowCode& c) {
  float r = t * c.ratio;
  const float a = fabsf(r);
  // borders: 2^-6 and up the middle of the 20 bits below e4m3's, below it the odd multiples of 2^-10
  const bool near_border = a >= 0.015625f
                               ? abs(static_cast<int>(__float_as_uint(a) & 0xFFFFFu) - 0x80000) <= 16
                               : fabsf(a * 512.0f - floorf(a * 512.0f) - 0.5f) < 1e-4f;
  if (near_border) {
    // toward zero with the last bit set when inexact: the second rounding then sees which side of a border it is on
    const double v = static_cast<double>(h) * static_cast<double>(g) * static_cast<double>(c.top) / c.peak;
    r = __double2float_rz(v);
    if (static_cast<double>(r) != v) r = __uint_as_float(__float_as_uint(r) | 1u);
  }
  return static_cast<uint8_t>(__nv_cvt_float_to_fp8(r, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ uint8_t code_of(float t, float h, float g, const RowCode& c, int q_dtype) {
  if (!c.live) return 0;
  return q_dtype == OSC_S8 ? code_s8(t, h, g, c) : code_e4m3(t, h, g, c);
}

// Sum and maximum over a row's threads: a warp's shuffles, then (rows of more
// than a warp) the warps' partials through shared memory, added in warp order.
template <bool WARP>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& peak, float2* part, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  peak = __reduce_max_sync(0xffffffffu, peak);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = make_float2(ss, __uint_as_float(peak));
    __syncthreads();
    float s = lane < warps ? part[lane].x : 0.0f;
    uint32_t m = lane < warps ? __float_as_uint(part[lane].y) : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    ss = s;
    peak = __reduce_max_sync(0xffffffffu, m);
    __syncthreads();  // part is used again
  }
}

// 1 / sqrt(mean + eps) from the row's sum of squares.
__device__ __forceinline__ float rstd_of(float ss, int cols, float eps) {
  return rsqrtf(ss / static_cast<float>(cols) + eps);
}

// Of a row whose finite elements' squares overflow FP32: the sum of (h / 2^64)^2
// (eps is lost against it). An infinite or NaN element gives 0 or NaN, as the formula does.
__device__ __forceinline__ float rstd_scaled(float ss, int cols) {
  return rsqrtf(ss / static_cast<float>(cols)) * 5.421010862427522e-20f;
}
constexpr float kDown = 5.421010862427522e-20f;  // 2^-64

__device__ __forceinline__ RowCode row_code(uint32_t peak, double exact_peak, int q_dtype) {
  RowCode c;
  const float p = __uint_as_float(peak);
  c.top = q_dtype == OSC_S8 ? 127.0f : 448.0f;
  c.live = p >= kTiny && peak < 0x7f800000u;
  c.ratio = c.live ? __fdiv_rn(c.top, p) : 0.0f;
  c.peak = exact_peak;
  return c;
}

__device__ __forceinline__ float row_scale(uint32_t peak, float rstd, const RowCode& c) {
  if (peak >= 0x7f800000u) return __uint_as_float(0x7fc00000u);  // no finite scale: the row is not a number
  return c.live ? __fdiv_rn(__uint_as_float(peak) * rstd, c.top) : 1.0f;
}

// max over the row of the bits that FP32 dropped of the largest |t|: products
// of two 24-bit factors have 48. (Products of 16-bit types fit FP32.)
template <bool WARP>
__device__ __forceinline__ float reduce_rest(float rest, float2* part, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) rest = fmaxf(rest, __shfl_xor_sync(0xffffffffu, rest, o));
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5].x = rest;
    __syncthreads();
    rest = lane < warps ? part[lane].x : -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rest = fmaxf(rest, __shfl_xor_sync(0xffffffffu, rest, o));
    __syncthreads();
  }
  return rest;
}
__device__ __forceinline__ float rest_of(float t, float h, float g, uint32_t peak) {
  if ((__float_as_uint(t) & 0x7fffffffu) != peak) return -INFINITY;
  const float rest = fmaf(h, g, -t);
  return t < 0.0f ? -rest : rest;
}

// A row in registers: WARP: one row a warp, several a CTA; else one row a CTA.
// Element (i * threads + thread) * VEC + e of the row is this thread's (i, e).
template <typename T, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : kMaxThreads) k_rmsnorm(const __grid_constant__ NormArgs p) {
  __shared__ float2 part[32];
  const int lanes = WARP ? 32 : static_cast<int>(blockDim.x);
  const int me = WARP ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int warps = static_cast<int>(blockDim.x) >> 5;
  const long long row = WARP ? static_cast<long long>(blockIdx.x) * warps + (threadIdx.x >> 5)
                             : static_cast<long long>(blockIdx.x);
  griddep_launch();
  griddep_wait();
  if (row >= p.rows) return;  // whole warps (WARP), none otherwise
  using V = Vec<T, VEC>;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* res = p.residual != nullptr ? static_cast<const T*>(p.residual) + row * p.res_ld : nullptr;
  const T* gamma = static_cast<const T*>(p.gamma);

  V raw[NV], add[NV], gv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e0 = (i * lanes + me) * VEC;
    if (e0 < p.cols) {
      raw[i] = *reinterpret_cast<const V*>(x + e0);
      if (res != nullptr) add[i] = *reinterpret_cast<const V*>(res + e0);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) raw[i].v[e] = from_f<T>(0.0f);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e0 = (i * lanes + me) * VEC;
    if (e0 < p.cols && gamma != nullptr) {
      gv[i] = *reinterpret_cast<const V*>(gamma + e0);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) gv[i].v[e] = from_f<T>(1.0f);
    }
  }
  float ss = 0.0f;
  uint32_t peak = 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e0 = (i * lanes + me) * VEC;
    if (e0 < p.cols && res != nullptr) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) raw[i].v[e] = from_f<T>(to_f<T>(raw[i].v[e]) + to_f<T>(add[i].v[e]));
      if (p.sum != nullptr) *reinterpret_cast<V*>(static_cast<T*>(p.sum) + row * p.sum_ld + e0) = raw[i];
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float h = to_f<T>(raw[i].v[e]);
      ss = fmaf(h, h, ss);
      if (p.q != nullptr) peak = max(peak, __float_as_uint(h * to_f<T>(gv[i].v[e])) & 0x7fffffffu);
    }
  }
  reduce_row<WARP>(ss, peak, part, warps);
  float rstd = rstd_of(ss, p.cols, p.eps);
  if (!(ss < INFINITY)) {  // the same in all of the row's threads
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float h = to_f<T>(raw[i].v[e]) * kDown;
        ss = fmaf(h, h, ss);
      }
    uint32_t none = 0u;
    reduce_row<WARP>(ss, none, part, warps);
    rstd = rstd_scaled(ss, p.cols);
  }

  if (p.y != nullptr) {
    T* y = static_cast<T*>(p.y) + row * p.y_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = (i * lanes + me) * VEC;
      if (e0 < p.cols) {
        V o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(to_f<T>(raw[i].v[e]) * rstd * to_f<T>(gv[i].v[e]));
        *reinterpret_cast<V*>(y + e0) = o;
      }
    }
  }
  if (p.q != nullptr) {
    double exact = static_cast<double>(__uint_as_float(peak));
    if constexpr (std::is_same<T, float>::value) {
      float rest = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = to_f<T>(raw[i].v[e]), g = to_f<T>(gv[i].v[e]);
          rest = fmaxf(rest, rest_of(h * g, h, g, peak));
        }
      exact += static_cast<double>(reduce_rest<WARP>(rest, part, warps));
    }
    const RowCode c = row_code(peak, exact, p.q_dtype);
    if (me == 0) p.scales[row] = row_scale(peak, rstd, c);
    uint8_t* q = p.q + row * p.q_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = (i * lanes + me) * VEC;
      if (e0 < p.cols) {
        Vec<uint8_t, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = to_f<T>(raw[i].v[e]), g = to_f<T>(gv[i].v[e]);
          o.v[e] = code_of(h * g, h, g, c, p.q_dtype);
        }
        *reinterpret_cast<Vec<uint8_t, VEC>*>(q + e0) = o;
      }
    }
  }
}

// Rows longer than a CTA's registers: the same steps element by element, the
// row read once more per step (from sum where it is kept: x or the residual may
// be sum's own buffer). A thread reads again only what it read and wrote itself.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads, 1) k_rmsnorm_long(const __grid_constant__ NormArgs p) {
  __shared__ float2 part[32];
  constexpr int warps = kMaxThreads / 32;
  const long long row = blockIdx.x;
  griddep_launch();
  griddep_wait();
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* res = p.residual != nullptr ? static_cast<const T*>(p.residual) + row * p.res_ld : nullptr;
  const T* gamma = static_cast<const T*>(p.gamma);
  T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.sum_ld : nullptr;
  const bool kept = res != nullptr && sum != nullptr;
  auto h_at = [&](int e) {
    if (kept) return to_f<T>(sum[e]);
    return res != nullptr ? to_f<T>(from_f<T>(to_f<T>(x[e]) + to_f<T>(res[e]))) : to_f<T>(x[e]);
  };
  auto g_at = [&](int e) { return gamma != nullptr ? to_f<T>(gamma[e]) : 1.0f; };
  float ss = 0.0f;
  uint32_t peak = 0u;
  for (int e = threadIdx.x; e < p.cols; e += kMaxThreads) {
    float h = to_f<T>(x[e]);
    if (res != nullptr) {
      const T s = from_f<T>(h + to_f<T>(res[e]));
      h = to_f<T>(s);
      if (kept) sum[e] = s;
    }
    ss = fmaf(h, h, ss);
    if (p.q != nullptr) peak = max(peak, __float_as_uint(h * g_at(e)) & 0x7fffffffu);
  }
  reduce_row<false>(ss, peak, part, warps);
  float rstd = rstd_of(ss, p.cols, p.eps);
  if (!(ss < INFINITY)) {
    ss = 0.0f;
    for (int e = threadIdx.x; e < p.cols; e += kMaxThreads) {
      const float h = h_at(e) * kDown;
      ss = fmaf(h, h, ss);
    }
    uint32_t none = 0u;
    reduce_row<false>(ss, none, part, warps);
    rstd = rstd_scaled(ss, p.cols);
  }
  RowCode c = {};
  if (p.q != nullptr) {
    double exact = static_cast<double>(__uint_as_float(peak));
    if constexpr (std::is_same<T, float>::value) {
      float rest = -INFINITY;
      for (int e = threadIdx.x; e < p.cols; e += kMaxThreads) {
        const float h = h_at(e), g = g_at(e);
        rest = fmaxf(rest, rest_of(h * g, h, g, peak));
      }
      exact += static_cast<double>(reduce_rest<false>(rest, part, warps));
    }
    c = row_code(peak, exact, p.q_dtype);
    if (threadIdx.x == 0) p.scales[row] = row_scale(peak, rstd, c);
  }
  T* y = p.y != nullptr ? static_cast<T*>(p.y) + row * p.y_ld : nullptr;
  uint8_t* q = p.q != nullptr ? p.q + row * p.q_ld : nullptr;
  for (int e = threadIdx.x; e < p.cols; e += kMaxThreads) {
    const float h = h_at(e), g = g_at(e);
    if (q != nullptr) q[e] = code_of(h * g, h, g, c, p.q_dtype);
    if (y != nullptr) y[e] = from_f<T>(h * rstd * g);
  }
}

// ------------------------------------------------------------------ host side
template <typename T, int VEC, int NV>
int launch_rows(osc_ctx* ctx, const NormArgs& p, int threads) {
  if (threads == 32) {
    constexpr int kRowsPerCta = 4;
    const long long blocks = (p.rows + kRowsPerCta - 1) / kRowsPerCta;
    return launch_pdl(ctx, k_rmsnorm<T, VEC, NV, true>, dim3(static_cast<unsigned>(blocks)), dim3(32 * kRowsPerCta), 0,
                      "k_rmsnorm", p);
  }
  return launch_pdl(ctx, k_rmsnorm<T, VEC, NV, false>, dim3(static_cast<unsigned>(p.rows)),
                    dim3(static_cast<unsigned>(threads)), 0, "k_rmsnorm", p);
}

template <typename T>
int launch_norm(osc_ctx* ctx, const NormArgs& p, bool vectors) {
  if (p.cols > kMaxRegCols)
    return launch_pdl(ctx, k_rmsnorm_long<T>, dim3(static_cast<unsigned>(p.rows)), dim3(kMaxThreads), 0,
                      "k_rmsnorm_long", p);
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  constexpr int NV = kRegFloats / VEC;
  // threads of a row: the fewest warps whose registers hold it
  const int threads = (p.cols + 32 * kRegFloats - 1) / (32 * kRegFloats) * 32;
  if (vectors) return launch_rows<T, VEC, NV>(ctx, p, threads);
  return launch_rows<T, 1, kRegFloats>(ctx, p, threads);
}

int type_bytes(int dtype) { return dtype == OSC_F32 ? 4 : 2; }

bool on(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace
}  // namespace osc

using namespace osc;

extern "C" {

OSC_API int osc_rmsnorm(osc_ctx* ctx, int dtype, const void* x, long long x_ld, const void* residual, long long res_ld,
                        long long rows, int cols, const void* gamma, float eps, void* sum, long long sum_ld, void* y,
                        long long y_ld, int q_dtype, void* q, long long q_ld, float* scales) {
  if (ctx == nullptr) return fail(OSC_EINVAL, "null context");
  if (dtype != OSC_F32 && dtype != OSC_F16 && dtype != OSC_BF16)
    return fail(OSC_EINVAL, "osc_rmsnorm: dtype %d is not f32, f16 or bf16", dtype);
  if (rows < 0 || cols <= 0 || rows >= (1ll << 31)) return fail(OSC_EINVAL, "osc_rmsnorm: bad shape [%lld, %d]", rows, cols);
  // smaller than this, eps cannot stand for the squares that FP32 drops
  if (!(eps >= 1e-30f) || !std::isfinite(eps)) return fail(OSC_EINVAL, "osc_rmsnorm: eps %g is not in [1e-30, inf)", static_cast<double>(eps));
  if (rows == 0) return OSC_OK;  // empty tensors may have no address
  if (y == nullptr && q == nullptr) return fail(OSC_EINVAL, "osc_rmsnorm: neither y nor q is asked for");
  if (q != nullptr && q_dtype != OSC_S8 && q_dtype != OSC_E4M3)
    return fail(OSC_EINVAL, "osc_rmsnorm: code type %d is not s8 or e4m3", q_dtype);
  if ((q != nullptr) != (scales != nullptr)) return fail(OSC_EINVAL, "osc_rmsnorm: codes and scales come together");
  if (sum != nullptr && residual == nullptr) return fail(OSC_EINVAL, "osc_rmsnorm: a sum without a residual");
  if (x_ld == 0) x_ld = cols;
  if (res_ld == 0) res_ld = cols;
  if (sum_ld == 0) sum_ld = cols;
  if (y_ld == 0) y_ld = cols;
  if (q_ld == 0) q_ld = cols;
  if (x_ld < cols || res_ld < cols || sum_ld < cols || y_ld < cols || q_ld < cols)
    return fail(OSC_EINVAL, "osc_rmsnorm: a row pitch below %d columns", cols);
  if (x == nullptr) return fail(OSC_EINVAL, "osc_rmsnorm: null x");
  const size_t e = static_cast<size_t>(type_bytes(dtype));
  if (!on(x, e) || !on(residual, e) || !on(gamma, e) || !on(sum, e) || !on(y, e) || !on(scales, 4))
    return fail(OSC_EINVAL, "osc_rmsnorm: a pointer is not aligned to its type");
  OSC_TRY(enter(ctx));
  if (fault_injected("launch")) return fail(OSC_EFAULT_INJECTED, "injected failure (launch)");
  NormArgs p = {};
  p.x = x;
  p.residual = residual;
  p.sum = sum;
  p.gamma = gamma;
  p.y = y;
  p.q = static_cast<uint8_t*>(q);
  p.scales = scales;
  p.x_ld = x_ld;
  p.res_ld = res_ld;
  p.sum_ld = sum_ld;
  p.y_ld = y_ld;
  p.q_ld = q_ld;
  p.rows = rows;
  p.cols = cols;
  p.q_dtype = q_dtype;
  p.eps = eps;
  // 16-byte accesses where every row of every tensor starts on one (codes: as many bytes as elements)
  const long long vec = 16 / static_cast<long long>(e);
  auto rows_fit = [&](const void* base, long long ld, size_t bytes) {
    return base == nullptr || (on(base, bytes) && ld % vec == 0);
  };
  const bool vectors = cols % vec == 0 && rows_fit(x, x_ld, 16) && rows_fit(residual, res_ld, 16) &&
                       rows_fit(sum, sum_ld, 16) && rows_fit(y, y_ld, 16) && rows_fit(gamma, 0, 16) &&
                       rows_fit(q, q_ld, static_cast<size_t>(vec));
  switch (dtype) {
    case OSC_F32: return launch_norm<float>(ctx, p, vectors);
    case OSC_F16: return launch_norm<__half>(ctx, p, vectors);
    default: return launch_norm<__nv_bfloat16>(ctx, p, vectors);
  }
}

}  // extern "C"
