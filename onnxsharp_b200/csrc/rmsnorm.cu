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
// rows) or CTA, 16 elements a thread (8 or 32 of a 16-bit type: 61.6 and 107 us
// in place of 53.5 for 8192 rows of 4096 bf16 with a residual; CTAs that walk
// rows, loading the next ahead, 84). Launch latency bounds a few rows: 1.7 us for
// one of 4096. Of 8192 rows of 4096, f32 reaches 6.3 TB/s (42.5 us); bf16 with a
// residual 5.1 (52.5 us), with e4m3 codes 3.7 (64 us): a thread's 16 elements
// are then too little beside a row's own steps (its sum over warps, its scale),
// and the codes' arithmetic fills 60 % of the issue slots.
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
constexpr int kRowsPerCta = 4;                        // rows of one warp each
constexpr int kSingles = 8;                           // elements, where they are loaded one by one

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

// The larger, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// What a row's codes are made from, the same in all of its threads.
struct RowCode {
  float ratio;  // top / peak in FP32; 0 where the codes are 0
  double peak;  // max|t|, exact
  float top;
};

// t * top / peak as FP64 has it, from the exact factors of t.
__device__ __forceinline__ double exact_ratio(float h, float g, const RowCode& c) {
  return static_cast<double>(h) * static_cast<double>(g) * static_cast<double>(c.top) / c.peak;
}

// N codes of t(e) = h(e) * g(e) as bytes. r = t * ratio is good to about 5 ulp;
// where a border between two codes is nearer than that, FP64 decides. Whether
// any of the N is that near is one minimum or maximum, so the branch is taken
// once for all of them (for one group in some hundreds).
template <int N, class Tt, class H, class G>
__device__ __forceinline__ void codes_s8(Tt t, H h, G g, const RowCode& c, uint8_t (&o)[N]) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to the nearest integer, ties to even
  constexpr float kNear = 0.4999f;
  float n[N], far = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float r = t(e) * c.ratio;
    n[e] = r + kRound;
    far = fmaxf(far, fabsf(r - (n[e] - kRound)));
  }
  if (far > kNear) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float r = t(e) * c.ratio;
      if (fabsf(r - (n[e] - kRound)) > kNear) n[e] = static_cast<float>(rint(exact_ratio(h(e), g(e), c))) + kRound;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = static_cast<uint8_t>(__float_as_uint(n[e]));  // the integer's low byte
}
template <int N, class Tt, class H, class G>
__device__ __forceinline__ void codes_e4m3(Tt t, H h, G g, const RowCode& c, uint8_t (&o)[N]) {
  // 0 where the 20 bits below e4m3's are within 16 of their middle, a border from 2^-6 up
  auto off_middle = [](float r) { return ((__float_as_uint(r) + 16u) & 0xFFFE0u) ^ 0x80000u; };
  constexpr float kSmall = 0.015625f;  // 2^-6: under it the borders lie otherwise, and every value but 0 is looked at
  float r[N], least = kSmall;
  uint32_t middle = 1u;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    r[e] = t(e) * c.ratio;
    least = fminf(least, fabsf(r[e]));
    middle = min(middle, off_middle(r[e]));
  }
  if (least < kSmall || middle == 0u) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (off_middle(r[e]) == 0u || (fabsf(r[e]) < kSmall && r[e] != 0.0f)) {
        // toward zero with the last bit set when inexact: the second rounding then sees which side of a border it is on
        const double v = exact_ratio(h(e), g(e), c);
        r[e] = __double2float_rz(v);
        if (static_cast<double>(r[e]) != v) r[e] = __uint_as_float(__float_as_uint(r[e]) | 1u);
      }
  }
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(r[e], r[e + 1]), __NV_SATFINITE, __NV_E4M3);
      o[e] = static_cast<uint8_t>(two);
      o[e + 1] = static_cast<uint8_t>(two >> 8);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = __nv_cvt_float_to_fp8(r[e], __NV_SATFINITE, __NV_E4M3);
  }
}
// A row that has no codes (its ratio is 0): zeros, whatever t is.
template <int N, class Tt, class H, class G>
__device__ __forceinline__ void codes_of(Tt t, H h, G g, const RowCode& c, int q_dtype, uint8_t (&o)[N]) {
  if (c.ratio == 0.0f) {
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0;
  } else if (q_dtype == OSC_S8) {
    codes_s8<N>(t, h, g, c, o);
  } else {
    codes_e4m3<N>(t, h, g, c, o);
  }
}

// Sum and maximum over a row's threads: a warp's shuffles, then (rows of more
// than a warp) the warps' partials through shared memory, added in warp order.
// `peak` is the bits of a float that is not negative.
template <bool WARP, bool PEAK>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& peak, float2* part, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (PEAK) peak = __reduce_max_sync(0xffffffffu, peak);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = make_float2(ss, __uint_as_float(peak));
    __syncthreads();
    ss = lane < warps ? part[lane].x : 0.0f;
    peak = lane < warps ? __float_as_uint(part[lane].y) : 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (PEAK) peak = __reduce_max_sync(0xffffffffu, peak);
  }
}

// What rstd is the inverse root of, from the row's sum of squares.
__device__ __forceinline__ float square_of(float ss, int cols, float eps) {
  return ss / static_cast<float>(cols) + eps;
}

// Where that overflows FP32 from finite elements: ss is the sum of (h / 2^80)^2.
// 2^31 elements below 2^128 stay below 2^127 so, a sum that overflowed is 2^-32 at
// least, and eps counts where it is large too. An infinite or NaN element gives 0
// or NaN, as the formula does.
constexpr float kDown = 8.27180612553028e-25f;  // 2^-80
__device__ __forceinline__ float rstd_scaled(float ss, int cols, float eps) {
  return rsqrtf(square_of(ss, cols, eps * kDown * kDown)) * kDown;
}

__device__ __forceinline__ bool live_peak(uint32_t peak) {
  return __uint_as_float(peak) >= kTiny && peak < 0x7f800000u;
}
__device__ __forceinline__ RowCode row_code(uint32_t peak, double exact_peak, int q_dtype) {
  RowCode c;
  c.top = q_dtype == OSC_S8 ? 127.0f : 448.0f;
  c.ratio = live_peak(peak) ? __fdiv_rn(c.top, __uint_as_float(peak)) : 0.0f;
  c.peak = exact_peak;
  return c;
}
__device__ __forceinline__ float row_scale(uint32_t peak, float rstd, const RowCode& c) {
  if (peak >= 0x7f800000u) return __uint_as_float(0x7fc00000u);  // no finite scale: the row is not a number
  return live_peak(peak) ? __fdiv_rn(__uint_as_float(peak) * rstd, c.top) : 1.0f;
}

// What FP32 dropped of the largest |t| (products of two 24-bit factors have 48
// bits; those of 16-bit types fit FP32): the maximum over the elements whose
// FP32 product is the peak, as an integer that orders like the float.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u >> 31) != 0u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
  return __uint_as_float((u >> 31) != 0u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t rest_of(float t, float h, float g, uint32_t peak) {
  if ((__float_as_uint(t) & 0x7fffffffu) != peak) return 0u;  // below every float
  const float rest = fmaf(h, g, -t);
  return ordered(t < 0.0f ? -rest : rest);
}
template <bool WARP>
__device__ __forceinline__ double exact_peak_of(uint32_t peak, uint32_t rest, uint32_t* shared_rest) {
  rest = __reduce_max_sync(0xffffffffu, rest);
  if constexpr (!WARP) {
    if ((threadIdx.x & 31) == 0 && rest != 0u) atomicMax(shared_rest, rest);
    __syncthreads();
    rest = *shared_rest;
  }
  return static_cast<double>(__uint_as_float(peak)) + (rest != 0u ? static_cast<double>(from_ordered(rest)) : 0.0);
}

// A row a warp (WARP) or a row a CTA, held in registers: element
// (i * lanes + me) * VEC + e is this thread's (i, e). Codes are a kernel of their
// own (CODES, y beside them if asked for): without them it needs fewer registers,
// and 8192 rows of 4096 bf16 with a residual take 52.1 us for 55.7.
template <typename T, int VEC, int NV, bool WARP, bool CODES>
__global__ void __launch_bounds__(WARP ? 32 * kRowsPerCta : kMaxThreads) k_rmsnorm(const __grid_constant__ NormArgs p) {
  using V = Vec<T, VEC>;
  constexpr bool kKeep = sizeof(T) == 2;  // t is kept where it takes more than a product to have it again
  __shared__ float2 part[32];
  __shared__ uint32_t shared_rest;
  const int warps = static_cast<int>(blockDim.x) >> 5;
  const long long row = WARP ? static_cast<long long>(blockIdx.x) * warps + (threadIdx.x >> 5)
                             : static_cast<long long>(blockIdx.x);
  if (!WARP && threadIdx.x == 0) shared_rest = 0u;  // (used behind the row's meeting)
  griddep_launch();
  griddep_wait();
  if (row >= p.rows) return;  // whole warps (WARP), none otherwise
  const int lanes = WARP ? 32 : static_cast<int>(blockDim.x);
  const int me = static_cast<int>(WARP ? threadIdx.x & 31 : threadIdx.x);
  auto at = [&](int i) { return (i * lanes + me) * VEC; };

  V raw[NV], add[NV], gv[NV];
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* res = p.residual != nullptr ? static_cast<const T*>(p.residual) + row * p.res_ld : nullptr;
  const T* gamma = static_cast<const T*>(p.gamma);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (at(i) < p.cols) {
      raw[i] = *reinterpret_cast<const V*>(x + at(i));
      if (res != nullptr) add[i] = *reinterpret_cast<const V*>(res + at(i));
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) raw[i].v[e] = add[i].v[e] = from_f<T>(0.0f);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (at(i) < p.cols && gamma != nullptr) {
      gv[i] = *reinterpret_cast<const V*>(gamma + at(i));
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) gv[i].v[e] = from_f<T>(1.0f);
    }
  }
  if (res != nullptr) {
    T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.sum_ld : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) raw[i].v[e] = from_f<T>(to_f<T>(raw[i].v[e]) + to_f<T>(add[i].v[e]));
      if (sum != nullptr && at(i) < p.cols) *reinterpret_cast<V*>(sum + at(i)) = raw[i];
    }
  }

  auto h_of = [&](int i, int e) { return to_f<T>(raw[i].v[e]); };
  auto g_of = [&](int i, int e) { return to_f<T>(gv[i].v[e]); };
  float t[kKeep ? NV : 1][kKeep ? VEC : 1] = {};
  auto t_of = [&](int i, int e) { return kKeep ? t[kKeep ? i : 0][kKeep ? e : 0] : h_of(i, e) * g_of(i, e); };
  float ss = 0.0f, top = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float h = h_of(i, e);
      ss = fmaf(h, h, ss);
      if (CODES) {
        if (kKeep) t[kKeep ? i : 0][kKeep ? e : 0] = h * g_of(i, e);
        top = max_nan(top, fabsf(t_of(i, e)));
      }
    }
  uint32_t peak = __float_as_uint(top) & 0x7fffffffu;  // a NaN is above every number
  reduce_row<WARP, CODES>(ss, peak, part, warps);
  const float square = square_of(ss, p.cols, p.eps);
  float rstd = rsqrtf(square);
  if (!(square < INFINITY)) {  // the same in all of the row's threads
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float h = h_of(i, e) * kDown;
        ss = fmaf(h, h, ss);
      }
    uint32_t none = 0u;
    if (!WARP) __syncthreads();  // part is written again
    reduce_row<WARP, false>(ss, none, part, warps);
    rstd = rstd_scaled(ss, p.cols, p.eps);
  }

  if (!CODES || p.y != nullptr) {
    T* y = static_cast<T*>(p.y) + row * p.y_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at(i) < p.cols) {
        V o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = from_f<T>(h_of(i, e) * rstd * g_of(i, e));
        *reinterpret_cast<V*>(y + at(i)) = o;
      }
  }
  if constexpr (CODES) {
    double exact = static_cast<double>(__uint_as_float(peak));
    if constexpr (std::is_same<T, float>::value) {
      uint32_t rest = 0u;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) rest = max(rest, rest_of(t_of(i, e), h_of(i, e), g_of(i, e), peak));
      exact = exact_peak_of<WARP>(peak, rest, &shared_rest);
    }
    const RowCode c = row_code(peak, exact, p.q_dtype);
    if (me == 0) p.scales[row] = row_scale(peak, rstd, c);
    uint8_t* q = p.q + row * p.q_ld;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at(i) < p.cols) {
        Vec<uint8_t, VEC> o;
        codes_of<VEC>([&](int e) { return t_of(i, e); }, [&](int e) { return h_of(i, e); },
                      [&](int e) { return g_of(i, e); }, c, p.q_dtype, o.v);
        *reinterpret_cast<Vec<uint8_t, VEC>*>(q + at(i)) = o;
      }
  }
}

// Rows longer than a CTA's registers: the same steps element by element, the
// row read once more per step (from sum where it is kept: x or the residual may
// be sum's own buffer). A thread reads again only what it read and wrote itself.
// Its squares are added 16 at a time in FP32 and those sums in FP64: rows of 2^24
// equal elements and more lost up to 4e-4 of their norm to additions that all round
// the same way. 148 x 20000 f32 takes 7.2 us for 6.8 so, 1000 x 33000 bf16 147 for
// 146 (a loop of 16 inside the other 9.0 and 151). Elements are counted unsigned:
// the step behind the last one may pass 2^31.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads, 1) k_rmsnorm_long(const __grid_constant__ NormArgs p) {
  __shared__ float2 part[32];
  __shared__ uint32_t shared_rest;
  if (threadIdx.x == 0) shared_rest = 0u;
  constexpr int warps = kMaxThreads / 32;
  const long long row = blockIdx.x;
  griddep_launch();
  griddep_wait();
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* res = p.residual != nullptr ? static_cast<const T*>(p.residual) + row * p.res_ld : nullptr;
  const T* gamma = static_cast<const T*>(p.gamma);
  T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.sum_ld : nullptr;
  const bool kept = res != nullptr && sum != nullptr;
  const uint32_t cols = static_cast<uint32_t>(p.cols);
  auto h_at = [&](uint32_t e) {
    if (kept) return to_f<T>(sum[e]);
    return res != nullptr ? to_f<T>(from_f<T>(to_f<T>(x[e]) + to_f<T>(res[e]))) : to_f<T>(x[e]);
  };
  auto g_at = [&](uint32_t e) { return gamma != nullptr ? to_f<T>(gamma[e]) : 1.0f; };
  auto squares = [&](auto h_of) {
    double total = 0.0;
    float some = 0.0f;
    uint32_t n = 0;
    for (uint32_t e = threadIdx.x; e < cols; e += kMaxThreads) {
      const float h = h_of(e);
      some = fmaf(h, h, some);
      if (++n % 16 == 0) {
        total += static_cast<double>(some);
        some = 0.0f;
      }
    }
    return static_cast<float>(total + static_cast<double>(some));
  };
  float top = 0.0f;
  float ss = squares([&](uint32_t e) {
    float h = to_f<T>(x[e]);
    if (res != nullptr) {
      const T s = from_f<T>(h + to_f<T>(res[e]));
      h = to_f<T>(s);
      if (kept) sum[e] = s;
    }
    if (p.q != nullptr) top = max_nan(top, fabsf(h * g_at(e)));
    return h;
  });
  uint32_t peak = __float_as_uint(top) & 0x7fffffffu;
  reduce_row<false, true>(ss, peak, part, warps);
  const float square = square_of(ss, p.cols, p.eps);
  float rstd = rsqrtf(square);
  if (!(square < INFINITY)) {
    ss = squares([&](uint32_t e) { return h_at(e) * kDown; });
    uint32_t none = 0u;
    __syncthreads();
    reduce_row<false, true>(ss, none, part, warps);
    rstd = rstd_scaled(ss, p.cols, p.eps);
  }
  RowCode c = {};
  if (p.q != nullptr) {
    double exact = static_cast<double>(__uint_as_float(peak));
    if constexpr (std::is_same<T, float>::value) {
      uint32_t rest = 0u;
      for (uint32_t e = threadIdx.x; e < cols; e += kMaxThreads) {
        const float h = h_at(e), g = g_at(e);
        rest = max(rest, rest_of(h * g, h, g, peak));
      }
      exact = exact_peak_of<false>(peak, rest, &shared_rest);
    }
    c = row_code(peak, exact, p.q_dtype);
    if (threadIdx.x == 0) p.scales[row] = row_scale(peak, rstd, c);
  }
  T* y = p.y != nullptr ? static_cast<T*>(p.y) + row * p.y_ld : nullptr;
  uint8_t* q = p.q != nullptr ? p.q + row * p.q_ld : nullptr;
  for (uint32_t e = threadIdx.x; e < cols; e += kMaxThreads) {
    const float h = h_at(e), g = g_at(e);
    if (q != nullptr) {
      uint8_t o[1];
      codes_of<1>([&](int) { return h * g; }, [&](int) { return h; }, [&](int) { return g; }, c, p.q_dtype, o);
      q[e] = o[0];
    }
    if (y != nullptr) y[e] = from_f<T>(h * rstd * g);
  }
}

// ------------------------------------------------------------------ host side
template <typename T, int VEC, int NV, bool CODES>
int launch_rows(osc_ctx* ctx, const NormArgs& p, int threads) {
  if (threads == 32) {
    const long long blocks = (p.rows + kRowsPerCta - 1) / kRowsPerCta;
    return launch_pdl(ctx, k_rmsnorm<T, VEC, NV, true, CODES>, dim3(static_cast<unsigned>(blocks)),
                      dim3(32 * kRowsPerCta), 0, "k_rmsnorm", p);
  }
  return launch_pdl(ctx, k_rmsnorm<T, VEC, NV, false, CODES>, dim3(static_cast<unsigned>(p.rows)),
                    dim3(static_cast<unsigned>(threads)), 0, "k_rmsnorm", p);
}

template <typename T, bool CODES>
int launch_norm(osc_ctx* ctx, const NormArgs& p, bool vectors) {
  constexpr int VEC = 16 / static_cast<int>(sizeof(T)), NV = 16 / VEC;  // 16 elements a thread
  auto threads_for = [&](int per) { return (p.cols + 32 * per - 1) / (32 * per) * 32; };
  if (p.cols > kMaxThreads * (vectors ? VEC * NV : kSingles))
    return launch_pdl(ctx, k_rmsnorm_long<T>, dim3(static_cast<unsigned>(p.rows)), dim3(kMaxThreads), 0,
                      "k_rmsnorm_long", p);
  if (vectors) {
    // few rows are spread over as many threads as the SMs hold: a vector a thread
    // instead of 16 elements takes 300 x 2048 f32 -> s8 from 5.4 to 4.2 us, 2048 x
    // 1024 bf16 from 5.5 to 5.3, but 1000 x 4096 bf16 -> e4m3 from 11.3 to 12.7
    if (p.rows * threads_for(VEC) <= 2048ll * ctx->num_sms && threads_for(VEC) <= kMaxThreads)
      return launch_rows<T, VEC, 1, CODES>(ctx, p, threads_for(VEC));
    return launch_rows<T, VEC, NV, CODES>(ctx, p, threads_for(VEC * NV));
  }
  if (threads_for(4) <= kMaxThreads) return launch_rows<T, 1, 4, CODES>(ctx, p, threads_for(4));
  return launch_rows<T, 1, kSingles, CODES>(ctx, p, threads_for(kSingles));
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
  const bool codes = q != nullptr;
  switch (dtype) {
    case OSC_F32: return codes ? launch_norm<float, true>(ctx, p, vectors) : launch_norm<float, false>(ctx, p, vectors);
    case OSC_F16: return codes ? launch_norm<__half, true>(ctx, p, vectors) : launch_norm<__half, false>(ctx, p, vectors);
    default: return codes ? launch_norm<__nv_bfloat16, true>(ctx, p, vectors) : launch_norm<__nv_bfloat16, false>(ctx, p, vectors);
  }
}

}  // extern "C"
