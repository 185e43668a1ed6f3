// linear.cu — the matrix product of a transformer block with everything around
// it in its epilogue, on the sm_100a tensor cores:
//
//   y[i, j] = round(act((sum_t a[i, t] * w[t, j]) * a_scale[i] * w_scale[j] + bias[j]) + residual[i, j])
//
// for bf16, fp16 (kind::f16), e4m3 (kind::f8f6f4, FP32 sums) and s8 (kind::i8,
// exact S32 sums) operands; everything after the sum is FP32 and rounded once.
// It stands beside the FP32 MatMul (gemm_tf32x3.cu) and the per-tensor u8
// DynamicQuantizeMatMul (dqmm_i8.cu) of the reference's operators
// (src/OnnxSharp/Ops/DnnOps.cs:2789-3102, Ops/QuantizedMatMulOps.cs:115-201);
// the reference has no 16-bit product and no residual in a product.
//
// Orientation. The weights are the MMA's 128-row operand and the tokens its N
// side, so a TMEM lane is an output column: the epilogue thread keeps that
// column's scale and bias in registers, and a warp's residual loads and output
// stores of one token are 32 consecutive elements whatever the row pitch or
// alignment of y is. The token side of a tile can be any multiple of 16, which
// is what fits ragged batches and evens out the last wave.
//
// Weights are laid out once as blocks of 128 columns x 128 bytes of K, each
// 16 KB contiguous: one TMA box reads one block as one run of DRAM pages, and
// K tails and ragged last columns are zeros of the copy.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <new>

#include "runtime.h"
#include "sm100.cuh"
#include "vmath.cuh"

struct osc_linear_weights {
  int device = 0;
  int dtype = 0;
  int k = 0, n = 0;
  int num_kb = 0, tiles = 0;  // blocks of 128 bytes of K, blocks of 128 columns
  uint8_t* blocks = nullptr;  // [tiles][num_kb][128][128]
  CUtensorMap map;            // the blocks as rows of 128 bytes, 128 of them a box
};

namespace osc {
namespace {

enum : int { LIN_F16 = 0, LIN_F8 = 1, LIN_I8 = 2 };  // MMA kinds

constexpr int kCols = 128;               // output columns of a CTA
constexpr int kKB = 128;                 // bytes of K in a block: one swizzle row
constexpr int kWBytes = kCols * kKB;     // 16 KB
constexpr int kMaxStages = 8;
constexpr int kBlocks = 2;               // k-blocks of a ring stage: one would wait, elect and commit for every block
                                         // (8192 x 4096 x 16384 bf16 737 us for 679), three or four leave too few stages
constexpr int kTileEpi = 16;             // epilogue warps of k_linear_tiles
constexpr int kSplitEpi = 4;             // of k_linear_split: several CTAs share an SM
constexpr int kSmemTail = 512;           // barriers
constexpr int kSmemOne = 232448 - 1024;  // one CTA per SM: the ring and the tail
constexpr int kSmemSm = 233472;          // of an SM, 1 KB of every CTA's the system's
constexpr int kMaxSplit = 8;             // portable cluster size

struct LinArgs {
  int M, N, num_kb, last_steps;  // last_steps: 32-byte K steps of the last block
  int bn;                        // tokens of a tile
  int stages, stage_bytes;
  int tiles_m, tiles_n;          // token tiles, column tiles (of 256 for a CTA pair)
  int split;                     // CTAs that share a tile's K
  uint32_t idesc;
  const float* a_scale;
  const float* w_scale;
  int w_scale_n;
  const float* bias;
  int act;
  int out;                       // osc_dtype of y and the residual
  const void* residual;
  long long ldr_bytes;
  void* y;
  long long ldy_bytes;
};

struct LinBars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t exit_bar;
  uint32_t tmem_slot;
  int abort_flag;
  int no_abort;
};
static_assert(sizeof(LinBars) <= kSmemTail, "barriers fit the tail");

// Where a walk around the ring stands: counted along, since a division by the
// number of stages per k-block (some 150 dependent cycles) held every k-block
// up to 920 cycles, whatever its tile.
struct RingPos {
  int s = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) {
      s = 0;
      phase ^= 1u;
    }
  }
};

template <int KIND>
__device__ __forceinline__ void mma_one(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  if constexpr (KIND == LIN_F16) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
  } else if constexpr (KIND == LIN_F8) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
  } else {
    mma_i8(d, da, db, idesc, acc);
  }
}

template <int KIND>
__device__ __forceinline__ void mma_two(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  if constexpr (KIND == LIN_F16) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
  } else if constexpr (KIND == LIN_F8) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
  }
}

// ------------------------------------------------------------------ epilogue
// An accumulator word as the FP32 sum (S32 sums are rounded once, to FP32).
template <int KIND>
__device__ __forceinline__ float sum_of(uint32_t r) {
  return KIND == LIN_I8 ? static_cast<float>(static_cast<int32_t>(r)) : __uint_as_float(r);
}

// Phi(v). (1 + erf(v / sqrt 2)) / 2 cancels for negative v: at -5 a tenth of it
// is gone. Here the tail Q(a) = Phi(-a), a = |v|, is computed as itself: the
// Gaussian times t P(1 - t) with t = 1 / (1 + 0.26 a), the form of Hastings
// ("Approximations for Digital Computers", 1955); P has degree 8, fitted for the
// least relative error over a <= 14 (Lawson's weighted least squares, 2.5e-8).
// 1 - t is taken as 0.26 a t, which is exact enough where a is small. In FP32 Q
// is good to (4 + a^2) 2^-23 relative, the square's rounding in the exponent the
// most of it, before the errors of ex2.approx (2^-22) and rcp.approx (2^-23).
// Behind a = 13 it is below FP32's range and comes out as 0. 4096 x 512 x 2048 s8 to
// f32 with GELU: 20.5 us, with erff 21.9 (without an activation 14.4); erfcf, which
// does not cancel either, makes every k_linear_tiles spill registers.
__device__ __forceinline__ float normal_cdf(float v) {
  const float a = fminf(fabsf(v), 16.0f), ca = 0.26f * a;
  float t, gauss;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(1.0f + ca));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(gauss) : "f"(a * a * -0.72134752f));  // exp(-a^2 / 2)
  const float s = ca * t;
  float p = 0.0305047967f;
  p = fmaf(p, s, -0.0912099406f);
  p = fmaf(p, s, 0.0358258262f);
  p = fmaf(p, s, 0.143133357f);
  p = fmaf(p, s, -0.035094697f);
  p = fmaf(p, s, -0.574419916f);
  p = fmaf(p, s, 1.12941158f);
  p = fmaf(p, s, -1.034392f);
  p = fmaf(p, s, 0.5f);
  const float q = gauss * (t * p);
  return v < 0.0f ? q : 1.0f - q;
}

// The other curves come from the hardware ex2 / rcp instructions (relative
// error under 1e-6 where the sigmoid is not saturated, see fast_sigmoid), two
// orders below the rounding of a 16-bit output and below an FP32 product's own.
template <int NV>
__device__ __forceinline__ void activate(float (&v)[NV], int act) {
  switch (act) {
    case OSC_ACT_SILU:
#pragma unroll
      for (int t = 0; t < NV; ++t) v[t] = act_fast<ACT_SILU>(v[t]);
      break;
    case OSC_ACT_RELU:
#pragma unroll
      for (int t = 0; t < NV; ++t) v[t] = v[t] < 0.0f ? 0.0f : v[t];  // keeps a NaN
      break;
    case OSC_ACT_SIGMOID:
#pragma unroll
      for (int t = 0; t < NV; ++t) v[t] = fast_sigmoid(v[t]);
      break;
    case OSC_ACT_GELU:  // v * Phi(v)
#pragma unroll
      for (int t = 0; t < NV; ++t) v[t] *= normal_cdf(v[t]);
      break;
    case OSC_ACT_GELU_TANH:  // 0.5 * (1 + tanh(u)) = sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3)
#pragma unroll
      for (int t = 0; t < NV; ++t)
        v[t] *= fast_sigmoid(1.5957691216057308f * (v[t] + 0.044715f * v[t] * v[t] * v[t]));
      break;
    default: break;
  }
}

// Raw words of column j (already in `base`) at tokens i0, i0 + step, ...: those below i_end.
template <typename T, int NV>
__device__ __forceinline__ void load_words(const char* base, long long pitch, int i0, int step, int i_end,
                                           uint32_t (&r)[NV]) {
  const char* at = base + i0 * pitch;
  const long long by = step * pitch;
  if (i0 + (NV - 1) * step < i_end) {
#pragma unroll
    for (int t = 0; t < NV; ++t) r[t] = *reinterpret_cast<const T*>(at + t * by);
  } else {
#pragma unroll
    for (int t = 0; t < NV; ++t) r[t] = i0 + t * step < i_end ? *reinterpret_cast<const T*>(at + t * by) : T(0);
  }
}
template <typename T, int NV>
__device__ __forceinline__ void store_words(char* base, long long pitch, int i0, int step, int i_end,
                                            const uint32_t (&r)[NV]) {
  char* at = base + i0 * pitch;
  const long long by = step * pitch;
  if (i0 + (NV - 1) * step < i_end) {
#pragma unroll
    for (int t = 0; t < NV; ++t) *reinterpret_cast<T*>(at + t * by) = static_cast<T>(r[t]);
  } else {
#pragma unroll
    for (int t = 0; t < NV; ++t)
      if (i0 + t * step < i_end) *reinterpret_cast<T*>(at + t * by) = static_cast<T>(r[t]);
  }
}

// What an epilogue thread keeps of its column.
struct Column {
  const char* residual;  // null: none
  char* y;
  float scale, bias;
};
__device__ __forceinline__ Column column_of(const LinArgs& p, int j) {
  Column c;
  const bool in = j < p.N;
  const long long off = static_cast<long long>(j) * (p.out == OSC_F32 ? 4 : 2);
  c.residual = p.residual != nullptr ? static_cast<const char*>(p.residual) + off : nullptr;
  c.y = static_cast<char*>(p.y) + off;
  c.scale = p.w_scale == nullptr ? 1.0f : in ? p.w_scale[p.w_scale_n > 1 ? j : 0] : 0.0f;
  c.bias = p.bias != nullptr && in ? p.bias[j] : 0.0f;
  return c;
}

template <int NV>
__device__ __forceinline__ void load_residual(const LinArgs& p, const Column& c, int i0, int step, int i_end,
                                              uint32_t (&r)[NV]) {
  if (c.residual == nullptr) return;
  if (p.out == OSC_F32) load_words<uint32_t, NV>(c.residual, p.ldr_bytes, i0, step, i_end, r);
  else load_words<uint16_t, NV>(c.residual, p.ldr_bytes, i0, step, i_end, r);
}

// Scale (as[t] * the column's), bias, activation, residual, rounding and the
// stores of tokens i0, i0 + step, ... (those below i_end). The residual's words
// were loaded by the thread that stores, so y may be the residual's own buffer.
template <int NV>
__device__ __forceinline__ void finish(const LinArgs& p, const Column& c, float (&v)[NV], const float (&as)[NV],
                                       uint32_t (&res)[NV], int i0, int step, int i_end) {
  if (p.a_scale != nullptr || p.w_scale != nullptr) {
#pragma unroll
    for (int t = 0; t < NV; ++t) v[t] *= as[t] * c.scale;
  }
  if (p.bias != nullptr) {
#pragma unroll
    for (int t = 0; t < NV; ++t) v[t] += c.bias;
  }
  activate<NV>(v, p.act);
  if (p.out == OSC_F32) {
#pragma unroll
    for (int t = 0; t < NV; ++t) res[t] = __float_as_uint(c.residual != nullptr ? v[t] + __uint_as_float(res[t]) : v[t]);
    store_words<uint32_t, NV>(c.y, p.ldy_bytes, i0, step, i_end, res);
  } else if (p.out == OSC_BF16) {
#pragma unroll
    for (int t = 0; t < NV; ++t)
      res[t] = __bfloat16_as_ushort(__float2bfloat16_rn(c.residual != nullptr ? v[t] + __uint_as_float(res[t] << 16) : v[t]));
    store_words<uint16_t, NV>(c.y, p.ldy_bytes, i0, step, i_end, res);
  } else {
#pragma unroll
    for (int t = 0; t < NV; ++t)
      res[t] = __half_as_ushort(__float2half_rn(
          c.residual != nullptr ? v[t] + __half2float(__ushort_as_half(static_cast<unsigned short>(res[t]))) : v[t]));
    store_words<uint16_t, NV>(c.y, p.ldy_bytes, i0, step, i_end, res);
  }
}

// One epilogue warp's share of a tile: its 32 columns (TMEM lanes) and every
// PARTS-th group of 16 tokens from group `part` on, the next group's residual
// and row scales in flight while this one is finished. A row scale is loaded by
// one lane and handed round.
template <int KIND, int PARTS>
struct TileShare {
  uint32_t res[16];
  float as;
  __device__ __forceinline__ void fetch(const LinArgs& p, const Column& c, int i0, int i_end, int lane, uint32_t (&r)[16],
                                        float& a) {
    load_residual<16>(p, c, i0, 1, i_end, r);
    a = 1.0f;
    if (p.a_scale != nullptr) a = i0 + (lane & 15) < p.M ? p.a_scale[i0 + (lane & 15)] : 0.0f;
  }
  __device__ __forceinline__ void begin(const LinArgs& p, const Column& c, int part, int m0, int j, int lane) {
    fetch(p, c, m0 + part * 16, j < p.N ? min(p.M, m0 + p.bn) : 0, lane, res, as);
  }
  __device__ __forceinline__ void drain(const LinArgs& p, const Column& c, uint32_t tmem_lane, int part, int m0, int j,
                                        int lane) {
    const int i_end = j < p.N ? min(p.M, m0 + p.bn) : 0;
    for (int g = part; g * 16 < p.bn; g += PARTS) {
      const int i0 = m0 + g * 16;
      if (i0 >= p.M) break;
      uint32_t r[16], next[16];
      float next_as;
      tmem_ld16(tmem_lane + g * 16, r);
      fetch(p, c, i0 + PARTS * 16, i_end, lane, next, next_as);
      tmem_wait_ld(r);
      float v[16], a[16];
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = sum_of<KIND>(r[t]);
      if (KIND != LIN_F16) {
#pragma unroll
        for (int t = 0; t < 16; ++t) a[t] = __shfl_sync(0xffffffffu, as, t);
      }
      finish<16>(p, c, v, a, res, i0, 1, i_end);
#pragma unroll
      for (int t = 0; t < 16; ++t) res[t] = next[t];
      as = next_as;
    }
  }
};

// ------------------------------------------------------------------ rows of A that no TMA box fits
// Rows at any pitch and alignment -> rows of whole 16-byte pieces, 16-byte
// aligned, zeros past k_bytes. A thread puts one piece together from the one or
// two aligned ones that hold it (each holds a byte of the row, so neither lies
// outside the tensor's allocation). 2000 x 2001 bf16 by 2048 columns takes 21 us
// with this copy; loader warps inside the product, which fetched such rows for
// every column tile again, took 95.
__global__ void k_linear_rows(const uint8_t* __restrict__ a, int m, int k_bytes, long long lda_bytes, int pieces,
                              uint8_t* __restrict__ out) {
  griddep_launch();
  griddep_wait();
  const long long total = static_cast<long long>(m) * pieces;
  for (long long x = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; x < total;
       x += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long i = x / pieces;
    const int off = static_cast<int>(x - i * pieces) * 16, valid = min(16, k_bytes - off);
    const uintptr_t at = reinterpret_cast<uintptr_t>(a + i * lda_bytes + off);
    const uint32_t s = static_cast<uint32_t>(at & 15u), q = s >> 2, bits = 8u * (s & 3u);
    const uint4* piece = reinterpret_cast<const uint4*>(at - s);
    const uint4 lo = piece[0];
    const uint4 hi = static_cast<int>(s) + valid > 16 ? piece[1] : make_uint4(0u, 0u, 0u, 0u);
    // the five words from the q-th of the eight on
    const uint32_t x0 = q < 2 ? (q == 0 ? lo.x : lo.y) : (q == 2 ? lo.z : lo.w);
    const uint32_t x1 = q < 2 ? (q == 0 ? lo.y : lo.z) : (q == 2 ? lo.w : hi.x);
    const uint32_t x2 = q < 2 ? (q == 0 ? lo.z : lo.w) : (q == 2 ? hi.x : hi.y);
    const uint32_t x3 = q < 2 ? (q == 0 ? lo.w : hi.x) : (q == 2 ? hi.y : hi.z);
    const uint32_t x4 = q < 2 ? (q == 0 ? hi.x : hi.y) : (q == 2 ? hi.z : hi.w);
    uint32_t o[4] = {__funnelshift_r(x0, x1, bits), __funnelshift_r(x1, x2, bits), __funnelshift_r(x2, x3, bits),
                     __funnelshift_r(x3, x4, bits)};
    if (valid < 16) {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int left = valid - 4 * y;
        o[y] = left >= 4 ? o[y] : left > 0 ? o[y] & ((1u << (8 * left)) - 1u) : 0u;
      }
    }
    *reinterpret_cast<uint4*>(out + x * 16) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// ------------------------------------------------------------------ many tokens
// Persistent CTAs (or CTA pairs, cta_group::2: 256 columns a tile, each CTA
// streams its own 128 columns of weights and half of the tokens) walk the
// tiles, sixteen token tiles by all column tiles at a time so that the tiles in
// flight share operands in L2. Two 256-column TMEM accumulators: the MMA warp
// fills one while the epilogue warps empty the other.
__device__ __forceinline__ void tile_at(const LinArgs& p, int t, int& tm, int& tn) {
  constexpr int kGroup = 16;  // 8192 x 4096 x 16384 bf16, clocks settled: 809 us, with 8 815
  const int per = kGroup * p.tiles_n;
  const int g = t / per, in = t - g * per;
  const int h = min(kGroup, p.tiles_m - g * kGroup);
  tn = in / h;
  tm = g * kGroup + (in - tn * h);
}

template <int KIND, bool PAIR>
__global__ void __launch_bounds__(64 + 32 * kTileEpi, 1)
    k_linear_tiles(const __grid_constant__ CUtensorMap mW, const __grid_constant__ CUtensorMap mA,
                   const __grid_constant__ LinArgs p, int* __restrict__ err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  LinBars* b = reinterpret_cast<LinBars*>(ring + p.stages * p.stage_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int P = PAIR ? 2 : 1;
  const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
  const int first = static_cast<int>(blockIdx.x) / P, walkers = static_cast<int>(gridDim.x) / P;
  const int tiles = p.tiles_m * p.tiles_n;
  const int arows = p.bn / P;  // token rows of this CTA

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&b->full[s], 1);
      mbar_init(&b->empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b->acc_full[i], 1);
      mbar_init(&b->acc_empty[i], P * kTileEpi);
    }
    mbar_init(&b->exit_bar, 1);
    b->abort_flag = 0;
    b->no_abort = 0;
    fence_mbar_init();
    tma_prefetch(&mW);
    tma_prefetch(&mA);
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc_pair(&b->tmem_slot, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&b->tmem_slot, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = b->tmem_slot;
  griddep_launch();

  // The producer and the MMA warp walk their loops as whole warps; one lane issues.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_wait(bar, parity, &b->abort_flag, err);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  if (warp == 0) {
    const uint32_t full0 = PAIR ? mapa_shared(&b->full[0], 0) : 0u;
    RingPos at;
    bool waited = false;
    int pre = 0;  // weight blocks issued before the previous kernel was waited for, not yet joined by their tokens
    bool ok = true;
    auto load_w = [&](int s, int row, int blocks) {
      if (elect_one()) {
        uint8_t* st = ring + s * p.stage_bytes;
        if (rank == 0) mbar_arrive_expect_tx(&b->full[s], P * blocks * (kWBytes + arows * kKB));
        for (int y = 0; y < blocks; ++y) {
          if (PAIR) tma_load_2d_pair(st + y * kWBytes, &mW, full0 + static_cast<uint32_t>(s * 8), 0, row + y * kCols);
          else tma_load_2d(st + y * kWBytes, &mW, &b->full[s], 0, row + y * kCols);
        }
      }
    };
    for (int t = first; t < tiles && ok; t += walkers) {
      int tm, tn;
      tile_at(p, t, tm, tn);
      const int w_row = (tn * P + rank) * p.num_kb * kCols, a_row = tm * p.bn + rank * arows;
      if (!waited) {
        // the weights were laid out before this launch was made: their first
        // blocks travel while the previous kernel on the stream drains
        for (int kb = 0; pre < p.stages && kb < p.num_kb; kb += kBlocks, ++pre)
          load_w(pre, w_row + kb * kCols, min(kBlocks, p.num_kb - kb));
        griddep_wait();
        waited = true;
      }
      for (int kb = 0; kb < p.num_kb; kb += kBlocks, at.next(p.stages)) {
        const int s = at.s, blocks = min(kBlocks, p.num_kb - kb);
        if (pre > 0) {
          --pre;
        } else {
          ok = wait(&b->empty[s], at.phase ^ 1u);
          if (!ok) break;
          load_w(s, w_row + kb * kCols, blocks);
        }
        if (elect_one()) {
          uint8_t* st = ring + s * p.stage_bytes + kBlocks * kWBytes;
          for (int y = 0; y < blocks; ++y) {
            if (PAIR) tma_load_2d_pair(st + y * arows * kKB, &mA, full0 + static_cast<uint32_t>(s * 8), (kb + y) * kKB, a_row);
            else tma_load_2d(st + y * arows * kKB, &mA, &b->full[s], (kb + y) * kKB, a_row);
          }
        }
      }
    }
  } else if (warp == 1) {
    griddep_wait();  // (its limited waits begin with this kernel's own work, not while the previous one runs)
    if (rank == 0) {
      const uint32_t own = PAIR ? mapa_shared(b, 0) : 0u, peer = PAIR ? mapa_shared(b, 1) : 0u;
      auto commit = [&](uint64_t* bar) {
        if (PAIR) {
          const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uint8_t*>(bar) - reinterpret_cast<uint8_t*>(b));
          mma_commit_pair(own + off);
          mma_commit_pair(peer + off);
        } else {
          mma_commit(bar);
        }
      };
      RingPos at;
      int it = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += walkers, ++it) {
        const int buf = it & 1;
        if (!wait(&b->acc_empty[buf], ((it >> 1) & 1u) ^ 1u)) break;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(buf * 256);
        for (int kb = 0; kb < p.num_kb; kb += kBlocks, at.next(p.stages)) {
          const int s = at.s, blocks = min(kBlocks, p.num_kb - kb);
          ok = wait(&b->full[s], at.phase);
          if (!ok) break;
          const uint32_t base = smem_addr(ring + s * p.stage_bytes);
          const uint64_t dw0 = sdesc_kmajor_sw128(base), da0 = sdesc_kmajor_sw128(base + kBlocks * kWBytes);
          if (elect_one()) {
            for (int y = 0; y < blocks; ++y) {
              const uint64_t dw = dw0 + static_cast<uint64_t>(y * (kWBytes >> 4)), da = da0 + static_cast<uint64_t>(y * (arows * kKB >> 4));
              const int steps = kb + y + 1 == p.num_kb ? p.last_steps : 4;
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                if (kk < steps) {
                  const uint64_t off = static_cast<uint64_t>(kk * 2);  // 32 bytes of K
                  if (PAIR) mma_two<KIND>(d, dw + off, da + off, p.idesc, (kb | y | kk) != 0 ? 1u : 0u);
                  else mma_one<KIND>(d, dw + off, da + off, p.idesc, (kb | y | kk) != 0 ? 1u : 0u);
                }
            }
            commit(&b->empty[s]);
            if (kb + kBlocks >= p.num_kb) commit(&b->acc_full[buf]);
          }
        }
      }
    }
  } else {
    const int q = warp & 3, part = (warp - 2) >> 2;
    const uint32_t acce0 = PAIR ? mapa_shared(&b->acc_empty[0], 0) : 0u;
    griddep_wait();
    int it = 0;
    for (int t = first; t < tiles; t += walkers, ++it) {
      int tm, tn;
      tile_at(p, t, tm, tn);
      const int m0 = tm * p.bn;
      const int j = (tn * P + rank) * kCols + q * 32 + lane;
      const Column c = column_of(p, j);
      TileShare<KIND, kTileEpi / 4> share;
      share.begin(p, c, part, m0, j, lane);
      const int buf = it & 1;
      const bool ok = mbar_wait(&b->acc_full[buf], (it >> 1) & 1u, &b->abort_flag, err);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      share.drain(p, c, tmem + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(buf * 256), part, m0, j,
                  lane);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(acce0 + static_cast<uint32_t>(buf * 8));
        else mbar_arrive(&b->acc_empty[buf]);
      }
    }
  }

  // Leave once nothing is in flight: after a wait that ran out the copies get
  // time to land, and a CTA of a pair stays until its peer has finished with it.
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    if (b->abort_flag) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 50ull * 1000ull * 1000ull) {
      }
    }
    if (PAIR) {
      mbar_arrive_cluster(mapa_shared(&b->exit_bar, rank ^ 1));
      mbar_wait(&b->exit_bar, 0, &b->no_abort, err);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem, 512);
    else tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ few tokens
// The weights' bytes bound these products, so every SM has to stream: a
// cluster of `split` CTAs shares a tile of 128 columns, each sums its own run
// of K blocks, and the partial sums meet in the cluster's shared memory, where
// CTA r adds the tokens of its slice in the order of the CTAs (the same result
// on every run; no workspace in global memory). Two CTAs fit an SM.
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int KIND>
__global__ void __launch_bounds__(64 + 32 * kSplitEpi, 2)
    k_linear_split(const __grid_constant__ CUtensorMap mW, const __grid_constant__ CUtensorMap mA,
                   const __grid_constant__ LinArgs p, uint32_t tmem_cols, int* __restrict__ err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  LinBars* b = reinterpret_cast<LinBars*>(ring + p.stages * p.stage_bytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.split;  // CTA of the cluster: clusters are runs of `split` blocks
  const int tile = static_cast<int>(blockIdx.x) / p.split;
  const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
  const int kb0 = static_cast<int>(static_cast<long long>(rank) * p.num_kb / p.split);
  const int kbn = static_cast<int>(static_cast<long long>(rank + 1) * p.num_kb / p.split) - kb0;  // this CTA's k-blocks
  const int m0 = tm * p.bn;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&b->full[s], 1);
      mbar_init(&b->empty[s], 1);
    }
    mbar_init(&b->acc_full[0], 1);
    b->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch(&mW);
    tma_prefetch(&mA);
  }
  if (warp == 1) {
    tmem_alloc(&b->tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = b->tmem_slot;
  griddep_launch();

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_wait(bar, parity, &b->abort_flag, err);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  if (warp == 0) {
    const int w_row = (tn * p.num_kb + kb0) * kCols;
    auto load_w = [&](int s, int kc) {
      if (elect_one()) {
        const int blocks = min(kBlocks, kbn - kc);
        mbar_arrive_expect_tx(&b->full[s], blocks * (kWBytes + p.bn * kKB));
        for (int y = 0; y < blocks; ++y)
          tma_load_2d(ring + s * p.stage_bytes + y * kWBytes, &mW, &b->full[s], 0, w_row + (kc + y) * kCols);
      }
    };
    // the weights were laid out before this launch was made: the first blocks
    // land while the previous kernel on the stream drains
    int pre = 0;
    for (int kc = 0; pre < p.stages && kc < kbn; kc += kBlocks, ++pre) load_w(pre, kc);
    griddep_wait();
    RingPos at;
    for (int kc = 0; kc < kbn; kc += kBlocks, at.next(p.stages)) {
      const int s = at.s;
      if (pre > 0) {
        --pre;
      } else {
        if (!wait(&b->empty[s], at.phase ^ 1u)) break;
        load_w(s, kc);
      }
      if (elect_one())
        for (int y = 0; y < min(kBlocks, kbn - kc); ++y)
          tma_load_2d(ring + s * p.stage_bytes + kBlocks * kWBytes + y * p.bn * kKB, &mA, &b->full[s], (kb0 + kc + y) * kKB, m0);
    }
  } else if (warp == 1) {
    griddep_wait();  // (its limited waits begin with this kernel's own work, not while the previous one runs)
    RingPos at;
    for (int kc = 0; kc < kbn; kc += kBlocks, at.next(p.stages)) {
      const int s = at.s, blocks = min(kBlocks, kbn - kc);
      if (!wait(&b->full[s], at.phase)) break;
      const uint32_t base = smem_addr(ring + s * p.stage_bytes);
      const uint64_t dw0 = sdesc_kmajor_sw128(base), da0 = sdesc_kmajor_sw128(base + kBlocks * kWBytes);
      if (elect_one()) {
        for (int y = 0; y < blocks; ++y) {
          const uint64_t dw = dw0 + static_cast<uint64_t>(y * (kWBytes >> 4)), da = da0 + static_cast<uint64_t>(y * (p.bn * kKB >> 4));
          const int steps = kb0 + kc + y + 1 == p.num_kb ? p.last_steps : 4;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < steps) {
              const uint64_t off = static_cast<uint64_t>(kk * 2);
              mma_one<KIND>(tmem, dw + off, da + off, p.idesc, (kc | y | kk) != 0 ? 1u : 0u);
            }
        }
        mma_commit(&b->empty[s]);
        if (kc + kBlocks >= kbn) mma_commit(&b->acc_full[0]);
      }
    }
  }

  const bool epi = warp >= 2;
  const int q = warp & 3, part = (warp - 2) >> 2;
  constexpr int kParts = kSplitEpi / 4;
  const int col = q * 32 + lane;
  const int j = tn * kCols + col;
  const bool in = j < p.N;
  const int tokens = min(p.bn, p.M - m0);
  Column c = {};
  if (epi) {
    griddep_wait();
    c = column_of(p, j);
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q * 32) << 16);
    if (p.split == 1) {
      TileShare<KIND, kSplitEpi / 4> share;
      share.begin(p, c, part, m0, j, lane);
      const bool ok = mbar_wait(&b->acc_full[0], 0, &b->abort_flag, err);
      if (__all_sync(0xffffffffu, ok)) {
        tc_fence_after();
        share.drain(p, c, lane_base, part, m0, j, lane);
      }
    } else {
      const bool ok = mbar_wait(&b->acc_full[0], 0, &b->abort_flag, err);
      if (__all_sync(0xffffffffu, ok)) {
        // every block of this CTA has been multiplied: the ring is free and
        // takes the partial sums, [token][column]
        tc_fence_after();
        uint32_t* sums = reinterpret_cast<uint32_t*>(ring);
        for (int g = part; g * 16 < tokens; g += kParts) {
          uint32_t r[16];
          tmem_ld16(lane_base + g * 16, r);
          tmem_wait_ld(r);
#pragma unroll
          for (int t = 0; t < 16; ++t) sums[(g * 16 + t) * kCols + col] = r[t];
        }
      }
    }
    tc_fence_before();
  }
  if (p.split > 1) {
    constexpr int U = 4;
    const int slice = (tokens + p.split - 1) / p.split;
    const int lo = rank * slice, hi = min(tokens, lo + slice);
    const int i_end = in ? m0 + hi : 0;
    // what the first tokens need beside the sums travels while the CTAs meet
    uint32_t res[U];
    float as[U];
    auto fetch = [&](int i) {
      load_residual<U>(p, c, m0 + i, kParts, i_end, res);
#pragma unroll
      for (int t = 0; t < U; ++t)
        as[t] = p.a_scale != nullptr && i + kParts * t < hi ? p.a_scale[m0 + i + kParts * t] : 1.0f;
    };
    if (epi) fetch(lo + part);
    __syncwarp();
    cluster_sync_all();
    if (epi) {
      const uint32_t own = smem_addr(ring) + static_cast<uint32_t>(col * 4);
      uint32_t peer[kMaxSplit];
#pragma unroll
      for (int x = 0; x < kMaxSplit; ++x)
        if (x < p.split) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer[x]) : "r"(own), "r"(x));
      for (int i = lo + part; i < hi; i += kParts * U) {
        // every CTA's part is on its way before the first is added
        uint32_t sums[kMaxSplit][U];
#pragma unroll
        for (int x = 0; x < kMaxSplit; ++x)
#pragma unroll
          for (int t = 0; t < U; ++t)
            sums[x][t] = x < p.split && i + kParts * t < hi ? ld_cluster(peer[x] + static_cast<uint32_t>((i + kParts * t) * kCols * 4)) : 0u;
        uint32_t acc[U] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int x = 0; x < kMaxSplit; ++x)
#pragma unroll
          for (int t = 0; t < U; ++t)
            acc[t] = KIND == LIN_I8 ? acc[t] + sums[x][t] : __float_as_uint(__uint_as_float(acc[t]) + __uint_as_float(sums[x][t]));
        float v[U];
#pragma unroll
        for (int t = 0; t < U; ++t) v[t] = sum_of<KIND>(acc[t]);
        finish<U>(p, c, v, as, res, m0 + i, kParts, i_end);
        if (i + kParts * U < hi) fetch(i + kParts * U);
      }
    }
    __syncwarp();
    cluster_sync_all();  // a CTA stays until its partial sums have been read
  }
  __syncwarp();
  __syncthreads();
  if (threadIdx.x == 0 && b->abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 50ull * 1000ull * 1000ull) {
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------ the weights' layout
// [k, n] (or [n, k]) -> [tiles][num_kb][128][128 bytes], zeros past n and k.
// A CTA moves a tile of 32 columns x one block of K through shared memory, so
// both sides run along their contiguous axis.
template <typename T>
__global__ void k_linear_pack(const T* __restrict__ w, int k, int n, int n_major, int num_kb, T* __restrict__ blocks) {
  constexpr int KE = kKB / static_cast<int>(sizeof(T));
  __shared__ T tile[32][KE + 4 / sizeof(T)];
  const int kb = blockIdx.x, c0 = static_cast<int>(blockIdx.y) * 32;
  const int t0 = kb * KE;
  if (n_major) {
    for (int x = threadIdx.x; x < 32 * KE; x += blockDim.x) {
      const int c = x / KE, t = x % KE;
      tile[c][t] = c0 + c < n && t0 + t < k ? w[static_cast<size_t>(c0 + c) * k + t0 + t] : T(0);
    }
  } else {
    for (int x = threadIdx.x; x < 32 * KE; x += blockDim.x) {
      const int c = x % 32, t = x / 32;
      tile[c][t] = c0 + c < n && t0 + t < k ? w[static_cast<size_t>(t0 + t) * n + c0 + c] : T(0);
    }
  }
  __syncthreads();
  T* dst = blocks + ((static_cast<size_t>(c0 / kCols) * num_kb + kb) * kCols + c0 % kCols) * KE;
  for (int x = threadIdx.x; x < 32 * KE; x += blockDim.x) dst[x] = tile[x / KE][x % KE];
}

// ------------------------------------------------------------------ host side
int dtype_bytes(int dtype) {
  switch (dtype) {
    case OSC_F32: return 4;
    case OSC_F16:
    case OSC_BF16: return 2;
    case OSC_S8:
    case OSC_E4M3: return 1;
    default: return 0;
  }
}

struct LinPlan {
  bool split_kernel;
  bool pair;
  int bn, split;
};

int div_up(int a, int b) { return (a + b - 1) / b; }

// Which kernel, tile and split: the least of a cost in microseconds whose
// constants were fitted to 8400 measured launches (m 1 to 4096, nine (n, k) from
// 256 x 256 to 16384 x 1024, bf16 and s8, every tile and split here): its choice
// is 1.8 % from the best of them in the geometric mean and 20 % at worst. Neither
// an FP32 output nor a residual was among them, and the times were bursts: it ranks
// plans and foretells no times (4096 x 512 x 2048 s8 to f32 with residual 12.1 us for
// 20.5, since a tile's last step knows nothing of the bytes it moves; 8192 x 4096 x
// 16384 bf16 437 for 676).
//   k_linear_split: a k-block of a CTA takes its issue and landing latency or its
//     share of what an SM takes in; a split adds the meeting of the cluster.
//   k_linear_tiles: a k-block takes its MMAs and their issue (a pair's tile of the
//     same width half the operand bytes); a tile's epilogue hides behind the next
//     tile's blocks, the last one's does not.
//   Either: no less than the bytes' own time.
struct LinShape {
  int m, n, num_kb, out;  // out: bytes of an element of y
};

LinPlan choose(int num_sms, const LinShape& z) {
  LinPlan best{};
  double best_t = 1e300;
  auto consider = [&](const LinPlan& c, double t) {
    if (t < best_t) {
      best_t = t;
      best = c;
    }
  };
  const int cols = div_up(z.n, kCols);
  const double kbytes = static_cast<double>(z.num_kb) * kKB;
  const double bytes_us = ((z.m + z.n) * kbytes + static_cast<double>(z.m) * z.n * 2 * z.out) / 8.6e6;
  for (int bn = 16; bn <= 128; bn += 16) {
    if (bn > 16 && bn - 16 >= z.m) break;
    for (int split = 1; split <= kMaxSplit && split <= z.num_kb; split *= 2) {
      const double ctas = static_cast<double>(cols) * div_up(z.m, bn) * split;
      const double waves = std::ceil(ctas / (2 * num_sms)), per_sm = ctas > num_sms ? 2 : 1;
      const double mma = 4 * std::max(50.0, bn / 2.0) / 1800;
      const double kb = std::max({0.37, per_sm * (kWBytes + bn * kKB) / 95e3, per_sm * mma});
      consider({true, false, bn, split},
               3.4 + std::max(bytes_us, waves * div_up(z.num_kb, split) * kb + 0.57 * (waves - 1)) + 0.018 * bn +
                   (split > 1 ? 1.7 + 0.02 * bn : 0));
    }
  }
  for (int pair = 0; pair <= 1; ++pair) {
    const int step = pair ? 32 : 16;
    for (int bn = step; bn <= 256; bn += step) {
      if (bn > step && bn - step >= z.m) break;
      const double tiles = static_cast<double>(div_up(cols, pair ? 2 : 1)) * div_up(z.m, bn);
      const double waves = std::ceil(tiles / (num_sms / (pair ? 2 : 1)));
      const double kb = std::max(0.154, pair ? 0.107 + 0.00052 * bn : 0.072 + 0.00093 * bn);
      const double main = z.num_kb * kb, tail = 0.76 + 0.0071 * bn;
      consider({false, pair != 0, bn, 1},
               3.9 + (pair ? 0.6 : 0) + std::max(bytes_us, main + (waves - 1) * std::max(main, tail) + tail));
    }
  }
  return best;
}

template <int KIND>
int launch_tiles(osc_ctx* ctx, const LinPlan& pl, const CUtensorMap& mW, const CUtensorMap& mA,
                 const LinArgs& p) {
  void (*kern)(CUtensorMap, CUtensorMap, LinArgs, int*) =
      pl.pair ? k_linear_tiles<KIND, true> : k_linear_tiles<KIND, false>;
  const int smem = p.stages * p.stage_bytes + kSmemTail + 1024;
  OSC_TRY(set_smem_attr(ctx, reinterpret_cast<const void*>(kern), smem));
  const int per = pl.pair ? 2 : 1;
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>(tiles, ctx->num_sms / per) * per));
  cfg.blockDim = dim3(64 + 32 * kTileEpi);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pl.pair ? 2 : 1;
  prof_begin(ctx);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mW, mA, p, ctx->d_err);
  if (e != cudaSuccess) return cuda_fail(e, "k_linear_tiles launch");
  char name[48] = "k_linear_tiles";  // with the plan where launches are recorded
  if (ctx->prof_pending != nullptr) std::snprintf(name, sizeof(name), "k_linear_tiles %s %d", pl.pair ? "pair" : "single", pl.bn);
  return check_launch(ctx, name);
}

template <int KIND>
int launch_split(osc_ctx* ctx, const CUtensorMap& mW, const CUtensorMap& mA, const LinArgs& p) {
  void (*kern)(CUtensorMap, CUtensorMap, LinArgs, uint32_t, int*) = k_linear_split<KIND>;
  const int smem = p.stages * p.stage_bytes + kSmemTail + 1024;
  OSC_TRY(set_smem_attr(ctx, reinterpret_cast<const void*>(kern), smem));
  uint32_t cols = 32;
  while (cols < static_cast<uint32_t>(p.bn)) cols *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.tiles_m * p.tiles_n * p.split));
  cfg.blockDim = dim3(64 + 32 * kSplitEpi);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.split);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  prof_begin(ctx);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mW, mA, p, cols, ctx->d_err);
  if (e != cudaSuccess) return cuda_fail(e, "k_linear_split launch");
  char name[48] = "k_linear_split";
  if (ctx->prof_pending != nullptr) std::snprintf(name, sizeof(name), "k_linear_split %d %d", p.split, p.bn);
  return check_launch(ctx, name);
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes)) == 0; }

int linear_prepack(osc_ctx* ctx, int dtype, const void* w, int k, int n, int layout, int host,
                   osc_linear_weights** out) {
  const int e = dtype_bytes(dtype);
  const size_t bytes = static_cast<size_t>(k) * n * e;
  auto* d = new (std::nothrow) osc_linear_weights();
  if (d == nullptr) return fail(OSC_ENOMEM, "osc_linear_prepack: out of host memory");
  d->device = ctx->device;
  d->dtype = dtype;
  d->k = k;
  d->n = n;
  d->num_kb = static_cast<int>((static_cast<long long>(k) * e + kKB - 1) / kKB);
  d->tiles = div_up(n, kCols);
  const size_t packed = static_cast<size_t>(d->tiles) * d->num_kb * kWBytes;
  void* staged = nullptr;
  cudaError_t err = cudaMalloc(&d->blocks, packed);
  if (err == cudaSuccess && host) {
    err = cudaMalloc(&staged, bytes);
    if (err == cudaSuccess) err = cudaMemcpyAsync(staged, w, bytes, cudaMemcpyHostToDevice, ctx->stream);
    w = staged;
  }
  int st = OSC_OK;
  if (err != cudaSuccess) {
    cudaGetLastError();
    st = fail(OSC_ENOMEM, "osc_linear_prepack: %s", cudaGetErrorString(err));
  }
  if (st == OSC_OK) {
    const dim3 grid(static_cast<unsigned>(d->num_kb), static_cast<unsigned>(d->tiles * (kCols / 32)));
    prof_begin(ctx);
    if (e == 2)
      k_linear_pack<uint16_t><<<grid, 256, 0, ctx->stream>>>(static_cast<const uint16_t*>(w), k, n, layout, d->num_kb,
                                                            reinterpret_cast<uint16_t*>(d->blocks));
    else
      k_linear_pack<uint8_t><<<grid, 256, 0, ctx->stream>>>(static_cast<const uint8_t*>(w), k, n, layout, d->num_kb,
                                                           d->blocks);
    st = check_launch(ctx, "k_linear_pack");
  }
  if (st == OSC_OK) {
    const uint64_t dims[2] = {kKB, static_cast<uint64_t>(d->tiles) * d->num_kb * kCols};
    const uint64_t pitch[1] = {kKB};
    const uint32_t box[2] = {kKB, kCols};
    st = encode_tiled(&d->map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, d->blocks, dims, pitch, box,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  }
  // the products start on the blocks before the previous kernel on their stream
  // is done, so the blocks are complete before the handle is given out
  const cudaError_t synced = cudaStreamSynchronize(ctx->stream);
  if (st == OSC_OK && synced != cudaSuccess) st = cuda_fail(synced, "osc_linear_prepack");
  cudaFree(staged);
  if (st != OSC_OK) {
    cudaFree(d->blocks);
    delete d;
    return st;
  }
  *out = d;
  return OSC_OK;
}

}  // namespace
}  // namespace osc

using namespace osc;

extern "C" {

OSC_API int osc_linear_prepack(osc_ctx* ctx, int dtype, const void* w, int k, int n, int layout, int host,
                               osc_linear_weights** out) {
  if (out == nullptr) return fail(OSC_EINVAL, "osc_linear_prepack: out is null");
  *out = nullptr;
  if (ctx == nullptr) return fail(OSC_EINVAL, "null context");
  if (dtype != OSC_F16 && dtype != OSC_BF16 && dtype != OSC_S8 && dtype != OSC_E4M3)
    return fail(OSC_EINVAL, "osc_linear_prepack: dtype %d is not f16, bf16, s8 or e4m3", dtype);
  if (w == nullptr || k <= 0 || n <= 0) return fail(OSC_EINVAL, "osc_linear_prepack: bad W [%d, %d]", k, n);
  if (layout != 0 && layout != 1) return fail(OSC_EINVAL, "osc_linear_prepack: layout %d", layout);
  // |s8 * s8| <= 2^14: k products stay inside S32
  if (dtype == OSC_S8 && k >= (1 << 17)) return fail(OSC_EINVAL, "osc_linear_prepack: k %d overflows S32 sums", k);
  // rows of 128 bytes are TMA coordinates (signed 32 bits); the grid's y axis holds groups of 32 columns
  const long long kb = (static_cast<long long>(k) * dtype_bytes(dtype) + kKB - 1) / kKB;
  if (n > 65532 * 32 || (static_cast<long long>(div_up(n, kCols)) + 1) * kb * kCols >= (1ll << 31))
    return fail(OSC_EINVAL, "osc_linear_prepack: W [%d, %d] is too large", k, n);
  if (!aligned(w, dtype_bytes(dtype))) return fail(OSC_EINVAL, "osc_linear_prepack: W is not aligned to its type");
  OSC_TRY(enter(ctx));
  if (capturing(ctx)) return fail(OSC_EINVAL, "osc_linear_prepack: the stream is being captured");
  if (fault_injected("prepack")) return fail(OSC_EFAULT_INJECTED, "injected failure (prepack)");
  return linear_prepack(ctx, dtype, w, k, n, layout, host, out);
}

OSC_API int osc_linear_weights_free(osc_linear_weights* w) {
  if (w == nullptr) return OSC_OK;
  cudaSetDevice(w->device);
  cudaDeviceSynchronize();
  cudaFree(w->blocks);
  delete w;
  return OSC_OK;
}

OSC_API int osc_linear(osc_ctx* ctx, const void* a, int m, long long lda, const osc_linear_weights* w,
                       const float* a_scale, const float* w_scale, int n_scale, const float* bias, int act,
                       const void* residual, long long ldr, int out_dtype, void* y, long long ldy) {
  if (ctx == nullptr) return fail(OSC_EINVAL, "null context");
  if (w == nullptr) return fail(OSC_EINVAL, "osc_linear: null weights");
  if (w->device != ctx->device) return fail(OSC_EINVAL, "osc_linear: weights of device %d on device %d", w->device, ctx->device);
  if (m < 0 || m > (1 << 30)) return fail(OSC_EINVAL, "osc_linear: m = %d", m);
  const bool coded = w->dtype == OSC_S8 || w->dtype == OSC_E4M3;
  if (out_dtype != OSC_F32 && out_dtype != OSC_F16 && out_dtype != OSC_BF16)
    return fail(OSC_EINVAL, "osc_linear: output dtype %d is not f32, f16 or bf16", out_dtype);
  if (act < OSC_ACT_NONE || act > OSC_ACT_GELU_TANH) return fail(OSC_EINVAL, "osc_linear: activation %d", act);
  if (!coded && (a_scale != nullptr || w_scale != nullptr))
    return fail(OSC_EINVAL, "osc_linear: scales belong to 8-bit operands");
  if (w_scale != nullptr && n_scale != 1 && n_scale != w->n)
    return fail(OSC_EINVAL, "osc_linear: %d column scales for %d columns", n_scale, w->n);
  if (lda == 0) lda = w->k;
  if (ldy == 0) ldy = w->n;
  if (ldr == 0) ldr = w->n;
  if (lda < w->k || ldy < w->n || (residual != nullptr && ldr < w->n))
    return fail(OSC_EINVAL, "osc_linear: a row pitch (%lld, %lld, %lld) below the row's length", lda, ldy, ldr);
  if (m == 0) return OSC_OK;
  if (a == nullptr || y == nullptr) return fail(OSC_EINVAL, "osc_linear: null pointer");
  const int e = dtype_bytes(w->dtype), o = dtype_bytes(out_dtype);
  if (!aligned(a, e) || !aligned(y, o) || !aligned(residual, o) || !aligned(a_scale, 4) || !aligned(w_scale, 4) ||
      !aligned(bias, 4))
    return fail(OSC_EINVAL, "osc_linear: a pointer is not aligned to its type");
  OSC_TRY(enter(ctx));
  if (fault_injected("launch")) return fail(OSC_EFAULT_INJECTED, "injected failure (launch)");

  const LinPlan pl = choose(ctx->num_sms, {m, w->n, w->num_kb, o});
  LinArgs p = {};
  p.M = m;
  p.N = w->n;
  p.num_kb = w->num_kb;
  const int k_bytes = w->k * e;
  p.last_steps = div_up(k_bytes - (w->num_kb - 1) * kKB, 32);
  p.bn = pl.bn;
  p.split = pl.split;
  const int arows = pl.pair ? pl.bn / 2 : pl.bn;
  p.stage_bytes = kBlocks * (kWBytes + arows * kKB);
  p.stages = std::min(kMaxStages, ((pl.split_kernel ? kSmemSm / 2 - 2048 : kSmemOne) - kSmemTail) / p.stage_bytes);
  p.tiles_m = div_up(m, pl.bn);
  p.tiles_n = div_up(w->n, pl.pair ? 2 * kCols : kCols);
  if (static_cast<long long>(p.tiles_m) * p.tiles_n * pl.split >= (1ll << 31))
    return fail(OSC_EINVAL, "osc_linear: %d rows are too many", m);
  const uint32_t rows = pl.pair ? 256u : 128u;
  const uint32_t size = (static_cast<uint32_t>(pl.bn >> 3) << 17) | ((rows >> 4) << 24);
  p.a_scale = a_scale;
  p.w_scale = w_scale;
  p.w_scale_n = n_scale;
  p.bias = bias;
  p.act = act;
  p.out = out_dtype;
  p.residual = residual;
  p.ldr_bytes = ldr * o;
  p.y = y;
  p.ldy_bytes = ldy * o;

  switch (w->dtype) {
    case OSC_F16: p.idesc = (1u << 4) | size; break;                           // F16 operands, F32 sums
    case OSC_BF16: p.idesc = (1u << 4) | (1u << 7) | (1u << 10) | size; break;  // BF16
    case OSC_E4M3: p.idesc = (1u << 4) | size; break;                          // E4M3
    default: p.idesc = (2u << 4) | (1u << 7) | (1u << 10) | size; break;       // signed 8-bit operands, S32 sums
  }

  // rows that start on 16-byte boundaries travel by TMA; others are first copied to such
  const bool direct = aligned(a, 16) && (m == 1 || (lda * e) % 16 == 0);
  const int pieces = div_up(k_bytes, 16);
  void* rows_copy = nullptr;
  uint64_t pitch[1] = {m == 1 ? static_cast<uint64_t>(pieces) * 16 : static_cast<uint64_t>(lda) * e};
  int st = OSC_OK;
  if (!direct) {
    const long long total = static_cast<long long>(m) * pieces;
    OSC_TRY(stream_alloc(ctx, static_cast<size_t>(total) * 16, &rows_copy));
    const long long blocks = std::min<long long>((total + 255) / 256, 8ll * ctx->num_sms);
    st = launch_pdl(ctx, k_linear_rows, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, "k_linear_rows",
                    static_cast<const uint8_t*>(a), m, k_bytes, lda * e, pieces, static_cast<uint8_t*>(rows_copy));
    a = rows_copy;
    pitch[0] = static_cast<uint64_t>(pieces) * 16;
  }
  CUtensorMap mA{};
  if (st == OSC_OK) {
    const uint64_t dims[2] = {static_cast<uint64_t>(k_bytes), static_cast<uint64_t>(m)};
    const uint32_t box[2] = {kKB, static_cast<uint32_t>(arows)};
    st = encode_tiled(&mA, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (st == OSC_OK) {
    switch (w->dtype) {
      case OSC_F16:
      case OSC_BF16:
        st = pl.split_kernel ? launch_split<LIN_F16>(ctx, w->map, mA, p) : launch_tiles<LIN_F16>(ctx, pl, w->map, mA, p);
        break;
      case OSC_E4M3:
        st = pl.split_kernel ? launch_split<LIN_F8>(ctx, w->map, mA, p) : launch_tiles<LIN_F8>(ctx, pl, w->map, mA, p);
        break;
      default:
        st = pl.split_kernel ? launch_split<LIN_I8>(ctx, w->map, mA, p) : launch_tiles<LIN_I8>(ctx, pl, w->map, mA, p);
        break;
    }
  }
  if (rows_copy != nullptr) {
    const int freed = stream_free(ctx, rows_copy);
    if (st == OSC_OK) st = freed;
  }
  return st;
}

}  // extern "C"
