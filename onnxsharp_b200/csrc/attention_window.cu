// attention_window.cu — causal attention over a cache with a sliding window and
// a few first tokens that stay visible, 16-bit, grouped heads:
//
//   the query at position p sees the keys j <= p with j > p - window or j < sinks
//   out = softmax(scale * q k^T over the seen keys) v, FP32 inside, rounded once
//
// It stands beside FusedAttention (attention_tf32x3.cu: FP32, every key, an
// additive mask; src/OnnxSharp/Ops/AttentionOps.cs:249-351); the reference has
// no cache, window or grouped heads.
//
// Both kernels below make one pass over the keys with the running maximum and
// sum of the softmax in FP32 registers and split the rows of a key/value head:
// row r of a tile is token r / G, query head r % G of the group (G query heads
// share a key/value head), so a key is read once for the group. A masked score
// is -inf by selection, whatever was computed for it; keys at and behind a
// sequence's length are never used (V rows there are zeroed where a tile
// brings them along: 0 * NaN would not vanish).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "runtime.h"
#include "sm100.cuh"

namespace osc {
namespace {

struct WinArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int* lengths;
  const int* starts;  // null: the queries end at the length
  long long q_b, q_t, q_h, k_b, k_s, k_h, v_b, v_s, v_h, o_b, o_t, o_h;
  int B, T, S, H, HK, G;
  int window, sinks;
  float scale2;       // scale * log2(e): softmax in powers of two
  int tokens;         // tokens of a 128-row tile (k_window_tiles)
  int token_tiles, items;
  int split;          // CTAs that share a row tile's keys (k_window_rows)
  int row_tiles;
};

constexpr int kFarPos = 1 << 30;

// Position of query 0 and the sequence's length, made safe whatever the device
// holds: a start at or behind the length is padding, and so is one below -T.
__device__ __forceinline__ void place_of(const WinArgs& p, int b, int& first, int& len) {
  len = max(0, min(p.lengths[b], p.S));
  first = p.starts != nullptr ? max(-kFarPos, min(p.starts[b], len)) : len - p.T;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two FP32 lanes in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ------------------------------------------------------------------ many rows
// Persistent CTAs walk the row tiles: 128 rows (128 / G consecutive tokens of
// one key/value head's group) against the 128-key tiles that some row sees,
// first those of the sinks, then those of the window. Per key tile ("step")
//   MMA warps      one for S = Q K^T, into one of two S buffers, so the softmax
//                  always has the next scores; one for O += P V, with P from
//                  TMEM and V as it lies, [key][d] (MN-major). (A single warp
//                  spends more cycles in its waits than its products take.)
//   softmax warps  two threads a row, one for the keys 0 .. 63 of every tile, one
//                  for 64 .. 127, each with a running maximum, sum and O of its
//                  own that meet once, at the row tile's end: two warps of an SM
//                  quadrant that need not wait for one another keep the
//                  special-function unit busy through each other's pauses
//   producer warps one for Q and K, one for V, two TMA stages each
// The result goes out by TMA from the Q buffer that it replaces. The
// special-function units bound it: 128 x 128 exponentials are 1024 cycles of an
// SM, as are the two products (16 MMAs of 64).
constexpr int kKeys = 128;
constexpr int kWinThreads = 384;  // Q and K producer, S, V producer, P V; 8 softmax warps
constexpr float kLazy = 8.0f;     // O is rescaled when a maximum has grown by more than 2^8: P stays
                                  // below that, far from overflow in FP16

struct WinBars {
  uint64_t q_full[2], q_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_ready[2], o_full, o_empty;
  uint32_t tmem_slot;
  int abort_flag;
};

template <int D>
struct WinCfg {
  static constexpr int CH = D / 64;                    // 128-byte columns of a row
  static constexpr int TILE = CH * kKeys * 128;        // a [128][D] tile
  static constexpr int BARS = 6 * TILE;                // after two stages of Q, K and V
  static constexpr int EXCHANGE = BARS + 512;          // maximum and sum: [2 halves][128 rows]
  static constexpr int SMEM = 1024 + EXCHANGE + 2 * 128 * 8;
};
static_assert(sizeof(WinBars) <= 512, "barriers fit");

// A row tile: which rows, which key tiles. Every role derives the same from the
// same item number.
struct Item {
  int b, hk, t0;       // sequence, key/value head, first token
  int first, len;      // position of query 0, the sequence's length
  int lo, hi;          // live positions of its rows (none: lo > hi)
  int sink_tiles, lo_tile, n;  // key tiles: sinks', then from lo_tile on; how many
  int plain_lo, plain_hi;      // every row sees every key of the tiles that start in [plain_lo, plain_hi]
  __device__ __forceinline__ int key0(int i) const { return (i < sink_tiles ? i : lo_tile + i - sink_tiles) * kKeys; }
};
__device__ __forceinline__ Item item_at(const WinArgs& p, int x) {
  Item w;
  const int per = p.HK * p.B;
  const int tile = x / per, rest = x - tile * per;
  w.t0 = (p.token_tiles - 1 - tile) * p.tokens;  // late tokens see the most keys of a prompt: they come first
  w.b = rest / p.HK;
  w.hk = rest - w.b * p.HK;
  place_of(p, w.b, w.first, w.len);
  w.lo = max(w.first + w.t0, 0);
  w.hi = min(w.first + min(w.t0 + p.tokens, p.T), w.len) - 1;
  w.sink_tiles = w.lo_tile = w.n = 0;
  if (w.lo <= w.hi) {
    w.lo_tile = (w.lo >= p.window ? w.lo - p.window + 1 : 0) / kKeys;
    w.sink_tiles = min((min(p.sinks, w.hi + 1) + kKeys - 1) / kKeys, w.lo_tile);
    w.n = w.sink_tiles + w.hi / kKeys - w.lo_tile + 1;
  }
  w.plain_lo = w.hi >= p.window ? w.hi - p.window + 1 : 0;
  w.plain_hi = w.lo == w.first + w.t0 ? w.lo - kKeys + 1 : -1;  // (a row before position 0 sees nothing)
  return w;
}
// Some row sees some key of the 64 from h0 on.
__device__ __forceinline__ bool wanted(const WinArgs& p, const Item& w, int h0) {
  return h0 <= w.hi && (h0 + 63 > w.lo - p.window || h0 < p.sinks);
}

// Walks the steps of a CTA's items in order.
struct Steps {
  Item w;
  int x, i;        // item, key tile
  uint32_t item;   // items with keys so far
  uint32_t step;   // steps so far
  bool more;
  __device__ __forceinline__ void seek(const WinArgs& p) {
    more = false;
    for (; x < p.items; x += static_cast<int>(gridDim.x)) {
      w = item_at(p, x);
      if (w.n > 0) {
        more = true;
        break;
      }
    }
  }
  __device__ __forceinline__ void start(const WinArgs& p) {
    x = static_cast<int>(blockIdx.x);
    i = 0;
    item = step = 0;
    seek(p);
  }
  __device__ __forceinline__ void next(const WinArgs& p) {
    ++step;
    if (++i == w.n) {
      i = 0;
      ++item;
      x += static_cast<int>(gridDim.x);
      seek(p);
    }
  }
};

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}
// MN-major 16-bit operand as a 128-byte-swizzled TMA box lays it: rows of 64
// elements along N, 8-row groups of K 1024 bytes apart, 64-column groups `lbo` apart.
__device__ __forceinline__ uint64_t sdesc_mn16(uint32_t saddr, uint32_t lbo) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
         (static_cast<uint64_t>(2u) << 61);
}

// The two warps of 32 rows (named barriers 1 .. 4); all softmax warps (5).
__device__ __forceinline__ void rows_meet(int q) { asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory"); }
__device__ __forceinline__ void softmax_meet() { asm volatile("bar.sync 5, 256;" ::: "memory"); }

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_addr(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// 32 TMEM lanes x 64 columns.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
  uint32_t(&a)[32] = *reinterpret_cast<uint32_t(*)[32]>(r);
  uint32_t(&b)[32] = *reinterpret_cast<uint32_t(*)[32]>(r + 32);
  tmem_ld32(taddr, a);
  tmem_ld32(taddr + 32, b);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kWinThreads, 1)
    k_window_tiles(const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mK,
                   const __grid_constant__ CUtensorMap mV, const __grid_constant__ CUtensorMap mO,
                   const __grid_constant__ WinArgs p, int* __restrict__ err) {
  using Cfg = WinCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sk = smem + 2 * Cfg::TILE;
  uint8_t* sv = smem + 4 * Cfg::TILE;
  WinBars* bar = reinterpret_cast<WinBars*>(smem + Cfg::BARS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->q_full[i], 1);
      mbar_init(&bar->q_empty[i], 1);
      mbar_init(&bar->k_full[i], 1);
      mbar_init(&bar->k_empty[i], 1);
      mbar_init(&bar->v_full[i], 1);
      mbar_init(&bar->v_empty[i], 1);
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_ready[i], 8);
    }
    mbar_init(&bar->o_full, 1);
    mbar_init(&bar->o_empty, 8);
    bar->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch(&mQ);
    tma_prefetch(&mK);
    tma_prefetch(&mV);
  }
  if (warp == 1) {
    tmem_alloc(&bar->tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_slot;
  griddep_launch();
  griddep_wait();

  constexpr uint32_t kFmt = BF16 ? 1u : 0u;
  constexpr uint64_t kStage = Cfg::TILE >> 4;  // in a descriptor's units
  // Producers and MMA warps walk their loops as whole warps; one lane issues.
  auto wait = [&](uint64_t* m, uint32_t parity) {
    const bool ok = mbar_wait(m, parity & 1u, &bar->abort_flag, err);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  if (warp == 0) {
    const uint32_t box = static_cast<uint32_t>(p.tokens * p.G * 128);
    Steps at;
    for (at.start(p); at.more; at.next(p)) {
      if (at.i == 0) {
        const int u = at.item & 1;
        if (!wait(&bar->q_empty[u], (at.item >> 1) ^ 1u)) break;
        if (elect_one()) {
          mbar_arrive_expect_tx(&bar->q_full[u], Cfg::CH * box);
          for (int c = 0; c < Cfg::CH; ++c)
            tma_load_4d(sq + u * Cfg::TILE + c * kKeys * 128, &mQ, &bar->q_full[u], c * 64, at.w.hk * p.G, at.w.t0, at.w.b);
        }
      }
      const int s = at.step & 1;
      if (!wait(&bar->k_empty[s], (at.step >> 1) ^ 1u)) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&bar->k_full[s], Cfg::TILE);
        for (int c = 0; c < Cfg::CH; ++c)
          tma_load_4d(sk + s * Cfg::TILE + c * kKeys * 128, &mK, &bar->k_full[s], c * 64, at.w.key0(at.i), at.w.hk, at.w.b);
      }
    }
  } else if (warp == 2) {
    Steps at;
    for (at.start(p); at.more; at.next(p)) {
      const int s = at.step & 1;
      if (!wait(&bar->v_empty[s], (at.step >> 1) ^ 1u)) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(&bar->v_full[s], Cfg::TILE);
        for (int c = 0; c < Cfg::CH; ++c)
          tma_load_4d(sv + s * Cfg::TILE + c * kKeys * 128, &mV, &bar->v_full[s], c * 64, at.w.key0(at.i), at.w.hk, at.w.b);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (static_cast<uint32_t>(kKeys >> 3) << 17) |
                               (static_cast<uint32_t>(128 >> 4) << 24);
    const uint64_t dq0 = sdesc_kmajor_sw128(smem_addr(sq)), dk0 = sdesc_kmajor_sw128(smem_addr(sk));
    Steps at;
    for (at.start(p); at.more; at.next(p)) {
      const int s = at.step & 1, u = at.item & 1;
      if (at.i == 0 && !wait(&bar->q_full[u], at.item >> 1)) break;
      if (!wait(&bar->k_full[s], at.step >> 1)) break;
      // P of the step before last lies in these columns until its product is done
      if (!wait(&bar->v_empty[s], (at.step >> 1) ^ 1u)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t dq = dq0 + (u != 0 ? kStage : 0), dk = dk0 + (s != 0 ? kStage : 0);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {  // 16 of D: 32 bytes of a 128-byte column
          const uint64_t off = (kk >> 2) * ((kKeys * 128) >> 4) + (kk & 3) * 2;
          mma_f16_ss(tmem + static_cast<uint32_t>(s * kKeys), dq + off, dk + off, idesc, kk != 0 ? 1u : 0u);
        }
        mma_commit(&bar->s_full[s]);
        mma_commit(&bar->k_empty[s]);
      }
    }
  } else if (warp == 3) {
    constexpr uint32_t idesc = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) |
                               (static_cast<uint32_t>(128 >> 4) << 24);
    const uint64_t dv0 = sdesc_mn16(smem_addr(sv), kKeys * 128);
    bool begun[2] = {false, false};  // this item's O of each half has been written
    Steps at;
    for (at.start(p); at.more; at.next(p)) {
      const int s = at.step & 1, j0 = at.w.key0(at.i);
      if (!wait(&bar->v_full[s], at.step >> 1)) break;
      if (j0 + kKeys > at.w.len) {
        // V rows behind the length: whatever the cache holds there must not meet P's zeros
        for (int x = (at.w.len - j0) * 8 + lane; x < kKeys * 8; x += 32)
          for (int c = 0; c < Cfg::CH; ++c)
            *reinterpret_cast<uint4*>(sv + s * Cfg::TILE + c * kKeys * 128 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_async_smem();
        __syncwarp();
      }
      if (at.i == 0) {
        begun[0] = begun[1] = false;
        if (!wait(&bar->o_empty, at.item ^ 1u)) break;
      }
      const bool half[2] = {wanted(p, at.w, j0), wanted(p, at.w, j0 + 64)};
      if (!wait(&bar->p_ready[s], at.step >> 1)) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          if (!half[part]) continue;
          const uint64_t dv = dv0 + (s != 0 ? kStage : 0) + static_cast<uint64_t>(part * (64 * 128 >> 4));
          const uint32_t o_at = tmem + 256u + static_cast<uint32_t>(part * 128);
          const uint32_t p_at = tmem + static_cast<uint32_t>(s * kKeys + part * 64);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 keys: 8 columns of P, two 8-row groups of V
            mma_f16_ts(o_at, p_at + static_cast<uint32_t>(kk * 8), dv + static_cast<uint64_t>(kk * (2048 >> 4)), idesc,
                       begun[part] || kk != 0 ? 1u : 0u);
        }
        mma_commit(&bar->v_empty[s]);
        if (at.i + 1 == at.w.n) mma_commit(&bar->o_full);
      }
      begun[0] = begun[0] || half[0];
      begun[1] = begun[1] || half[1];
    }
  } else if (warp >= 4) {
    const int part = (warp - 4) >> 2, q = warp & 3;
    const int r = q * 32 + lane;  // row of the tile
    const int row_token = r / p.G;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t o_own = lane_base + 256u + static_cast<uint32_t>(part * 128);
    float2* exchange = reinterpret_cast<float2*>(smem + Cfg::EXCHANGE) + r;
    uint32_t item = 0, step = 0;
    bool ok = true;       // after a wait that ran out the meetings go on, over whatever TMEM holds, and nothing is stored
    int unreleased = -1;  // Q buffer that still holds a result on its way out
    auto release = [&]() {  // warp 4, lane by election: the thread that issued the stores
      if (unreleased >= 0 && warp == 4 && elect_one()) {
        bulk_wait_read_all();
        mbar_arrive(&bar->q_empty[unreleased]);
      }
      unreleased = -1;
    };
    for (int x = static_cast<int>(blockIdx.x); x < p.items; x += static_cast<int>(gridDim.x)) {
      const Item w = item_at(p, x);
      const int t = w.t0 + row_token, pos = w.first + t;
      const bool mine = r < p.tokens * p.G && t < p.T;
      const bool live = mine && pos >= 0 && pos < w.len;
      float m = 0.0f, l = 0.0f;
      bool seen = false;     // the row has had a key of this half
      int had = 0;           // steps of this item that wanted this half
      uint32_t s[64];
      bool loaded = false;   // the scores of the step at hand are on their way to s
      for (int i = 0; i < w.n; ++i, ++step) {
        const int j0 = w.key0(i);
        const uint32_t s_at = lane_base + static_cast<uint32_t>((step & 1u) * kKeys + part * 64);
        const bool plain = j0 >= w.plain_lo && j0 <= w.plain_hi;
        // both halves take part in every step: the scores after next wait for both
        if (!loaded) {
          if (ok) ok = wait(&bar->s_full[step & 1u], step >> 1);
          tc_fence_after();
        }
        if (plain || wanted(p, w, j0 + part * 64)) {
          if (!loaded) tmem_ld64(s_at, s);
          loaded = false;
          // The probabilities are taken relative to the maximum so far (0 before a
          // row's first key) while this tile's own is still being found; should that
          // be more than 2^8 above it, or a row's first keys all below it, the
          // maximum moves and the sweep is repeated: S is intact until P is stored.
          uint32_t pk[32];
          float2 sum;
          for (int again = 0; again < 3; ++again) {  // the second sweep passes
            tmem_wait_ld(s);
            if (!plain) {
              // a bit for each key that this row sees: those up to its own position, from the window's start or among the sinks
              auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };  // keys 0 .. n - 1
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int g0 = j0 + part * 64 + h * 32;
                const int to = live ? pos - g0 : -1;
                const int from = pos >= p.window ? pos - p.window + 1 - g0 : 0;
                const uint32_t bits = below(to + 1) & (~below(from) | below(p.sinks - g0));
#pragma unroll
                for (int y = 0; y < 32; ++y)
                  if ((bits & (1u << y)) == 0u) s[h * 32 + y] = 0xff800000u;  // -inf
              }
            }
            const float2 mul = make_float2(p.scale2, p.scale2), off = make_float2(-m, -m);
            float top = -INFINITY;
            sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              const float2 a = make_float2(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1]));
              top = fmaxf(top, fmaxf(a.x, a.y));
              const float2 z = fma2(a, mul, off);
              const float2 e = make_float2(exp2_fast(z.x), exp2_fast(z.y));
              sum = add2(sum, e);
              pk[y] = pack2<BF16>(e.x, e.y);
            }
            const float peak = top * p.scale2;
            const bool low = !seen && peak < m && peak > -INFINITY;
            if (!__any_sync(0xffffffffu, low || peak > m + kLazy)) {
              seen = seen || peak > -INFINITY;
              break;
            }
            const float up = low ? peak : fmaxf(m, peak);
            const float alpha = seen ? exp2_fast(m - up) : 1.0f;  // O is zero before a row's first key
            l *= alpha;
            m = up;
            if (had > 0) {
              // O is at rest once the last step's product is done: this step's waits for P
              const uint32_t last = step - 1u;
              if (ok) ok = wait(&bar->v_empty[last & 1u], last >> 1);
              tc_fence_after();
#pragma unroll
              for (int g = 0; g < D / 32; ++g) {
                uint32_t o[32];
                tmem_ld32(o_own + g * 32, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
                tmem_st32(o_own + g * 32, o);
              }
            }
            tmem_ld64(s_at, s);
          }
          l += sum.x + sum.y;
          tmem_st32(s_at, pk);
          ++had;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->p_ready[step & 1u]);
        if (i == 0) release();
      }
      // the row tile is done: join the halves, through the Q buffer, out
      if (w.n > 0) {
        exchange[part * 128] = make_float2(had > 0 ? m : -INFINITY, l);
        rows_meet(q);
        const float2 his = exchange[(part ^ 1) * 128];
        if (ok) ok = wait(&bar->o_full, item);
        tc_fence_after();
        // weights of the halves' O; a half without a key has l = 0
        const float top = l > 0.0f ? (his.y > 0.0f ? fmaxf(m, his.x) : m) : his.x;
        const float mine_w = l > 0.0f ? exp2_fast(m - top) : 0.0f, his_w = his.y > 0.0f ? exp2_fast(his.x - top) : 0.0f;
        const float total = l * mine_w + his.y * his_w;
        const float inv = live && total > 0.0f ? 1.0f / total : 0.0f;
        const float f_mine = mine_w * inv, f_his = his_w * inv;
        const uint32_t o_his = lane_base + 256u + static_cast<uint32_t>((part ^ 1) * 128);
        uint8_t* stage = sq + (item & 1u) * Cfg::TILE;
#pragma unroll
        for (int g = 0; g < D / 32; ++g) {
          const int c0 = part * (D / 2) + g * 16;  // this thread's columns of the result
          uint32_t a[16], c[16];
          tmem_ld16(o_own + static_cast<uint32_t>(c0), a);
          tmem_ld16(o_his + static_cast<uint32_t>(c0), c);
          tmem_wait_ld(a);
          tmem_wait_ld(c);
          float o[16];
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            // selected, not multiplied away: a half without a product was never written
            const float own = f_mine > 0.0f ? __uint_as_float(a[y]) * f_mine : 0.0f;
            o[y] = f_his > 0.0f ? fmaf(__uint_as_float(c[y]), f_his, own) : own;
          }
          const int col = (c0 >> 6) * kKeys * 128, chunk0 = (c0 & 63) >> 3;
#pragma unroll
          for (int y = 0; y < 16; y += 8)
            *reinterpret_cast<uint4*>(stage + col + r * 128 + (((chunk0 + (y >> 3)) ^ (r & 7)) << 4)) =
                make_uint4(pack2<BF16>(o[y], o[y + 1]), pack2<BF16>(o[y + 2], o[y + 3]), pack2<BF16>(o[y + 4], o[y + 5]),
                           pack2<BF16>(o[y + 6], o[y + 7]));
        }
        tc_fence_before();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->o_empty);
        release();  // (an item of one step that this half did not want)
        softmax_meet();
        if (warp == 4 && elect_one()) {
          if (ok)
            for (int c = 0; c < Cfg::CH; ++c)
              tma_store_4d(&mO, stage + c * kKeys * 128, c * 64, w.hk * p.G, w.t0, w.b);
          bulk_commit();
        }
        unreleased = static_cast<int>(item & 1u);
        ++item;
      } else if (mine) {  // padding alone
        uint16_t* dst = static_cast<uint16_t*>(p.out) + w.b * p.o_b + static_cast<long long>(t) * p.o_t +
                        (w.hk * p.G + r % p.G) * p.o_h + part * (D / 2);
        for (int y = 0; y < D / 2; y += 8) *reinterpret_cast<uint4*>(dst + y) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    if (warp == 4 && elect_one()) bulk_wait_all();
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (threadIdx.x == 0 && bar->abort_flag) {  // copies in flight land before the CTA leaves
    const uint64_t c0 = globaltimer_ns();
    while (globaltimer_ns() - c0 < 50ull * 1000ull * 1000ull) {
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ few rows
// A decode step: 16 rows (tokens x grouped heads) against a long cache, bound
// by the cache's bytes. The seen keys of the row tile are numbered through
// (sinks, then the window), cut into runs for the CTAs of a cluster and walked
// in tiles of 64 by cp.async; each of four warps takes 16 keys of a tile with
// its own running maximum, sum and O (mma.sync m16n8k16: at 16 rows the tensor
// rate is not the limit, and the 128-row tcgen05 tile would be seven eighths
// empty). Warps, then CTAs, are joined in a fixed order, through shared memory
// and the cluster's shared memory: no workspace, the same bits every run.
constexpr int kRowKeys = 64, kRowStages = 3, kRowThreads = 128;

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes; valid == false writes zeros without reading src.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ld_cluster_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int D>
struct RowCfg {
  static constexpr int TILE = kRowKeys * D * 2;
  static constexpr int SMEM = kRowStages * 2 * TILE;
  // after the last tile the ring holds the warps' O [4][16][D], the CTA's O [16][D], maxima and sums
  static constexpr int OFF_CTA = 4 * 16 * D * 4, OFF_M = OFF_CTA + 16 * D * 4, OFF_L = OFF_M + 4 * 16 * 4,
                       OFF_CM = OFF_L + 4 * 16 * 4, OFF_CL = OFF_CM + 64;
  static_assert(OFF_CL + 64 <= SMEM, "the join fits the ring");
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kRowThreads, 2) k_window_rows(const __grid_constant__ WinArgs p) {
  using Cfg = RowCfg<D>;
  extern __shared__ __align__(1024) uint8_t ring[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.split, rt = static_cast<int>(blockIdx.x) / p.split;
  const int hk = blockIdx.y, b = blockIdx.z;
  griddep_launch();
  griddep_wait();
  int first, len;
  place_of(p, b, first, len);
  const int row0 = rt * 16, nrows = p.T * p.G;
  const int t_lo = row0 / p.G, t_hi = min(row0 + 15, nrows - 1) / p.G;
  const int lo_pos = max(first + t_lo, 0), hi_pos = min(first + t_hi, len - 1);
  auto out_row = [&](int r) {
    return static_cast<uint16_t*>(p.out) + b * p.o_b + static_cast<long long>((row0 + r) / p.G) * p.o_t +
           (hk * p.G + (row0 + r) % p.G) * p.o_h;
  };
  if (lo_pos > hi_pos) {  // padding alone: the same in the whole cluster
    if (rank == 0)
      for (int x = tid; x < 16 * D / 8; x += kRowThreads) {
        const int r = x / (D / 8);
        if (row0 + r < nrows) *reinterpret_cast<uint4*>(out_row(r) + (x % (D / 8)) * 8) = make_uint4(0u, 0u, 0u, 0u);
      }
    return;
  }
  const int lo = lo_pos >= p.window ? lo_pos - p.window + 1 : 0;
  const int nsink = min(p.sinks, lo);
  const int total = nsink + hi_pos - lo + 1;
  const int tiles = (total + kRowKeys - 1) / kRowKeys;
  const int i0 = static_cast<int>(static_cast<long long>(rank) * tiles / p.split);
  const int i1 = static_cast<int>(static_cast<long long>(rank + 1) * tiles / p.split);

  // a thread copies the same 16 bytes of every (128 / CHUNKS)-th row of a tile
  constexpr int CHUNKS = D / 8, ROWS_STEP = kRowThreads / CHUNKS;
  const int ch = tid % CHUNKS, crow = tid / CHUNKS;
  const uint16_t* kbase = static_cast<const uint16_t*>(p.k) + b * p.k_b + hk * p.k_h + ch * 8;
  const uint16_t* vbase = static_cast<const uint16_t*>(p.v) + b * p.v_b + hk * p.v_h + ch * 8;
  const uint32_t ring_at = smem_addr(ring);
  auto fetch = [&](int i) {
    const uint32_t at = ring_at + static_cast<uint32_t>(((i - i0) % kRowStages) * 2 * Cfg::TILE);
#pragma unroll
    for (int x = 0; x < kRowKeys / ROWS_STEP; ++x) {
      const int row = crow + x * ROWS_STEP;
      const int vi = i * kRowKeys + row;
      const bool valid = vi < total;
      const long long j = !valid ? 0 : vi < nsink ? vi : lo + vi - nsink;
      const uint32_t off = static_cast<uint32_t>(row * D * 2 + ((ch ^ (row & 7)) << 4));
      cp_async16(at + off, kbase + j * p.k_s, valid);
      cp_async16(at + Cfg::TILE + off, vbase + j * p.v_s, valid);
    }
  };

  // Q: the A fragments of 16 rows, straight from global memory
  const int ra = lane >> 2, rb = ra + 8;
  uint32_t qf[D / 16][4];
  {
    const bool in_a = row0 + ra < nrows, in_b = row0 + rb < nrows;
    auto q_row = [&](int r) {
      return static_cast<const uint16_t*>(p.q) + b * p.q_b + static_cast<long long>((row0 + r) / p.G) * p.q_t +
             (hk * p.G + (row0 + r) % p.G) * p.q_h + (lane & 3) * 2;
    };
    const uint16_t* qa = q_row(in_a ? ra : 0);
    const uint16_t* qb = q_row(in_b ? rb : 0);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qf[ks][0] = in_a ? *reinterpret_cast<const uint32_t*>(qa + ks * 16) : 0u;
      qf[ks][1] = in_b ? *reinterpret_cast<const uint32_t*>(qb + ks * 16) : 0u;
      qf[ks][2] = in_a ? *reinterpret_cast<const uint32_t*>(qa + ks * 16 + 8) : 0u;
      qf[ks][3] = in_b ? *reinterpret_cast<const uint32_t*>(qb + ks * 16 + 8) : 0u;
    }
  }
  // positions of this thread's two rows; -1 sees nothing
  auto pos_of = [&](int r) {
    const int pos = first + (row0 + r) / p.G;
    return row0 + r < nrows && pos >= 0 && pos < len ? pos : -1;
  };
  const int pos_a = pos_of(ra), pos_b = pos_of(rb);

  float o[D / 8][4];
#pragma unroll
  for (int x = 0; x < D / 8; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[x][e] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

#pragma unroll
  for (int s = 0; s < kRowStages - 1; ++s) {
    if (i0 + s < i1) fetch(i0 + s);
    cp_async_commit();
  }
  for (int i = i0; i < i1; ++i) {
    cp_async_wait<kRowStages - 2>();
    __syncthreads();
    if (i + kRowStages - 1 < i1) fetch(i + kRowStages - 1);
    cp_async_commit();
    const uint32_t at = ring_at + static_cast<uint32_t>(((i - i0) % kRowStages) * 2 * Cfg::TILE);
    float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    {
      const int key = warp * 16 + ((lane >> 4) << 3) + (lane & 7);
      const uint32_t krow = at + static_cast<uint32_t>(key * D * 2);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t kf[4];
        ldmatrix4(kf, krow + static_cast<uint32_t>((((ks * 2 + ((lane >> 3) & 1)) ^ (key & 7)) << 4)));
        mma_16816<BF16>(s[0], qf[ks], kf[0], kf[1]);
        mma_16816<BF16>(s[1], qf[ks], kf[2], kf[3]);
      }
    }
    // c0, c1 belong to row a, c2, c3 to row b
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int vi = i * kRowKeys + warp * 16 + n * 8 + (lane & 3) * 2 + (e & 1);
        const int j = vi < nsink ? vi : lo + vi - nsink;
        const int pos = e < 2 ? pos_a : pos_b;
        const bool seen = vi < total && j <= pos && (pos - j < p.window || j < p.sinks);
        s[n][e] = seen ? s[n][e] * p.scale2 : -INFINITY;
      }
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float next = fmaxf(m[h], top);
      const float base = next == -INFINITY ? 0.0f : next;
      alpha[h] = exp2_fast(m[h] - base);
      m[h] = next;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][2 * h + e] = exp2_fast(s[n][2 * h + e] - base);
          sum += s[n][2 * h + e];
        }
      l[h] = l[h] * alpha[h] + sum;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
      for (int x = 0; x < D / 8; ++x) {
        o[x][0] *= alpha[0];
        o[x][1] *= alpha[0];
        o[x][2] *= alpha[1];
        o[x][3] *= alpha[1];
      }
    }
    const uint32_t pf[4] = {pack2<BF16>(s[0][0], s[0][1]), pack2<BF16>(s[0][2], s[0][3]), pack2<BF16>(s[1][0], s[1][1]),
                            pack2<BF16>(s[1][2], s[1][3])};
    {
      const int key = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
      const uint32_t vrow = at + Cfg::TILE + static_cast<uint32_t>(key * D * 2);
#pragma unroll
      for (int dn = 0; dn < D / 16; ++dn) {
        uint32_t vf[4];
        ldmatrix4_trans(vf, vrow + static_cast<uint32_t>((((dn * 2 + (lane >> 4)) ^ (key & 7)) << 4)));
        mma_16816<BF16>(o[2 * dn], pf, vf[0], vf[1]);
        mma_16816<BF16>(o[2 * dn + 1], pf, vf[2], vf[3]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // join the warps: each leaves its O, maximum and sum in the ring
  float* wo = reinterpret_cast<float*>(ring);
  float* co = reinterpret_cast<float*>(ring + Cfg::OFF_CTA);
  float* wm = reinterpret_cast<float*>(ring + Cfg::OFF_M);
  float* wl = reinterpret_cast<float*>(ring + Cfg::OFF_L);
  float* cm = reinterpret_cast<float*>(ring + Cfg::OFF_CM);
  float* cl = reinterpret_cast<float*>(ring + Cfg::OFF_CL);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = ra + 8 * h;
    if ((lane & 3) == 0) {
      wm[warp * 16 + r] = m[h];
      wl[warp * 16 + r] = l[h];
    }
#pragma unroll
    for (int x = 0; x < D / 8; ++x)
      *reinterpret_cast<float2*>(wo + (warp * 16 + r) * D + x * 8 + (lane & 3) * 2) = make_float2(o[x][2 * h], o[x][2 * h + 1]);
  }
  __syncthreads();
  auto weight = [](float part, float whole) { return part == -INFINITY ? 0.0f : exp2_fast(part - whole); };
  for (int x = tid; x < 16 * D; x += kRowThreads) {
    const int r = x / D;
    const float top = fmaxf(fmaxf(wm[r], wm[16 + r]), fmaxf(wm[32 + r], wm[48 + r]));
    float acc = 0.0f, sum = 0.0f;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float f = weight(wm[y * 16 + r], top);
      acc = fmaf(f, wo[y * 16 * D + x], acc);
      sum = fmaf(f, wl[y * 16 + r], sum);
    }
    co[x] = acc;
    if (x % D == 0) {
      cm[r] = top;
      cl[r] = sum;
    }
  }
  if (p.split > 1) cluster_sync_all();
  else __syncthreads();
  // then the CTAs: CTA `rank` finishes the pairs of columns rank, rank + split, ...
  const uint32_t co_at = smem_addr(co), cm_at = smem_addr(cm), cl_at = smem_addr(cl);
  for (int x = rank * kRowThreads + tid; x < 16 * D / 2; x += p.split * kRowThreads) {
    const int r = x / (D / 2);
    if (row0 + r >= nrows) continue;
    float top = -INFINITY;
    for (int c = 0; c < p.split; ++c) {
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(cm_at + r * 4), "r"(c));
      top = fmaxf(top, ld_cluster_f(at));
    }
    float a0 = 0.0f, a1 = 0.0f, sum = 0.0f;
    for (int c = 0; c < p.split; ++c) {
      uint32_t at_m, at_l, at_o;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_m) : "r"(cm_at + r * 4), "r"(c));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_l) : "r"(cl_at + r * 4), "r"(c));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_o) : "r"(co_at + x * 8), "r"(c));
      const float f = weight(ld_cluster_f(at_m), top);
      sum = fmaf(f, ld_cluster_f(at_l), sum);
      a0 = fmaf(f, ld_cluster_f(at_o), a0);
      a1 = fmaf(f, ld_cluster_f(at_o + 4), a1);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    *reinterpret_cast<uint32_t*>(out_row(r) + (x % (D / 2)) * 2) = pack2<BF16>(a0 * inv, a1 * inv);
  }
  if (p.split > 1) cluster_sync_all();  // a CTA stays until its part has been read
}

// ------------------------------------------------------------------ host side
template <int D, bool BF16>
int launch_tiles(osc_ctx* ctx, const WinArgs& p) {
  using Cfg = WinCfg<D>;
  CUtensorMap mQ, mK, mV, mO;
  const uint32_t box_q[4] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(p.tokens), 1};
  const uint32_t box_k[4] = {64, kKeys, 1, 1};
  const uint64_t one = D * 2;  // a stride for axes of length one
  auto stride = [&](long long elems, int n) { return n > 1 ? static_cast<uint64_t>(elems) * 2 : one; };
  const uint64_t dq[4] = {D, static_cast<uint64_t>(p.H), static_cast<uint64_t>(p.T), static_cast<uint64_t>(p.B)};
  const uint64_t sq[3] = {stride(p.q_h, p.H), stride(p.q_t, p.T), stride(p.q_b, p.B)};
  const uint64_t dk[4] = {D, static_cast<uint64_t>(p.S), static_cast<uint64_t>(p.HK), static_cast<uint64_t>(p.B)};
  const uint64_t sk[3] = {stride(p.k_s, p.S), stride(p.k_h, p.HK), stride(p.k_b, p.B)};
  const uint64_t so[3] = {stride(p.o_h, p.H), stride(p.o_t, p.T), stride(p.o_b, p.B)};
  const uint64_t sv[3] = {stride(p.v_s, p.S), stride(p.v_h, p.HK), stride(p.v_b, p.B)};
  const auto type = CU_TENSOR_MAP_DATA_TYPE_UINT16;
  OSC_TRY(encode_tiled(&mQ, type, 4, p.q, dq, sq, box_q, CU_TENSOR_MAP_SWIZZLE_128B));
  OSC_TRY(encode_tiled(&mK, type, 4, p.k, dk, sk, box_k, CU_TENSOR_MAP_SWIZZLE_128B));
  OSC_TRY(encode_tiled(&mV, type, 4, p.v, dk, sv, box_k, CU_TENSOR_MAP_SWIZZLE_128B));
  OSC_TRY(encode_tiled(&mO, type, 4, p.out, dq, so, box_q, CU_TENSOR_MAP_SWIZZLE_128B));
  OSC_TRY(set_smem_attr(ctx, reinterpret_cast<const void*>(k_window_tiles<D, BF16>), Cfg::SMEM));
  return launch_pdl(ctx, k_window_tiles<D, BF16>, dim3(std::min(p.items, ctx->num_sms)), dim3(kWinThreads), Cfg::SMEM, "k_window_tiles", mQ, mK, mV, mO, p,
                    ctx->d_err);
}

template <int D, bool BF16>
int launch_rows(osc_ctx* ctx, const WinArgs& p) {
  using Cfg = RowCfg<D>;
  OSC_TRY(set_smem_attr(ctx, reinterpret_cast<const void*>(k_window_rows<D, BF16>), Cfg::SMEM));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.row_tiles * p.split), p.HK, p.B);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM;
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_window_rows<D, BF16>, p);
  if (e != cudaSuccess) return cuda_fail(e, "k_window_rows launch");
  return check_launch(ctx, "k_window_rows");
}

template <int D, bool BF16>
int launch(osc_ctx* ctx, WinArgs& p) {
  const long long rows = static_cast<long long>(p.T) * p.G;
  if (rows <= 32) {
    p.row_tiles = static_cast<int>((rows + 15) / 16);
    // CTAs to fill the SMs twice, each with two tiles of keys at least
    const long long keys = std::min<long long>(p.S, static_cast<long long>(p.window) + p.T + p.sinks);
    const long long groups = static_cast<long long>(p.row_tiles) * p.HK * p.B;
    p.split = 1;
    while (p.split < 8 && groups * p.split < 2ll * ctx->num_sms && keys > 2ll * p.split * 2 * kRowKeys) p.split *= 2;
    return launch_rows<D, BF16>(ctx, p);
  }
  p.tokens = 128 / p.G;
  p.token_tiles = (p.T + p.tokens - 1) / p.tokens;
  const long long items = static_cast<long long>(p.token_tiles) * p.HK * p.B;
  if (items >= (1ll << 30)) return fail(OSC_EINVAL, "osc_attention_window: %lld row tiles are too many", items);
  p.items = static_cast<int>(items);
  return launch_tiles<D, BF16>(ctx, p);
}

}  // namespace
}  // namespace osc

using namespace osc;

extern "C" {

OSC_API int osc_attention_window(osc_ctx* ctx, int dtype, const void* q, const long long* q_strides, const void* k,
                                 const long long* k_strides, const void* v, const long long* v_strides,
                                 const int* lengths, const int* starts, int B, int T, int S, int H, int HK, int D,
                                 int window, int sinks, float scale, void* out, const long long* out_strides) {
  if (ctx == nullptr) return fail(OSC_EINVAL, "null context");
  if (dtype != OSC_F16 && dtype != OSC_BF16) return fail(OSC_EINVAL, "osc_attention_window: dtype %d is not f16 or bf16", dtype);
  if (B < 0 || T < 0 || S <= 0 || H <= 0 || HK <= 0 || T > kFarPos || S > kFarPos)
    return fail(OSC_EINVAL, "osc_attention_window: bad shape B %d T %d S %d heads %d / %d", B, T, S, H, HK);
  if (H % HK != 0 || H / HK > 128) return fail(OSC_EINVAL, "osc_attention_window: %d heads over %d key/value heads", H, HK);
  if (D != 64 && D != 128) return fail(OSC_EUNSUPPORTED, "osc_attention_window: head size %d (64 and 128 are built)", D);
  if (window < 1 || sinks < 0) return fail(OSC_EINVAL, "osc_attention_window: window %d, sinks %d", window, sinks);
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(OSC_EINVAL, "osc_attention_window: scale %g", static_cast<double>(scale));
  if (HK > 65535 || B > 65535) return fail(OSC_EINVAL, "osc_attention_window: %d sequences, %d key/value heads: at most 65535", B, HK);
  if (q_strides == nullptr || k_strides == nullptr || v_strides == nullptr || out_strides == nullptr)
    return fail(OSC_EINVAL, "osc_attention_window: null strides");
  if (B == 0 || T == 0) return OSC_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || lengths == nullptr)
    return fail(OSC_EINVAL, "osc_attention_window: null pointer");
  auto fits = [](const void* at, const long long* s, int n0, int n1, int n2) {
    const int n[3] = {n0, n1, n2};
    bool ok = reinterpret_cast<uintptr_t>(at) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (n[i] == 1 || (s[i] >= 0 && s[i] % 8 == 0 && s[i] < (1ll << 39)));
    return ok;
  };
  if (!fits(q, q_strides, B, T, H) || !fits(k, k_strides, B, S, HK) || !fits(v, v_strides, B, S, HK) ||
      !fits(out, out_strides, B, T, H))
    return fail(OSC_EINVAL, "osc_attention_window: head rows must start on 16-byte boundaries (strides in multiples of 8 elements)");
  if (reinterpret_cast<uintptr_t>(lengths) % 4 != 0 || reinterpret_cast<uintptr_t>(starts) % 4 != 0)
    return fail(OSC_EINVAL, "osc_attention_window: a pointer is not aligned to its type");
  OSC_TRY(enter(ctx));
  if (fault_injected("launch")) return fail(OSC_EFAULT_INJECTED, "injected failure (launch)");
  WinArgs p = {};
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lengths = lengths;
  p.starts = starts;
  p.q_b = q_strides[0], p.q_t = q_strides[1], p.q_h = q_strides[2];
  p.k_b = k_strides[0], p.k_s = k_strides[1], p.k_h = k_strides[2];
  p.v_b = v_strides[0], p.v_s = v_strides[1], p.v_h = v_strides[2];
  p.o_b = out_strides[0], p.o_t = out_strides[1], p.o_h = out_strides[2];
  p.B = B;
  p.T = T;
  p.S = S;
  p.H = H;
  p.HK = HK;
  p.G = H / HK;
  p.window = window;
  p.sinks = std::min(sinks, kFarPos);
  p.scale2 = scale * 1.4426950408889634f;
  if (D == 64) return dtype == OSC_BF16 ? launch<64, true>(ctx, p) : launch<64, false>(ctx, p);
  return dtype == OSC_BF16 ? launch<128, true>(ctx, p) : launch<128, false>(ctx, p);
}

}  // extern "C"
