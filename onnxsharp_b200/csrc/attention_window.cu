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
// sequence's length or between the sinks and every row's window are never used
// (V rows there are zeroed where a tile brings them along: 0 * NaN would not
// vanish).
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
  int row_tiles;      // of 16 rows (k_window_rows)
  int teams;          // of HK CTAs, that share all key tiles
  void* parts;        // what they leave of cut groups
};

constexpr int kFarPos = 1 << 30;

// Position of query 0 and the sequence's length, made safe whatever the device
// holds: a start at or behind the length is padding, and so is one below -T.
__device__ __forceinline__ int2 read_place(const WinArgs& p, int b) {
  return make_int2(p.lengths[b], p.starts != nullptr ? p.starts[b] : 0);
}
__device__ __forceinline__ void place_of(const WinArgs& p, int2 read, int& first, int& len) {
  len = max(0, min(read.x, p.S));
  first = p.starts != nullptr ? max(-kFarPos, min(read.y, len)) : len - p.T;
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
// SM, as are the two products (16 MMAs of 64). Two prompts of 4096 (16 heads over
// 4, window 1024): 65.5 us, some 1400 cycles a key tile and 3000 from row tile to
// row tile. (Four more warps that finish row tiles meanwhile, on registers that
// the others give up: 82 us; the softmax then has too few.)
constexpr int kKeys = 128;
constexpr int kWinThreads = 384;  // Q and K producer, S, V producer, P V; 8 softmax warps
constexpr float kLazy = 8.0f;     // O is rescaled when a maximum has grown by more than 2^8 (a published
                                  // refinement of the running softmax): P stays below that, far from
                                  // overflow in FP16

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
  int wlo;             // first key of the window of the lowest
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
  place_of(p, read_place(p, w.b), w.first, w.len);
  w.lo = max(w.first + w.t0, 0);
  w.hi = min(w.first + min(w.t0 + p.tokens, p.T), w.len) - 1;
  w.sink_tiles = w.lo_tile = w.n = 0;
  w.wlo = w.lo >= p.window ? w.lo - p.window + 1 : 0;
  if (w.lo <= w.hi) {
    w.lo_tile = w.wlo / kKeys;
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
      // V rows behind the length and between the sinks and the window: whatever
      // the cache holds there must not meet P's zeros. (Halves that consist of
      // such rows are skipped below: what counts is the rest of the border's half.)
      const int gone0 = max(p.sinks - j0, 0), gone1 = min(at.w.wlo - j0, kKeys), end = at.w.len - j0;
      if (gone0 < gone1 || end < kKeys) {
        auto clear = [&](int from, int to) {
          for (int x = from * 8 + lane; x < to * 8; x += 32)
            for (int c = 0; c < Cfg::CH; ++c)
              *reinterpret_cast<uint4*>(sv + s * Cfg::TILE + c * kKeys * 128 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
        };
        auto half_up = [](int row) { return (row + 63) & ~63; };
        if (gone0 < gone1) {
          clear(gone0, min(gone1, half_up(gone0)));
          clear(max(half_up(gone0), gone1 & ~63), gone1);
        }
        if (end < kKeys) clear(end, half_up(end));
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
      for (int i = 0; i < w.n; ++i, ++step) {
        const int j0 = w.key0(i);
        const uint32_t s_at = lane_base + static_cast<uint32_t>((step & 1u) * kKeys + part * 64);
        const bool plain = j0 >= w.plain_lo && j0 <= w.plain_hi;
        // both halves take part in every step: the scores after next wait for both
        if (ok) ok = wait(&bar->s_full[step & 1u], step >> 1);
        tc_fence_after();
        if (plain || wanted(p, w, j0 + part * 64)) {
          tmem_ld64(s_at, s);
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
              // rounded to the type of V, which its product needs; the sum keeps FP32. Half
              // a step of each probability: the result is 1.3 to 1.4 times as far from 64
              // bits as rounding it alone would leave it (bf16 2.2e-3 for 1.6e-3 in norm)
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
        // weights of the halves' O; a half without a key has l = 0. (Asked by !=, not by
        // >: a NaN among the row's scores has made l NaN and has to come out. A row that
        // is padding may hold one too, and is zeros.)
        const bool mine_has = live && l != 0.0f, his_has = live && his.y != 0.0f;
        const float top = mine_has ? (his_has ? fmaxf(m, his.x) : m) : his.x;
        const float mine_w = mine_has ? exp2_fast(m - top) : 0.0f, his_w = his_has ? exp2_fast(his.x - top) : 0.0f;
        const float inv = 1.0f / (l * mine_w + his.y * his_w);
        const float f_mine = mine_has ? mine_w * inv : 0.0f, f_his = his_has ? his_w * inv : 0.0f;
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
            const float own = f_mine != 0.0f ? __uint_as_float(a[y]) * f_mine : 0.0f;
            o[y] = f_his != 0.0f ? fmaf(__uint_as_float(c[y]), f_his, own) : own;
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
// by the cache's bytes. A producer warp brings the tiles of 64 keys that some row
// sees (sinks', then the window's) by TMA; each of four warps takes 16 keys of a
// tile with its own running maximum, sum and O (mma.sync m16n8k16: at 16 rows
// the tensor rate is not the limit, and the 128-row tcgen05 tile would be seven
// eighths empty). A row tile's work for one key/value head is a "group".
//
// Lengths are known on the device alone and differ, so the tiles of all row
// tiles are laid end to end and every team of CTAs, one per key/value head,
// takes the same number of them, whatever sequence they belong to. (Heads that
// walk the same keys side by side read whole rows of the cache between them.)
// A group that lies in one CTA is finished there; of one that is cut the parts
// go to a workspace of the call and k_window_join adds them up in the order of
// the keys: where the cuts lie depends on lengths and the number of SMs alone,
// so the bits are the same every run. One token of 16 sequences (8 key/value
// heads of 128, 210 MB of cache): 43.4 us, 4.8 TB/s; a cluster of up to 8 CTAs a
// group took 48.3. One of 32768 keys: 32.7 for 57.3.
constexpr int kRowKeys = 64, kRowStages = 3;
constexpr int kRowThreads = 160;  // four warps of keys, the producer

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
// The four warps of keys.
__device__ __forceinline__ void keys_meet() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

struct RowBars {
  uint64_t full[kRowStages], empty[kRowStages];
  int part[kRowThreads / 32];
  int found[2];
  int abort_flag;
};

template <int D>
struct RowCfg {
  static constexpr int CH = D / 64, CHUNK = kRowKeys * 128;  // 128-byte columns of a row
  static constexpr int TILE = CH * CHUNK;
  // behind the ring: O of two warps as fragments, their maxima and sums
  static constexpr int JOIN = kRowStages * 2 * TILE, JOIN_ML = JOIN + 2 * 16 * D * 4;
  static constexpr int BARS = JOIN_ML + 2 * 16 * 8;
  static constexpr int SMEM = BARS + static_cast<int>(sizeof(RowBars));
};

// A row tile of a sequence ("unit": the groups of its key/value heads are alike).
struct Unit {
  int b, row0, first, len;
  int lo, hi;                  // keys that some row sees: [lo, hi] and the sinks
  int sink_tiles, lo_tile, tiles;  // key tiles: sinks', then from lo_tile on; how many
  __device__ __forceinline__ int key0(int i) const {
    return (i < sink_tiles ? i : lo_tile + i - sink_tiles) * kRowKeys;
  }
};
__device__ __forceinline__ Unit unit_of(const WinArgs& p, int x, int2 read) {
  Unit u;
  u.b = x / p.row_tiles;
  u.row0 = (x - u.b * p.row_tiles) * 16;
  place_of(p, read, u.first, u.len);
  const int t_lo = u.row0 / p.G, t_hi = min(u.row0 + 15, p.T * p.G - 1) / p.G;
  const int lo_pos = max(u.first + t_lo, 0);
  u.hi = min(u.first + t_hi, u.len - 1);
  u.lo = lo_pos >= p.window ? lo_pos - p.window + 1 : 0;
  u.lo_tile = u.sink_tiles = u.tiles = 0;
  if (lo_pos <= u.hi) {
    u.lo_tile = u.lo / kRowKeys;
    u.sink_tiles = min((min(p.sinks, u.hi + 1) + kRowKeys - 1) / kRowKeys, u.lo_tile);
    u.tiles = u.sink_tiles + u.hi / kRowKeys - u.lo_tile + 1;
  }
  return u;
}
__device__ __forceinline__ Unit unit_at(const WinArgs& p, int x) { return unit_of(p, x, read_place(p, x / p.row_tiles)); }

// Tiles of all units before this thread's share of them, of the share, and of all.
struct Tally {
  int before, own, all;
  int x0, x1;  // the share
};
template <int THREADS>
__device__ __forceinline__ Tally tally(const WinArgs& p, int* part) {
  const int units = p.B * p.row_tiles, each = (units + THREADS - 1) / THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Tally t;
  t.x0 = min(static_cast<int>(threadIdx.x) * each, units);
  t.x1 = min(t.x0 + each, units);
  t.own = 0;
  for (int x = t.x0; x < t.x1; ++x) t.own += unit_at(p, x).tiles;
  int upto = t.own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) part[warp] = upto;
  __syncthreads();
  t.all = 0;
  t.before = upto - t.own;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) t.before += part[w];
    t.all += part[w];
  }
  return t;
}
// Tiles a team takes; fewer than kMinTiles are not worth a part of their own.
constexpr int kMinTiles = 2;
__device__ __forceinline__ int tiles_each(const WinArgs& p, int all) {
  return max(kMinTiles, (all + p.teams - 1) / p.teams);
}

// Where a CTA's walk stands. The next unit's place is read a unit ahead and not
// touched until then: behind the copies in flight such a load takes microseconds.
struct Walk {
  Unit u;
  int2 after;  // of unit x + 1, as read
  int x, tile;
  __device__ __forceinline__ void at(const WinArgs& p, int units, int unit, int first_tile) {
    x = unit;
    tile = first_tile;
    u = unit_at(p, x);
    after = read_place(p, min(x + 1, units - 1) / p.row_tiles);
  }
  __device__ __forceinline__ void next(const WinArgs& p, int units) {
    if (++tile < u.tiles) return;
    tile = 0;
    do {
      if (++x >= units) {  // past the last tile
        u.tiles = 0;
        return;
      }
      u = unit_of(p, x, after);
      after = read_place(p, min(x + 1, units - 1) / p.row_tiles);
    } while (u.tiles == 0);
  }
};

template <int D, bool BF16>
__device__ __forceinline__ uint16_t* out_row(const WinArgs& p, const Unit& u, int hk, int r) {
  return static_cast<uint16_t*>(p.out) + u.b * p.o_b + static_cast<long long>((u.row0 + r) / p.G) * p.o_t +
         (hk * p.G + (u.row0 + r) % p.G) * p.o_h;
}

// Parts of cut groups: CTA c leaves the group that it entered in the middle in
// slot 2 c, the one that it began and left unfinished in slot 2 c + 1. The team
// that begins a row tile says which teams have it: from span.x to span.y.
template <int D>
struct Parts {
  float* o;     // [slots][16][D]
  float2* ml;   // [slots][16]
  int2* span;   // [units]
  __device__ __forceinline__ Parts(const WinArgs& p)
      : o(static_cast<float*>(p.parts)),
        ml(reinterpret_cast<float2*>(o + 2ll * p.teams * p.HK * 16 * D)),
        span(reinterpret_cast<int2*>(ml + 2ll * p.teams * p.HK * 16)) {}
  static size_t bytes(int ctas, int units) { return 2ull * ctas * 16 * (D * 4 + 8) + 8ull * units; }
};

// CUT: the tiles of all units, evenly over p.teams teams; else a CTA a group.
template <int D, bool BF16, bool CUT>
__global__ void __launch_bounds__(kRowThreads, 2)
    k_window_rows(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV,
                  const __grid_constant__ WinArgs p, int* __restrict__ err) {
  using Cfg = RowCfg<D>;
  extern __shared__ __align__(1024) uint8_t ring[];
  RowBars* bar = reinterpret_cast<RowBars*>(ring + Cfg::BARS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int units = p.B * p.row_tiles, nrows = p.T * p.G;
  const int team = static_cast<int>(blockIdx.x / p.HK), hk = static_cast<int>(blockIdx.x - team * p.HK);
  if (tid == 0) {
    for (int i = 0; i < kRowStages; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 4);
    }
    bar->abort_flag = 0;
    fence_mbar_init();
    tma_prefetch(&mK);
    tma_prefetch(&mV);
  }
  __syncthreads();
  griddep_launch();
  griddep_wait();
  auto clear = [&](const Unit& u) {  // a group that is padding alone
    for (int y = tid; y < 16 * D / 8; y += kRowThreads) {
      const int r = y / (D / 8);
      if (u.row0 + r < nrows)
        *reinterpret_cast<uint4*>(out_row<D, BF16>(p, u, hk, r) + (y % (D / 8)) * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
  };
  Walk at;
  int left, each = 0;
  if constexpr (CUT) {
    const Tally t = tally<kRowThreads>(p, bar->part);
    each = tiles_each(p, t.all);
    left = min(each, t.all - team * each);
    const int rel = team * each - t.before;
    if (left > 0 && rel >= 0 && rel < t.own) {
      int rest = rel, x = t.x0;
      for (int n = unit_at(p, x).tiles; rest >= n; n = unit_at(p, x).tiles) {
        rest -= n;
        ++x;
      }
      bar->found[0] = x;
      bar->found[1] = rest;
    }
    __syncthreads();
    if (left > 0) at.at(p, units, bar->found[0], bar->found[1]);
  } else {
    at.at(p, units, team, 0);
    left = at.u.tiles;
    if (left == 0) {
      clear(at.u);
      return;
    }
  }

  const uint32_t ring_at = smem_addr(ring);
  bool ok = true;  // after a wait that ran out the meetings go on, over whatever the ring holds, and nothing is stored
  auto wait = [&](uint64_t* m, uint32_t parity) {
    const bool fine = mbar_wait(m, parity & 1u, &bar->abort_flag, err);
    return __all_sync(0xffffffffu, fine) != 0;
  };
  int slot = 0;
  uint32_t turn = 0;  // of the ring
  auto advance = [&]() {
    if (++slot == kRowStages) {
      slot = 0;
      ++turn;
    }
  };
  if (warp == 4) {
    for (; left > 0; --left, at.next(p, units), advance()) {
      if (!wait(&bar->empty[slot], turn ^ 1u)) break;
      if (elect_one()) {
        uint8_t* dst = ring + slot * 2 * Cfg::TILE;
        const int key = at.u.key0(at.tile);
        mbar_arrive_expect_tx(&bar->full[slot], 2 * Cfg::TILE);
        for (int c = 0; c < Cfg::CH; ++c) {
          tma_load_4d(dst + c * Cfg::CHUNK, &mK, &bar->full[slot], c * 64, key, hk, at.u.b);
          tma_load_4d(dst + Cfg::TILE + c * Cfg::CHUNK, &mV, &bar->full[slot], c * 64, key, hk, at.u.b);
        }
      }
    }
    left = 0;
  }

  const int ra = lane >> 2, rb = ra + 8;
  while (left > 0) {
    const Unit u = at.u;
    const int x = at.x, i0 = at.tile, i1 = i0 + min(left, u.tiles - i0);
    // Q: the A fragments of 16 rows, straight from global memory
    uint32_t qf[D / 16][4];
    {
      const bool in_a = u.row0 + ra < nrows, in_b = u.row0 + rb < nrows;
      auto q_row = [&](int r) {
        return static_cast<const uint16_t*>(p.q) + u.b * p.q_b + static_cast<long long>((u.row0 + r) / p.G) * p.q_t +
               (hk * p.G + (u.row0 + r) % p.G) * p.q_h + (lane & 3) * 2;
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
      const int pos = u.first + (u.row0 + r) / p.G;
      return u.row0 + r < nrows && pos >= 0 && pos < u.len ? pos : -1;
    };
    const int pos_a = pos_of(ra), pos_b = pos_of(rb);

    float o[D / 8][4];
#pragma unroll
    for (int x = 0; x < D / 8; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[x][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    // every row of the tile sees every key of the key tiles that start in [plain_lo, plain_hi]
    const int t_lo = u.row0 / p.G;
    const bool all_live = u.first + t_lo >= 0 && u.first + min(u.row0 + 15, nrows - 1) / p.G < u.len;
    const int plain_lo = u.hi >= p.window ? u.hi - p.window + 1 : 0;
    const int plain_hi = all_live ? u.first + t_lo - kRowKeys + 1 : -1;

    for (int i = i0; i < i1; ++i) {
      const int j0 = u.key0(i), key0 = j0 + warp * 16;
      const bool plain = j0 >= plain_lo && j0 <= plain_hi;
      const uint32_t tile = ring_at + static_cast<uint32_t>(slot * 2 * Cfg::TILE);
      if (ok) ok = wait(&bar->full[slot], turn);
      // V rows that no row sees: whatever the cache holds there must not meet P's zeros
      if (!plain && (key0 + 15 > u.hi || (key0 < u.lo && key0 + 15 >= p.sinks))) {
        const int y = lane >> 1, j = key0 + y;
        if (j > u.hi || (j < u.lo && j >= p.sinks)) {
          uint8_t* v = ring + slot * 2 * Cfg::TILE + Cfg::TILE + (warp * 16 + y) * 128 + (lane & 1) * 64;
#pragma unroll
          for (int c = 0; c < Cfg::CH; ++c)
#pragma unroll
            for (int z = 0; z < 4; ++z) *reinterpret_cast<uint4*>(v + c * Cfg::CHUNK + z * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async_smem();
        __syncwarp();
      }
      // (two sums each, of every other 16 of D: half as long a chain of products)
      float s[2][4] = {}, s2[2][4] = {};
      {
        const int key = warp * 16 + ((lane >> 4) << 3) + (lane & 7);
        const uint32_t krow = tile + static_cast<uint32_t>(key * 128);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t kf[4];
          const int c = (ks & 3) * 2 + ((lane >> 3) & 1);
          ldmatrix4(kf, krow + static_cast<uint32_t>((ks >> 2) * Cfg::CHUNK + ((c ^ (key & 7)) << 4)));
          mma_16816<BF16>(ks % 2 == 0 ? s[0] : s2[0], qf[ks], kf[0], kf[1]);
          mma_16816<BF16>(ks % 2 == 0 ? s[1] : s2[1], qf[ks], kf[2], kf[3]);
        }
      }
      // c0, c1 belong to row a, c2, c3 to row b
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = (s[n][e] + s2[n][e]) * p.scale2;
      if (!plain) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = key0 + n * 8 + (lane & 3) * 2 + (e & 1);
            const int pos = e < 2 ? pos_a : pos_b;
            if (!(j <= pos && (pos - j < p.window || j < p.sinks))) s[n][e] = -INFINITY;
          }
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
      const uint32_t pf[4] = {pack2<BF16>(s[0][0], s[0][1]), pack2<BF16>(s[0][2], s[0][3]),
                              pack2<BF16>(s[1][0], s[1][1]), pack2<BF16>(s[1][2], s[1][3])};
      {
        const int key = warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
        const uint32_t vrow = tile + Cfg::TILE + static_cast<uint32_t>(key * 128);
#pragma unroll
        for (int dn = 0; dn < D / 16; ++dn) {
          uint32_t vf[4];
          const int c = (dn & 3) * 2 + (lane >> 4);
          ldmatrix4_trans(vf, vrow + static_cast<uint32_t>((dn >> 2) * Cfg::CHUNK + ((c ^ (key & 7)) << 4)));
          mma_16816<BF16>(o[2 * dn], pf, vf[0], vf[1]);
          mma_16816<BF16>(o[2 * dn + 1], pf, vf[2], vf[3]);
        }
      }
      // every lane's reads of the tile come before the copies that take its place:
      // without the fence the last 16 columns of V were now and then the next tile's
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->empty[slot]);
      advance();
    }

    // join the warps in pairs, 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
#pragma unroll
    for (int half = 2; half > 0; half >>= 1) {
      const int w = warp & (half - 1);
      float4* jo = reinterpret_cast<float4*>(ring + Cfg::JOIN) + w * (16 * D / 4) + lane;
      float2* jml = reinterpret_cast<float2*>(ring + Cfg::JOIN_ML) + w * 16 + ra;
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int x = 0; x < D / 8; ++x) jo[x * 32] = make_float4(o[x][0], o[x][1], o[x][2], o[x][3]);
        if ((lane & 3) == 0) {
          jml[0] = make_float2(m[0], l[0]);
          jml[8] = make_float2(m[1], l[1]);
        }
      }
      keys_meet();
      if (warp < half) {
        float own[2], his[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float2 other = jml[8 * h];
          const float top = fmaxf(m[h], other.x), base = top == -INFINITY ? 0.0f : top;
          own[h] = exp2_fast(m[h] - base);
          his[h] = exp2_fast(other.x - base);
          l[h] = l[h] * own[h] + other.y * his[h];
          m[h] = top;
        }
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          const float4 f = jo[x * 32];
          o[x][0] = o[x][0] * own[0] + f.x * his[0];
          o[x][1] = o[x][1] * own[0] + f.y * his[0];
          o[x][2] = o[x][2] * own[1] + f.z * his[1];
          o[x][3] = o[x][3] * own[1] + f.w * his[1];
        }
      }
      keys_meet();
    }
    if (warp == 0 && ok) {
      const bool whole = !CUT || (i0 == 0 && i1 == u.tiles);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = ra + 8 * h;
        if (u.row0 + r >= nrows) continue;
        if (whole) {
          const float inv = l[h] > 0.0f ? 1.0f / l[h] : 0.0f;
          uint16_t* dst = out_row<D, BF16>(p, u, hk, r) + (lane & 3) * 2;
#pragma unroll
          for (int x = 0; x < D / 8; ++x)
            *reinterpret_cast<uint32_t*>(dst + x * 8) = pack2<BF16>(o[x][2 * h] * inv, o[x][2 * h + 1] * inv);
        } else {
          const Parts<D> parts(p);
          const long long row = (2ll * blockIdx.x + (i0 == 0 ? 1 : 0)) * 16 + r;
#pragma unroll
          for (int x = 0; x < D / 8; ++x)
            *reinterpret_cast<float2*>(parts.o + row * D + x * 8 + (lane & 3) * 2) = make_float2(o[x][2 * h], o[x][2 * h + 1]);
          if ((lane & 3) == 0) parts.ml[row] = make_float2(m[h], l[h]);
        }
      }
    }
    if (CUT && tid == 0 && hk == 0 && i0 == 0)
      Parts<D>(p).span[x] = make_int2(team, team + (u.tiles - i1 + each - 1) / each);
    left -= i1 - i0;
    at.tile = u.tiles - 1;
    at.next(p, units);
  }
  if constexpr (CUT) {  // units without a key are shared out by number
    for (int x = team; x < units; x += p.teams) {
      const Unit u = unit_at(p, x);
      if (u.tiles > 0) continue;
      clear(u);
      if (tid == 0 && hk == 0) Parts<D>(p).span[x] = make_int2(0, 0);
    }
  }
  __syncthreads();
  if (tid == 0 && bar->abort_flag) {  // copies in flight land before the CTA leaves
    const uint64_t c0 = globaltimer_ns();
    while (globaltimer_ns() - c0 < 50ull * 1000ull * 1000ull) {
    }
  }
  __syncthreads();
}

// A CTA a row of a group: adds up the parts of one that was cut, in the order
// of its keys; each of eight warps takes every eighth part.
constexpr int kJoinThreads = 256;
template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) k_window_join(const __grid_constant__ WinArgs p) {
  constexpr int WARPS = kJoinThreads / 32, EACH = D / 32;
  __shared__ float sums[WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int x = static_cast<int>(blockIdx.x / p.HK), hk = static_cast<int>(blockIdx.x - x * p.HK);
  const int r = static_cast<int>(blockIdx.y);
  griddep_launch();
  griddep_wait();
  const Parts<D> parts(p);
  int2 span = parts.span[x];
  span.x = max(0, min(span.x, p.teams - 1));
  span.y = max(span.x, min(span.y, p.teams - 1));  // (in bounds whatever memory holds)
  Unit u;
  u.b = x / p.row_tiles;
  u.row0 = (x - u.b * p.row_tiles) * 16;
  if (span.x == span.y || u.row0 + r >= p.T * p.G) return;  // finished where it was computed
  auto row_of = [&](int c) { return (2ll * (c * p.HK + hk) + (c == span.x ? 1 : 0)) * 16 + r; };
  float top = -INFINITY;
  for (int c = span.x + lane; c <= span.y; c += 32) top = fmaxf(top, parts.ml[row_of(c)].x);
  float part[4][EACH];  // (asked for before the maximum is known)
  auto load = [&](int c0) {
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int c = c0 + y * WARPS;
      if (c <= span.y) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) part[y][e] = parts.o[row_of(c) * D + e * 32 + lane];
      }
    }
  };
  load(span.x + warp);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, acc[EACH];
  for (int c = span.x + lane; c <= span.y; c += 32) {
    const float2 ml = parts.ml[row_of(c)];
    total = fmaf(ml.y, exp2_fast(ml.x - base), total);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll
  for (int e = 0; e < EACH; ++e) acc[e] = 0.0f;
  for (int c0 = span.x + warp; c0 <= span.y; c0 += 4 * WARPS) {
    if (c0 != span.x + warp) load(c0);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int c = c0 + y * WARPS;
      if (c > span.y) break;
      const float f = exp2_fast(parts.ml[row_of(c)].x - base);
#pragma unroll
      for (int e = 0; e < EACH; ++e) acc[e] = fmaf(part[y][e], f, acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) sums[warp][e * 32 + lane] = acc[e];
  __syncthreads();
  if (threadIdx.x < D) {
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += sums[w][threadIdx.x];
    sum *= total > 0.0f ? 1.0f / total : 0.0f;
    uint16_t* dst = out_row<D, BF16>(p, u, hk, r) + threadIdx.x;
    if constexpr (BF16) *reinterpret_cast<__nv_bfloat16*>(dst) = __float2bfloat16_rn(sum);
    else *reinterpret_cast<__half*>(dst) = __float2half_rn(sum);
  }
}

// ------------------------------------------------------------------ host side
uint64_t map_stride(long long elems, int n, int D) {  // axes of length one may have any
  return static_cast<uint64_t>(n > 1 ? elems : D) * 2;
}
template <int D>
int cache_map(CUtensorMap* map, const WinArgs& p, const void* at, long long s_s, long long s_h, long long s_b, int keys) {
  const uint32_t box[4] = {64, static_cast<uint32_t>(keys), 1, 1};
  const uint64_t dims[4] = {D, static_cast<uint64_t>(p.S), static_cast<uint64_t>(p.HK), static_cast<uint64_t>(p.B)};
  const uint64_t strides[3] = {map_stride(s_s, p.S, D), map_stride(s_h, p.HK, D), map_stride(s_b, p.B, D)};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, at, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
template <int D>
int rows_map(CUtensorMap* map, const WinArgs& p, const void* at, long long s_t, long long s_h, long long s_b) {
  const uint32_t box[4] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(p.tokens), 1};
  const uint64_t dims[4] = {D, static_cast<uint64_t>(p.H), static_cast<uint64_t>(p.T), static_cast<uint64_t>(p.B)};
  const uint64_t strides[3] = {map_stride(s_h, p.H, D), map_stride(s_t, p.T, D), map_stride(s_b, p.B, D)};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, at, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, bool BF16>
int launch_tiles(osc_ctx* ctx, const WinArgs& p) {
  using Cfg = WinCfg<D>;
  CUtensorMap mQ, mK, mV, mO;
  OSC_TRY(rows_map<D>(&mQ, p, p.q, p.q_t, p.q_h, p.q_b));
  OSC_TRY(cache_map<D>(&mK, p, p.k, p.k_s, p.k_h, p.k_b, kKeys));
  OSC_TRY(cache_map<D>(&mV, p, p.v, p.v_s, p.v_h, p.v_b, kKeys));
  OSC_TRY(rows_map<D>(&mO, p, p.out, p.o_t, p.o_h, p.o_b));
  OSC_TRY(set_smem_attr(ctx, reinterpret_cast<const void*>(k_window_tiles<D, BF16>), Cfg::SMEM));
  return launch_pdl(ctx, k_window_tiles<D, BF16>, dim3(std::min(p.items, ctx->num_sms)), dim3(kWinThreads), Cfg::SMEM, "k_window_tiles", mQ, mK, mV, mO, p,
                    ctx->d_err);
}

template <int D, bool BF16>
int launch_rows(osc_ctx* ctx, WinArgs& p) {
  using Cfg = RowCfg<D>;
  CUtensorMap mK, mV;
  OSC_TRY(cache_map<D>(&mK, p, p.k, p.k_s, p.k_h, p.k_b, kRowKeys));
  OSC_TRY(cache_map<D>(&mV, p, p.v, p.v_s, p.v_h, p.v_b, kRowKeys));
  const long long groups = static_cast<long long>(p.row_tiles) * p.HK * p.B;
  if (groups >= (1ll << 31)) return fail(OSC_EINVAL, "osc_attention_window: %lld row tiles are too many", groups);
  // the keys that a row tile can see at most
  const long long keys = std::min<long long>(p.S, static_cast<long long>(p.window) + p.T + p.sinks);
  const long long tiles = (keys + kRowKeys - 1) / kRowKeys;
  const int slots = 2 * ctx->num_sms;  // CTAs that run at once
  // Uncut, the call takes a group's time; cut, the CTAs' even share of all tiles,
  // and some 7 us (12 tiles) for the look at the lengths, the cuts and the second
  // kernel. 8 key/value heads of 128, ragged lengths, us uncut and cut: 8 x 512
  // keys 8.8 and 12.1, 8 x 1024 13.7 and 12.7, 16 x 1024 15.0 and 17.7, 8 x 4096
  // 41.1 and 21.8, 24 x 4096 48.6 and 44.2, 40 x 4096 63.9 and 66.9, 72 x 4096
  // 95.6 and 116.1. (Tiles of all groups are counted in 31 bits.)
  const bool cut = groups < slots && groups * tiles < (1ll << 30) && 10 * (tiles - 12) * slots > 11 * tiles * groups;
  if (!cut) {
    const auto kernel = k_window_rows<D, BF16, false>;
    OSC_TRY(set_smem_attr(ctx, reinterpret_cast<const void*>(kernel), Cfg::SMEM));
    return launch_pdl(ctx, kernel, dim3(static_cast<unsigned>(groups)), dim3(kRowThreads), Cfg::SMEM, "k_window_rows",
                      mK, mV, p, ctx->d_err);
  }
  const int units = p.B * p.row_tiles;
  p.teams = static_cast<int>(std::min<long long>(slots / p.HK, (units * tiles + kMinTiles - 1) / kMinTiles));
  const int ctas = p.teams * p.HK;
  OSC_TRY(stream_alloc(ctx, Parts<D>::bytes(ctas, units), &p.parts));
  const auto kernel = k_window_rows<D, BF16, true>;
  int st = set_smem_attr(ctx, reinterpret_cast<const void*>(kernel), Cfg::SMEM);
  if (st == OSC_OK)
    st = launch_pdl(ctx, kernel, dim3(static_cast<unsigned>(ctas)), dim3(kRowThreads), Cfg::SMEM, "k_window_rows", mK, mV,
                    p, ctx->d_err);
  if (st == OSC_OK)
    st = launch_pdl(ctx, k_window_join<D, BF16>, dim3(static_cast<unsigned>(groups), std::min(16, p.T * p.G)),
                    dim3(kJoinThreads), 0, "k_window_join", p);
  const int freed = stream_free(ctx, p.parts);
  return st != OSC_OK ? st : freed;
}

template <int D, bool BF16>
int launch(osc_ctx* ctx, WinArgs& p) {
  const long long rows = static_cast<long long>(p.T) * p.G;
  p.tokens = 128 / p.G;
  p.token_tiles = (p.T + p.tokens - 1) / p.tokens;
  // Up to 16 rows the cache's bytes count alone. From there to 64 k_window_rows
  // takes them once more for every 16 rows, but all SMs share them; k_window_tiles
  // takes them once and walks a row tile's keys one after the other. 32/8 heads of
  // 128, us by rows and by tiles: 1 x 4096 keys, 8 tokens 14.5 and 37.7, 16 tokens
  // 19.3 and 37.6; 4 x 1024, 8 tokens 17.1 and 13.7; 16 x 8192, 5 tokens 55.3 and
  // 44.5; 64 x 1024, 8 tokens 44.6 and 35.0. (64 rows are as far as the two were
  // measured, not where they meet: for one long sequence the rule itself would
  // choose k_window_rows up to some 190 rows of 8192 keys.)
  bool by_rows = rows <= 16;
  if (!by_rows && rows <= 64) {
    const double keys = std::min<double>(p.S, static_cast<double>(p.window) + p.T + p.sinks), sms = ctx->num_sms;
    const double groups = std::ceil(rows / 16.0) * p.HK * p.B;
    const double waves = std::ceil(static_cast<double>(p.token_tiles) * p.HK * p.B / sms);
    by_rows = 12 + 1.5 * groups * std::ceil(keys / kRowKeys) / (2 * sms) < 4 + 1.1 * waves * std::ceil(keys / kKeys);
  }
  if (by_rows) {
    p.row_tiles = static_cast<int>((rows + 15) / 16);
    return launch_rows<D, BF16>(ctx, p);
  }
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
  constexpr float kLog2E = 1.4426950408889634f;
  if (!(scale > 0.0f) || !std::isfinite(scale * kLog2E)) return fail(OSC_EINVAL, "osc_attention_window: scale %g", static_cast<double>(scale));
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
  p.scale2 = scale * kLog2E;
  if (D == 64) return dtype == OSC_BF16 ? launch<64, true>(ctx, p) : launch<64, false>(ctx, p);
  return dtype == OSC_BF16 ? launch<128, true>(ctx, p) : launch<128, false>(ctx, p);
}

}  // extern "C"
