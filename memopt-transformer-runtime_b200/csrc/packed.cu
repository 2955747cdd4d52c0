// packed.cu — attention over packed prompts of different lengths, with
// grouped heads, on the 5th-generation tensor cores.
//
// Row i of a sequence of n tokens sees its tokens [max(0, c - W), c), c = i + 1
// (causal) or n; out = softmax(q k^T / sqrt(D)) v over them.
//
// Work item = (sequence, block of tokens, head unit).  A head unit is Gp query
// heads that share a KV head (the largest power of two dividing the group, at
// most 16), and a tile is 128 rows = 128 / Gp tokens x Gp heads: one TMA box of
// the query tensor lays them out token by token, so grouped heads share every
// K and V tile and a short prompt still fills rows.  An item has two tiles of
// consecutive tokens over the same key blocks of 128, one CTA to an SM; or one
// tile, two CTAs to an SM, for short prompts and few items (measured at the rule
// in plan_of).  Few rows with many keys make fewer or longer items than the SMs
// need: items are then split along the keys, each piece writes its unscaled sum with
// its rows' maxima and sums, and a second kernel joins them (join_pieces_kernel).
//
// The launch has a CTA per item at most, long items first.  A CTA that has done
// its item takes over one that has not begun (cluster launch control), so the SMs
// stay balanced: on 2 x 8192 tokens causal, 32 heads, the CTAs end within 2% of
// each other.  Head units go in chunks whose K and V fit L2: all heads at once
// read them from DRAM again for every item (148 heads of 8192 tokens: 4 TB/s and
// 20% slower under the power cap).  Warps of a CTA:
//   * four per tile for the softmax, one thread per row (= TMEM lane);
//   * one per tile issues its tcgen05.mma: S = Q K^T (128 x 128 x D) into its 128
//     score columns, O += P V (128 x D x 128) with P from tensor memory.  One warp
//     for both tiles made each wait of one tile a hole in the other's products
//     (period of a pair of blocks 4280 cycles against 2950);
//   * one loads Q and the K/V blocks by TMA (128-byte swizzle) into a ring;
//   * one finds the next item from cu_seqlens while the others work.
// The tiles take turns on the tensor pipe: while one tile's scores become weights,
// the other's products run.  With D = 128 P (16-bit pairs) overwrites the scores it
// came from, so a block is the chain scores -> maximum -> weights -> P V -> scores;
// P V starts on its first 96 keys while the last 32 weights are being computed
// (starting at 64 or at 128: 15% slower).  With D = 64 tensor memory has room for
// P beside the scores, and the next scores run during the softmax.  O is rescaled
// only when the running maximum grows by more than 2^8 (weights stay <= 2^8 and
// the sums fp32), which is rare.  Weights are rounded to 16 bits for P V, as its A
// operand has to be of V's type; the row sum adds them in fp32.  Against 64 bits a
// result is off by 9 to 38% more than with fp32 weights (fp16 2.1e-4 to 2.9e-4 over
// an output, bf16 2.1e-3; the rounding of the result alone 1.9e-4 and 1.65e-3).
//
// What bounds it: for each tile and block 1024 cycles of the tensor pipe (D = 128)
// and 1024 of the exponential unit, which the two tiles overlap to 2950 cycles a
// pair of blocks (70% of the tensor pipe); in long runs the power cap (1000 W,
// 1.4 GHz).  148 heads x 8192 tokens, not causal: 3.82-3.94 ms = 1290-1330 TFLOP/s,
// 0.92-0.95 of the measured sustained cuBLAS rate; 2 x 8192 causal, 32 heads:
// 1.02-1.08 ms = 1020-1080, of which about an eighth is the ends of its 13.8 items an
// SM (the warps that compute weights also scale and store).  A quarter of the exponentials on the FMA pipe saves 3% of the
// cycles and costs as much power: equal or slower by the clock, not kept.
//
// Masked scores are replaced, so a hidden key never matters.  A hidden value
// meets a weight of exactly 0, which only a non-finite value survives: rows
// behind the sequence's end are zeroed in shared memory, and a row whose result
// is not finite is computed again over its visible tokens alone (row_by_row), so
// a NaN or an infinity reaches exactly the rows that see it.
//
// Every wait is bounded; a wait that runs out ends the CTA with NaN in the rows
// of the item at hand.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include "tc.cuh"

namespace memopt {
namespace packed {

constexpr int kBN = 128;       // keys per block
constexpr int kFirst = 6;       // of the 8 steps of 16 keys, those that P.V starts with
constexpr int kAhead = 3;       // blocks before an item's last loads at which the next item is taken
constexpr int kMaxGp = 16;      // query heads packed into a tile
// Splitting along the keys.  Writing, launching and joining the pieces takes 6-14 us,
// about 6 blocks' time, which the longest walk has to save: one prompt of 4000 tokens,
// 4/1 heads 57 -> 33 us, 8192 of 4 heads 114 -> 87, 16384 of 2 heads 220 -> 150, 1200
// of 4 heads not causal 25 -> 20; below that a split loses (2000 tokens of 16/4 heads,
// 4 blocks: 35.2 -> 35.7, 1000 of 32/8 heads, 1 block: 22 -> 27).
constexpr double kSplitGain = 6;
// What an item takes beside its walk, in key blocks: its ends 1.3 (one tile; 2 with
// two tiles), the rest a CTA's start and the wait for its first loads.
constexpr double kItemBlocks = 4;
constexpr int kMaxPieces = 16;
constexpr int64_t kMaxWorkspace = int64_t(256) << 20;

struct Params {
  const void *q, *k, *v;
  void* out;
  const int32_t* cu;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  int T, S, H, group;
  int gshift;       // log2 of the heads packed into a tile
  int units;        // head units: H >> gshift
  int chunk;        // head units walked together
  int window, causal;
  int zero_rest;    // rows behind the last sequence are written as 0
  float qscale;     // log2(e) / sqrt(D)
  // Split items: key blocks of a piece, most pieces of a tile, and for every tile,
  // head unit and piece the unscaled O [D/4][128 rows] float4 and the rows' (m, l).
  // The first `whole` tiles of a sequence stay whole.
  int split, pieces, whole;
  float4* part_o;
  float2* part_ml;
};

// TILES: 128-row tiles of an item.  Two share the K/V blocks and take turns on the
// tensor pipe, one CTA per SM; with one, two CTAs share the SM.
template <int D, int TILES>
struct Cfg {
  // Warps: 4 for the softmax of each tile, then a warpgroup of MMA warps (one per
  // tile), the load warp and the scheduler.
  static constexpr int MMA_WARP = 4 * TILES, LOAD_WARP = 5 * TILES, SCHED_WARP = LOAD_WARP + 1;
  static constexpr int THREADS = 128 * TILES + 128;
  static constexpr int LAUNCH_REGS = TILES == 2 ? 168 : 128;  // a thread, of 65536 / THREADS / CTAs
  static constexpr int SOFTMAX_REGS = TILES == 2 ? 208 : 184, OTHER_REGS = 72;
  static_assert(128 * TILES * SOFTMAX_REGS + 128 * OTHER_REGS <= THREADS * LAUNCH_REGS, "within the launch's registers");
  static constexpr int ITEM_READERS = 5 * TILES + 1;  // softmax, MMA and load warps
  static constexpr int HALVES = D / 64;
  static constexpr int HALF = kBN * 128;          // 128 rows x 128 B
  static constexpr int TILE = HALVES * HALF;      // a Q tile, a K block or a V block
  static constexpr int STAGES = TILES == 2 ? (D == 128 ? 5 : 8) : (D == 128 ? 2 : 5);
  static constexpr int KV_OFF = TILES * TILE;
  static constexpr int SMEM = KV_OFF + STAGES * TILE + 1024;  // + alignment slack
  // cu_seqlens kept in shared memory up to this many values: read from global
  // memory they cost the scheduler 900 cycles a step beside the loads of K and V.
  static constexpr int CU = TILES == 2 && D == 128 ? 256 : 3000;
  // With D = 64 tensor memory has room for P beside the scores: the next scores
  // are computed while the weights are, and a block takes its softmax alone.
  static constexpr bool OWN_P = kBN + D + kBN / 2 <= 256;
  static_assert(SMEM <= (TILES == 2 ? 227 : 112) * 1024, "shared memory");
  static_assert(kBN + D <= 256, "tensor memory columns of a tile");
};

struct Item {
  int start, n, t0, unit;  // first packed row, length, first token, head unit (n < 0: no more items)
  int piece, slot;         // split items: which piece, and where its partial result goes
};

// Bounded wait: ten seconds by the global timer, read every 4096 polls.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t began = 0;
  for (uint32_t polls = 1;; ++polls) {
    if (mbar_try_wait_hint(bar, parity, 1000)) return true;
    if ((polls & 4095u) == 0) {
      uint64_t now;
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
      if (began == 0) began = now;
      else if (now - began > 10000000000ull) return false;
    }
  }
}

// Key blocks [lo, hi) of an item's tile.
struct Range {
  int lo, hi;
  int last;  // keys below this index are the tile's (visible to some row)
};
template <int TILES>
__device__ __forceinline__ Range tile_range(const Params& p, const Item& it, int t) {
  const int tokens = 128 >> p.gshift;
  const int first = it.t0 + t * tokens;
  if (t >= TILES || first >= it.n) return {0, 0, 0};
  const int end = min(first + tokens, it.n);
  const int c_last = p.causal ? end : it.n, c_first = p.causal ? first + 1 : it.n;
  const int from = p.window > 0 && c_first > p.window ? c_first - p.window : 0;
  return {from / kBN, (c_last + kBN - 1) / kBN, c_last};
}

// Pieces of a tile (its number in the sequence) that walks over some key blocks; the
// last piece takes what is left.
__device__ __forceinline__ int pieces_of(const Params& p, int tile, int blocks) {
  return tile < p.whole ? 1 : min(p.pieces, (blocks + p.split - 1) / p.split);
}
// What an item does of its tile's range.
template <int TILES, bool SPLIT>
__device__ __forceinline__ Range item_range(const Params& p, const Item& it, int t) {
  Range r = tile_range<TILES>(p, it, t);
  if (SPLIT && r.hi > 0 && it.t0 >= p.whole << (7 - p.gshift)) {
    const int lo = r.lo + it.piece * p.split;
    if (it.piece < p.pieces - 1) r.hi = min(r.hi, lo + p.split);
    r.lo = lo;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// u * 0 + sum in both halves: 0, or NaN once a u was not finite.
template <typename T>
__device__ __forceinline__ uint32_t odd2(uint32_t u, uint32_t sum);
template <>
__device__ __forceinline__ uint32_t odd2<__half>(uint32_t u, uint32_t sum) {
  asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(u), "r"(0u));
  return sum;
}
template <>
__device__ __forceinline__ uint32_t odd2<__nv_bfloat16>(uint32_t u, uint32_t sum) {
  asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(u), "r"(0u));
  return sum;
}

// Weights are held as 2^kLift of themselves (O and the row's sum alike, so it cancels).
// P.V takes them in 16 bits, relative to a running maximum that may lag by 2^8: fp16
// weights then end at 2^15, and those that would be subnormal or nothing keep 7 bits
// more. Without it thousands of weights below 2^-25 beside one large key were lost
// (65536 of them 2^-25.2 each: 0 for 1.6e-3).  bf16 has the range of fp32.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Position in the K/V ring: stage and phase of its barriers.
template <int N>
struct Slot {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// The exponential unit's 2^x, kept in program order: left free, the compiler
// moves the second half of a block's exponentials before the first half's store.
__device__ __forceinline__ float ex2_mufu(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One row from its definition, by one warp: lane l holds dims [l D/32, (l+1) D/32),
// four keys at a time.  Only rows whose fast result is not finite come here.
template <typename T, int D>
__device__ __noinline__ void row_by_row(const Params& p, int64_t row, int h, int64_t key0, int begin, int end,
                                        int dim0 = 0, int dims = D) {
  constexpr int E = D / 64;  // 32-bit words per lane
  const int lane = threadIdx.x & 31, hk = h / p.group;
  auto words = [&](const void* base, int64_t at, uint32_t (&w)[E]) {
    const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(base) + at) + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = src[e];
  };
  float q[2 * E], acc[2 * E], m = -INFINITY, l = 0.f;
  {
    uint32_t w[E];
    words(p.q, row * p.q_stride + static_cast<int64_t>(h) * D, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 f = unpack2<T>(w[e]);
      q[2 * e] = f.x * p.qscale;
      q[2 * e + 1] = f.y * p.qscale;
      acc[2 * e] = acc[2 * e + 1] = 0.f;
    }
  }
  for (int j0 = begin; j0 < end; j0 += 4) {
    uint32_t kw[4][E], vw[4][E];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t j = key0 + min(j0 + u, end - 1);
      words(p.k, j * p.k_stride + static_cast<int64_t>(hk) * D, kw[u]);
      words(p.v, j * p.v_stride + static_cast<int64_t>(hk) * D, vw[u]);
      s[u] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 f = unpack2<T>(kw[u][e]);
        s[u] += q[2 * e] * f.x + q[2 * e + 1] * f.y;
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (j0 + u < end) {
        const float mn = fmaxf(m, s[u]), a = l > 0.f ? exp2f(m - mn) : 0.f;
        const float w = s[u] == -INFINITY ? 0.f : exp2f(s[u] - mn);
        l = l > 0.f ? l * a + w : l + w;  // NaN stays: l > 0 is false then and w is added to it
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 f = unpack2<T>(vw[u][e]);
          acc[2 * e] = (l > 0.f ? acc[2 * e] * a : acc[2 * e]) + w * f.x;
          acc[2 * e + 1] = (l > 0.f ? acc[2 * e + 1] * a : acc[2 * e + 1]) + w * f.y;
        }
      }
    }
  }
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + (row * p.H + h) * D) + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = 2 * (lane * E + e);
    if (d >= dim0 && d < dim0 + dims) dst[e] = pack2<T>(acc[2 * e] / l, acc[2 * e + 1] / l);
  }
}

// Index i's share of the rows behind the last sequence, which end at row `rest`.
// Every index of the grid passes through one scheduler or another once, so this
// costs no launch (and out of line no instructions where there are no such rows).
template <typename T, int D>
__device__ __noinline__ void zero_share(const Params& p, int rest, uint32_t i) {
  rest = max(rest, 0);
  const int64_t share = (static_cast<int64_t>(p.T - rest) + gridDim.x - 1) / gridDim.x, first = rest + i * share;
  if (first >= p.T) return;
  const int64_t row = static_cast<int64_t>(p.H) * D, n = min(share, p.T - first) * row / 8;
  uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + first * row);
  for (int64_t e = threadIdx.x & 31; e < n; e += 32) dst[e] = make_uint4(0, 0, 0, 0);
}

// Barriers: items (2 slots: filled by the scheduler, read by the warps that
// work on it), Q (filled by TMA, free by commit), K/V ring, and per tile: scores
// ready (commit), first and second part of P ready (4 warps), P.V done
// (commit).
template <int STAGES>
struct Bars {
  uint64_t item_full[2], item_free[2], q_full, q_free, kv_full[STAGES], kv_free[STAGES];
  uint64_t s_full[2], p_part[2][2], pv_done[2], s_read[2], end[2], next, near_end;
};

template <typename T, int D, int TILES, bool SPLIT>
__global__ void __launch_bounds__(128 * TILES + 128, 3 - TILES)
packed_attention_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap qmap,
                        const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D, TILES>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t kIdescS = tc::idesc_f16(128, kBN, false, false, kBf16);
  constexpr uint32_t kIdescS64 = tc::idesc_f16(128, 64, false, false, kBf16);
  constexpr uint32_t kIdescPV = tc::idesc_f16(128, D, false, true, kBf16);
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) Bars<C::STAGES> bars;
  __shared__ Item items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int32_t cu_copy[C::CU];
  __shared__ __align__(16) uint4 next_cta;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform, and known to be
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(base);
  auto at = [](const uint64_t& b) { return smem_u32(&b); };
  const int tile_tokens = 128 >> p.gshift;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(at(bars.item_full[i]), 1);
      mbar_init(at(bars.item_free[i]), C::ITEM_READERS);
      mbar_init(at(bars.s_full[i]), 1);
      mbar_init(at(bars.p_part[i][0]), 4);
      mbar_init(at(bars.p_part[i][1]), 4);
      mbar_init(at(bars.pv_done[i]), 1);
      mbar_init(at(bars.s_read[i]), 4);
      mbar_init(at(bars.end[i]), 1);
    }
    mbar_init(at(bars.next), 1);
    mbar_init(at(bars.near_end), 1);
    mbar_init(at(bars.q_full), 1);
    mbar_init(at(bars.q_free), TILES);
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(at(bars.kv_full[i]), 1);
      mbar_init(at(bars.kv_free[i]), TILES);
    }
    fence_mbar_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(smem_u32(&tmem_slot), 256 * TILES);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  after_previous();
  const bool copied = p.S + 1 <= C::CU;
  if (copied) {
    for (int i = tid; i <= p.S; i += C::THREADS) cu_copy[i] = p.cu[i];
    __syncthreads();
  }
  const uint32_t tmem = tmem_slot;
  // Tile t: scores at its first 128 columns, O behind them, P over the scores or behind O.
  auto tS = [&](int t) { return tmem + 256u * t; };
  auto tO = [&](int t) { return tS(t) + 128u; };
  auto tP = [&](int t) { return C::OWN_P ? tO(t) + static_cast<uint32_t>(D) : tS(t); };

  // The k-th item of this CTA (read by every warp but the scheduler).
  auto next_item = [&](int k, Item& it) -> bool {
    const bool ok = __all_sync(0xffffffffu, wait_bar(at(bars.item_full[k & 1]), (k >> 1) & 1));
    if (!ok) return false;
    // Broadcast from one lane: the compiler then keeps what follows from the
    // item (descriptors, loop bounds) in uniform registers.
    const Item& src = items[k & 1];
    it.start = __shfl_sync(0xffffffffu, src.start, 0);
    it.n = __shfl_sync(0xffffffffu, src.n, 0);
    it.t0 = __shfl_sync(0xffffffffu, src.t0, 0);
    it.unit = __shfl_sync(0xffffffffu, src.unit, 0);
    if (SPLIT) {
      it.piece = __shfl_sync(0xffffffffu, src.piece, 0);
      it.slot = __shfl_sync(0xffffffffu, src.slot, 0);
    }
    if (lane == 0) mbar_arrive(at(bars.item_free[k & 1]));
    return it.n >= 0;
  };

  if (warp < C::MMA_WARP) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    // =========================== softmax warps ===========================
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint64_t qs2 = f32x2_pack(p.qscale, p.qscale);
    uint32_t blocks = 0;  // key blocks of this tile so far (phases of its barriers)
    bool ok = true;
    // The next item is read during the wait for an item's last P V where that is
    // faster: with one tile of 128 dims (64 x 128 tokens 40.2 -> 39.4 us, one prompt of
    // 2500 not causal 46.2 -> 44.7); with two tiles or 64 dims it is 2-5% slower.
    constexpr bool kEarly = TILES == 1 && D == 128;
    Item it, next;
    bool early = false, more = false;
    auto take = [&](int k) -> bool {
      if (!kEarly || !early) return next_item(k, it);
      early = false;
      it = next;
      return more;
    };
    for (int k = 0; ok && take(k); ++k) {
      const Range r = item_range<TILES, SPLIT>(p, it, t);
      if (r.hi == 0) continue;
      const int tok = it.t0 + t * tile_tokens + (row >> p.gshift);
      const int h = (it.unit << p.gshift) + (row & ((1 << p.gshift) - 1));
      const int c = p.causal ? min(tok + 1, it.n) : it.n;
      const int ws = p.window > 0 && c > p.window ? c - p.window : 0;
      float m_run = -INFINITY, l_run = 0.f;
      // The running maximum takes a block's maximum in: it moves only when it
      // grows by more than 2^8, and then O and the sum are rescaled.
      auto take_max = [&](float mx, int j) -> bool {
        const float m_new = fmaxf(m_run, mx * p.qscale);  // qscale > 0
        float alpha = 1.f;
        bool rescale = false;
        if (m_run == -INFINITY) {
          m_run = m_new;  // nothing accumulated yet
        } else if (m_new > m_run + 8.f) {
          alpha = tc::ex2(m_run - m_new);
          m_run = m_new;
          rescale = true;
        }
        if (__any_sync(0xffffffffu, rescale)) {
          // O holds the earlier blocks only once P.V of the last one completed.
          if (j > r.lo && !__all_sync(0xffffffffu, wait_bar(at(bars.pv_done[t]), (blocks - 1) & 1))) return false;
          tc::fence_after_sync();
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t v[16];
            tc::ld16_wait(tO(t) + lane_base + cc * 16, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
            tc::st16(tO(t) + lane_base + cc * 16, v);
          }
          tc::wait_st();
          l_run *= alpha;
        }
        return true;
      };
      // The scores are in registers: the next ones may overwrite them (OWN_P).
      auto s_read = [&] {
        if (!C::OWN_P) return;
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(at(bars.s_read[t]));
      };
      // P of the last block is no longer needed (OWN_P; else its scores say so).
      auto p_free = [&](int j) -> bool {
        if (!C::OWN_P || j == r.lo) return true;
        return __all_sync(0xffffffffu, wait_bar(at(bars.pv_done[t]), (blocks - 1) & 1));
      };
      auto p_ready = [&](int half) {
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(at(bars.p_part[t][half]));
      };
      for (int j = r.lo; j < r.hi && ok; ++j, ++blocks) {
        ok = __all_sync(0xffffffffu, wait_bar(at(bars.s_full[t]), blocks & 1));
        if (!ok) break;
        tc::fence_after_sync();
        const int lo = ws - j * kBN, hi = c - j * kBN;  // visible columns [lo, hi)
        uint64_t sum2[4] = {0, 0, 0, 0};
        if (__any_sync(0xffffffffu, lo > 0 || hi < kBN)) {
          // An edge of the mask: 32 columns at a time up to the last one that the
          // tile sees, the maximum first, then the weights from the scores read
          // again (where P lies over the scores, P of a chunk is below the scores of
          // the next one).
          const int chunks = (min(kBN, r.last - j * kBN) + 31) / 32;
          // Chunks [begin, end) hold a column that a row of this warp sees; the
          // others get weights of 0 without a look at their scores.
          const int begin = max(__reduce_min_sync(0xffffffffu, lo), 0) / 32;
          const int end = min(chunks, (max(__reduce_max_sync(0xffffffffu, hi), 0) + 31) / 32);
          auto chunk = [&](int cc, float (&v)[32]) {
            tc::ld32(tS(t) + lane_base + cc * 32, v);
            tc::wait_ld(v);
            const int l = lo - cc * 32, u = hi - cc * 32;
            if (__any_sync(0xffffffffu, l > 0 || u < 32)) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = (i >= l && i < u) ? v[i] : -INFINITY;
            }
          };
          float mx = -INFINITY;
#pragma unroll 1
          for (int cc = begin; cc < end; ++cc) {
            float v[32];
            chunk(cc, v);
            float m0 = v[0], m1 = v[1];
#pragma unroll
            for (int i = 2; i < 32; i += 2) {
              m0 = fmaxf(m0, v[i]);
              m1 = fmaxf(m1, v[i + 1]);
            }
            mx = fmaxf(mx, fmaxf(m0, m1));
          }
          ok = take_max(mx, j) && p_free(j);
          if (!ok) break;
          const float add = kLift<T> - (m_run == -INFINITY ? 0.f : m_run);  // nothing visible yet: every weight is 2^-inf = 0
          const uint64_t nm2 = f32x2_pack(add, add);
#pragma unroll 1
          for (int cc = 0; cc < chunks; ++cc) {
            uint32_t ph[16] = {};
            if (cc >= begin && cc < end) {
              float v[32];
              chunk(cc, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float x0, x1;
                f32x2_unpack(f32x2_fma(f32x2_pack(v[2 * i], v[2 * i + 1]), qs2, nm2), x0, x1);
                x0 = tc::ex2(x0);
                x1 = tc::ex2(x1);
                sum2[i & 3] = f32x2_add(sum2[i & 3], f32x2_pack(x0, x1));
                ph[i] = pack2<T>(x0, x1);
              }
            }
            if (cc == chunks - 1) s_read();
            tc::st16(tP(t) + lane_base + cc * 16, ph);
            if (2 * (cc + 1) == kFirst) p_ready(0);
          }
          if (2 * chunks < kFirst) p_ready(0);
          p_ready(1);
        } else {
          float s[kBN];
          {
            float v[4][32];
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) tc::ld32(tS(t) + lane_base + cc * 32, v[cc]);
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
              tc::wait_ld(v[cc]);
#pragma unroll
              for (int i = 0; i < 32; ++i) s[cc * 32 + i] = v[cc][i];
            }
          }
          s_read();
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int i = 4; i < kBN; i += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(fmaxf(mx[e], s[i + e]), s[i + 4 + e < kBN ? i + 4 + e : i + e]);
          }
          ok = take_max(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), j);
          if (!ok) break;
          const float add = kLift<T> - (m_run == -INFINITY ? 0.f : m_run);
          const uint64_t nm2 = f32x2_pack(add, add);
          ok = p_free(j);
          if (!ok) break;
          // 32 keys at a time; P.V starts on the first kFirst steps of 16 keys.
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t ph[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int e = cc * 32 + 2 * i;
              float x0, x1;
              f32x2_unpack(f32x2_fma(f32x2_pack(s[e], s[e + 1]), qs2, nm2), x0, x1);
              x0 = ex2_mufu(x0);
              x1 = ex2_mufu(x1);
              sum2[i & 3] = f32x2_add(sum2[i & 3], f32x2_pack(x0, x1));  // the row sum adds them unrounded
              ph[i] = pack2<T>(x0, x1);
            }
            tc::st16(tP(t) + lane_base + cc * 16, ph);
            if (2 * (cc + 1) == kFirst) p_ready(0);
          }
          p_ready(1);
        }
        float a0, a1, b0, b1;
        f32x2_unpack(f32x2_add(sum2[0], sum2[1]), a0, a1);
        f32x2_unpack(f32x2_add(sum2[2], sum2[3]), b0, b1);
        l_run += (a0 + a1) + (b0 + b1);
      }
      if (kEarly && ok) {
        early = true;
        more = next_item(k + 1, next);
      }
      if (ok) ok = __all_sync(0xffffffffu, wait_bar(at(bars.pv_done[t]), (blocks - 1) & 1));
      tc::fence_after_sync();
      if (SPLIT) {
        const Range all = tile_range<TILES>(p, it, t);
        if (pieces_of(p, it.t0 >> (7 - p.gshift), all.hi - all.lo) > 1) {
          // One of several pieces: O as it is, and the row's maximum and sum.
          const int64_t at = static_cast<int64_t>(it.slot) * p.pieces + it.piece;
          float4* po = p.part_o + at * (D / 4) * 128 + row;
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            float v[32];
            tc::ld32(tO(t) + lane_base + cc * 32, v);
            tc::wait_ld(v);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              po[(cc * 8 + e) * 128] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
          p.part_ml[at * 128 + row] = make_float2(m_run, ok ? l_run : __int_as_float(0x7fffffff));
          tc::fence_before_sync();
          continue;
        }
      }
      // Epilogue: 32 dims of a row are four 16-byte pieces of its thread; the four
      // threads of neighbouring rows exchange pieces, so that a store writes 64
      // contiguous bytes of each of 8 rows instead of 16 bytes of 32 rows.
      const float inv = ok ? 1.f / l_run : __int_as_float(0x7fffffff);
      const uint64_t inv2 = f32x2_pack(inv, inv);
      uint32_t odd = 0;  // becomes NaN when an element is not finite
      T* rows[4];       // the four rows of this thread's group (null: behind the sequence)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tr = (row & ~3) + i, to = it.t0 + t * tile_tokens + (tr >> p.gshift);
        const int ho = (it.unit << p.gshift) + (tr & ((1 << p.gshift) - 1));
        rows[i] = to < it.n ? static_cast<T*>(p.out) + (static_cast<int64_t>(it.start + to) * p.H + ho) * D + (lane & 3) * 8
                            : nullptr;
      }
#pragma unroll 1
      for (int cc = 0; cc < D / 32; ++cc) {
        float v[32];
        tc::ld32(tO(t) + lane_base + cc * 32, v);
        tc::wait_ld(v);
        uint32_t w[4][4];  // piece, word
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x0, x1;
          f32x2_unpack(f32x2_mul(f32x2_pack(v[2 * i], v[2 * i + 1]), inv2), x0, x1);
          w[i / 4][i % 4] = pack2<T>(x0, x1);
          odd = odd2<T>(w[i / 4][i % 4], odd);
        }
        // 4 x 4 transpose: piece c of row r goes to thread c, place r.
#pragma unroll
        for (int step = 1; step < 4; step <<= 1) {
          const bool up = lane & step;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c & step) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[c][i] : w[c + step][i], step);
              if (up) w[c][i] = got;
              else w[c + step][i] = got;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (rows[r]) *reinterpret_cast<uint4*>(rows[r] + cc * 32) = make_uint4(w[r][0], w[r][1], w[r][2], w[r][3]);
        }
      }
      tc::fence_before_sync();
      // A weight of the row's maximum is at least 1 and no weight exceeds 2^15 (both
      // with the lift), so a sum outside [1/2, 2^100) is not one of finite scores.
      uint32_t redo = __ballot_sync(0xffffffffu, ok && tok < it.n && !((odd & 0x7fff7fffu) == 0 && l_run >= 0.5f && l_run < 1.2e30f));
      __syncwarp();
      while (redo) {
        const int from = __ffs(redo) - 1;
        redo &= redo - 1;
        const int rt = __shfl_sync(0xffffffffu, tok, from), rh = __shfl_sync(0xffffffffu, h, from);
        const int rb = __shfl_sync(0xffffffffu, ws, from), re = __shfl_sync(0xffffffffu, c, from);
        row_by_row<T, D>(p, it.start + rt, rh, it.start, rb, re);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
    if (warp < C::LOAD_WARP) {
      // ============================= MMA warps =============================
      // One warp per tile, so that a wait of one leaves the tensor pipe to the
      // other.  Warp-uniform code; elect.sync issues each instruction once.
      // Both follow every K/V block of the item, used or not: a block is free
      // when both have let it go.
      const int t = warp - C::MMA_WARP;
      const uint64_t dq = tc::sdesc_sw128(sbase + t * C::TILE, 16, 1024);
      const uint64_t dk0 = tc::sdesc_sw128(sbase + C::KV_OFF, 16, 1024);
      const uint64_t dv0 = tc::sdesc_sw128(sbase + C::KV_OFF, C::HALF, 1024);
      Slot<C::STAGES> ring;        // of the next block to use
      uint32_t blocks = 0;         // P blocks of the tile so far
      bool ok = true;
      auto wait_for = [&](const uint64_t& b, uint32_t parity) { ok &= wait_bar(at(b), parity & 1); };
      auto in_step = [&] {  // the waits' outcome, the same in every lane
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after_sync();
        return ok;
      };
      Item it;
      for (int k = 0; ok && next_item(k, it); ++k) {
        const Range r0 = item_range<TILES, SPLIT>(p, it, 0), r1 = item_range<TILES, SPLIT>(p, it, 1);
        const int LO = r0.lo, HI = max(r0.hi, r1.hi);  // tile 0 exists and starts first
        const int lo = t ? r1.lo : r0.lo, hi = t ? r1.hi : r0.hi, last = t ? r1.last : r0.last;
        auto scores = [&](int j) {  // S(j) if the tile has the block; lets K(j) and, at the end, Q go
          if (j >= lo && j < hi) {
            // The softmax reads 64 columns where no key behind them is seen.
            const uint32_t idesc = last - j * kBN > 64 ? kIdescS : kIdescS64;
            const uint64_t dk = dk0 + static_cast<uint64_t>((ring.stage * C::TILE) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint64_t off = static_cast<uint64_t>(((kk / 4) * C::HALF + (kk % 4) * 32) >> 4);
              tc::mma_f16_elect(tS(t), dq + off, dk + off, idesc, kk > 0);
            }
            tc::commit_elect(at(bars.s_full[t]));
          }
          tc::commit_elect(at(bars.kv_free[ring.stage]));
          if (j == HI - 1) tc::commit_elect(at(bars.q_free));
          ring.next();
        };
        wait_for(bars.q_full, k);
        wait_for(bars.kv_full[ring.stage], ring.phase);
        if (!in_step()) break;
        scores(LO);
        for (int j = LO; j < HI; ++j) {
          const Slot<C::STAGES> v = ring;
          wait_for(bars.kv_full[v.stage], v.phase);
          if (j == HI - 1 && HI * kBN > it.n && (it.n & 15)) {
            // The block runs past the sequence's end: its rows there, up to the
            // 16 keys of an instruction, become zero.
            const int first = it.n - j * kBN, rows = 16 - (first & 15);
            uint8_t* v0 = base + C::KV_OFF + v.stage * C::TILE + first * 128;
            for (int i = lane; i < rows * C::HALVES * 8; i += 32)
              *reinterpret_cast<uint4*>(v0 + (i % C::HALVES) * C::HALF + (i / C::HALVES) * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
          ring.next();
          if (j + 1 < HI) wait_for(bars.kv_full[ring.stage], ring.phase);
          if (C::OWN_P && j + 1 < HI) {
            if (j >= lo && j < hi) wait_for(bars.s_read[t], blocks);
            if (!in_step()) break;
            scores(j + 1);
          }
          if (j >= lo && j < hi) {
            const uint64_t dv = dv0 + static_cast<uint64_t>((v.stage * C::TILE) >> 4);
            const int steps = min(kBN, last - j * kBN + 15) / 16;  // of 16 keys, up to the last one seen
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              wait_for(bars.p_part[t][part], blocks);
              if (!in_step()) break;
#pragma unroll
              for (int kk = part ? kFirst : 0; kk < (part ? 8 : kFirst); ++kk) {
                if (kk < steps)
                  tc::mma_f16_tmem_a_elect(tO(t), tP(t) + 8u * kk, dv + static_cast<uint64_t>((kk * 2048) >> 4),
                                           kIdescPV, (j > lo || kk > 0) ? 1u : 0u);
              }
            }
            if (!ok) break;
            tc::commit_elect(at(bars.pv_done[t]));
            ++blocks;
          } else if (!in_step()) {
            break;
          }
          tc::commit_elect(at(bars.kv_free[v.stage]));
          if (!C::OWN_P && j + 1 < HI) scores(j + 1);
        }
      }
      // The last commit's arrival lands before the CTA ends.
      if (ok) {
        tc::commit_elect(at(bars.end[t]));
        wait_bar(at(bars.end[t]), 0);
      }
    } else if (warp == C::LOAD_WARP) {
      // ============================== loads ==============================
      if (lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
      }
      uint32_t loads = 0;
      bool ok = true;
      Item it;
      for (int k = 0; ok && next_item(k, it); ++k) {
        const Range r0 = item_range<TILES, SPLIT>(p, it, 0), r1 = item_range<TILES, SPLIT>(p, it, 1);
        const int LO = r0.lo, HI = max(r0.hi, r1.hi);
        const int h0 = it.unit << p.gshift, hk = h0 / p.group;
        if (lane == 0) {
          if (k > 0) ok = wait_bar(at(bars.q_free), (k - 1) & 1);
          if (ok) {
            const int ntiles = r1.hi > 0 ? 2 : 1;
            mbar_arrive_expect_tx(at(bars.q_full), ntiles * C::TILE);
            for (int t = 0; t < ntiles; ++t)
              for (int hh = 0; hh < C::HALVES; ++hh)
                tma_load_3d(sbase + t * C::TILE + hh * C::HALF, &qmap, hh * 64, h0,
                            it.start + it.t0 + t * tile_tokens, at(bars.q_full));
          }
          for (int j = LO; j < HI && ok; ++j) {
            if (j == max(HI - kAhead, LO)) mbar_arrive(at(bars.near_end));
            for (int v = 0; v < 2 && ok; ++v, ++loads) {
              const int st = loads % C::STAGES;
              const uint32_t use = loads / C::STAGES;
              if (use > 0) ok = wait_bar(at(bars.kv_free[st]), (use - 1) & 1);
              if (!ok) break;
              mbar_arrive_expect_tx(at(bars.kv_full[st]), C::TILE);
              for (int hh = 0; hh < C::HALVES; ++hh)
                tma_load_3d(sbase + C::KV_OFF + st * C::TILE + hh * C::HALF, v ? &vmap : &kmap, hh * 64, hk,
                            it.start + j * kBN, at(bars.kv_full[st]));
            }
          }
          if (!ok) {  // nothing may be in flight when the CTA ends
            for (uint32_t u = loads > C::STAGES ? loads - C::STAGES : 0; u < loads; ++u)
              wait_bar(at(bars.kv_full[u % C::STAGES]), (u / C::STAGES) & 1);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        loads = __shfl_sync(0xffffffffu, loads, 0);
      }
    } else if (warp == C::SCHED_WARP) {
      // ============================ scheduler ============================
      // Head units in chunks (their keys and values stay in L2 while the chunk's
      // items run); within a chunk the items in descending order of work, within a
      // token block the units.
      const int tshift = 7 - p.gshift + (TILES - 1), tokens = 1 << tshift;
      const int32_t* cu = copied ? cu_copy : p.cu;
      auto bounds = [&](int s, int& lo, int& hi) {  // device data: kept inside the tensors
        lo = min(max(cu[s], 0), p.T);
        hi = min(max(cu[s + 1], lo), p.T);
      };
      auto nblocks = [&](int s) {
        int lo = 0, hi = 0;
        if (s < p.S) bounds(s, lo, hi);
        return (hi - lo + tokens - 1) >> tshift;
      };
      int most = 0;
      int64_t all = 0;
#pragma unroll 4
      for (int s = lane; s < p.S; s += 32) {
        const int nb = nblocks(s);
        most = max(most, nb);
        all += nb;
      }
      most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
      for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
      // Token blocks are walked level by level.  Causal: level = index of the
      // block in its sequence, descending; a sequence has one block on it if it
      // is long enough.  Not causal: level = blocks of the sequence, descending;
      // a sequence of that many has all of them on it.
      auto reaches = [&](int nb, int L) { return p.causal ? nb > L : nb == L; };
      auto on_level = [&](int s, int L) { return reaches(nblocks(s), L); };
      // Up to 32 sequences, a sequence to a lane, are counted without a loop: few
      // sequences have many levels, and a CTA's first item may lie far down (one
      // prompt of 4000 tokens, 16/4 heads 89 -> 71 us).
      const int own_blocks = nblocks(lane);
      // Pieces of a token block on a level, at most (a shorter last block may have
      // fewer; what is too many is skipped).
      auto pieces_on = [&](int L) {
        if (!SPLIT) return 1;
        const int hi = ((p.causal ? L + 1 : L) * tokens + kBN - 1) / kBN;
        const int first = (p.causal ? L : L - 1) * tokens + 1;
        return pieces_of(p, p.whole, hi - (p.window > 0 && first > p.window ? (first - p.window) / kBN : 0));
      };
      // Items of a sequence on a level: one tile's pieces, or (not causal) all L tiles,
      // the first of them whole.
      auto items_on = [&](int L) {
        if (p.causal) return pieces_on(L);
        return SPLIT ? min(L, p.whole) + max(L - p.whole, 0) * pieces_on(L) : L;
      };
      auto count_on = [&](int L) {  // token blocks (split: their pieces) on a level
        int n = 0;
        if (p.S <= 32) {
          n = __popc(__ballot_sync(0xffffffffu, reaches(own_blocks, L)));
        } else {
#pragma unroll 4
          for (int s = lane; s < p.S; s += 32) n += on_level(s, L);
          n = __reduce_add_sync(0xffffffffu, n);
        }
        return static_cast<uint32_t>(n) * items_on(L);
      };
      auto next_level = [&](int L) {
        if (p.causal) return L - 1;
        int below = 0;
        for (int s = lane; s < p.S; s += 32) {
          const int nb = nblocks(s);
          if (nb < L) below = max(below, nb);
        }
        return static_cast<int>(__reduce_max_sync(0xffffffffu, below));
      };
      // The launch has at least as many CTAs as items, fewer than 2^31: indexes are
      // 32-bit.  (Overlapping sequences, which the host cannot see, may have more
      // items; those past the launch are not computed.)
      const uint32_t blocks_all = static_cast<uint32_t>(min(all, static_cast<int64_t>(0x7fffffff) / p.units));
      const uint32_t total = blocks_all * p.units, per_chunk = blocks_all * p.chunk;
      int L = 0;
      uint32_t chunk_first = 0, chunk_units = 0;  // the present chunk's head units
      uint32_t above = 0, here = 0, on_first = 0;  // token blocks on the levels above, on this one, on the first
      int found_level = -1, found_s0 = 0, found_before = 0;  // sequences on the level before found_s0
      bool ok = true, more = true;  // more: there may be CTAs that have not begun
      uint32_t i = blockIdx.x;
      uint32_t asked = 0;
      // Takes the index of a CTA that has not begun; false when there is none left.
      // Nothing promises an order of the indexes, so each of them is looked up, also
      // behind one that had no item.
      auto take_next = [&]() -> bool {
        if (lane == 0) {
          mbar_arrive_expect_tx(at(bars.next), 16);
          tc::try_cancel(smem_u32(&next_cta), at(bars.next));
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, wait_bar(at(bars.next), asked++ & 1));
        uint32_t cta = 0;
        const bool got = ok && tc::query_cancel(smem_u32(&next_cta), cta);
        fence_proxy_async_smem();  // read before the next answer is written
        __syncwarp();
        i = cta;
        return got;
      };
      const bool zero = p.zero_rest && cu[p.S] < p.T;  // there are rows behind the last sequence
      // The item of index i; false when there is none.  The items are those of the
      // indexes below `end` (split: an upper bound that every miss lowers).
      uint32_t end = SPLIT ? 0xffffffffu : total;
      auto find = [&](Item& it) -> bool {
        if (i >= end) return false;
        if (SPLIT) {
          chunk_units = p.units;  // few items: all units at once
        } else if (chunk_units == 0 || i < chunk_first * blocks_all || i >= (chunk_first + chunk_units) * blocks_all) {
          chunk_first = i / per_chunk * p.chunk;
          chunk_units = min(static_cast<uint32_t>(p.chunk), p.units - chunk_first);
          above = here = 0;
        }
        const uint32_t in_chunk = SPLIT ? i : i - chunk_first * blocks_all, b = in_chunk / chunk_units;
        if (here == 0 || b < above) {
          above = 0;
          L = p.causal ? most - 1 : most;
          if (on_first == 0 && most > 0) on_first = count_on(L);
          here = on_first;
        }
        while (b >= above + here) {
          above += here;
          L = next_level(L);
          if (SPLIT && (p.causal ? L < 0 : L <= 0)) {
            here = 0;
            end = i;
            return false;
          }
          if (!SPLIT || !p.causal) {
            here = count_on(L);
            continue;
          }
          // Split items are found by a level to a lane, 32 levels at once: each has
          // its own number of pieces (one prompt of 4000 tokens, 4/1 heads 52 -> 33 us).
          const int own = max(L - lane, 0);
          uint32_t n = 0;
          for (int s = 0; s < p.S; ++s) n += reaches(p.S <= 32 ? __shfl_sync(0xffffffffu, own_blocks, s) : nblocks(s), own);
          n = L >= lane ? n * pieces_on(own) : 0;
          uint32_t sum = n;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += v;
          }
          const uint32_t reached = __ballot_sync(0xffffffffu, b < above + sum);
          const int from = reached ? __ffs(reached) - 1 : 31;
          above += __shfl_sync(0xffffffffu, reached ? sum - n : sum, from);
          here = reached ? __shfl_sync(0xffffffffu, n, from) : 0;
          L -= from;
        }
        const int at_level = static_cast<int>(b - above), pieces = pieces_on(L);
        // The sequence is the rank-th on the level.  Ranks grow from item to item:
        // the search goes on where the last one ended.
        const int per_seq = items_on(L);
        const int rank = p.causal && !SPLIT ? at_level : at_level / per_seq;
        if (L != found_level || rank < found_before) {
          found_level = L;
          found_s0 = found_before = 0;
        }
        int skip = rank - found_before;
        for (int s0 = found_s0; s0 < p.S; s0 += 32) {
          const uint32_t has = __ballot_sync(0xffffffffu, on_level(s0 + lane, L));
          const int n = __popc(has);
          if (skip < n) {
            const bool found = ((has >> lane) & 1u) && __popc(has & ((1u << lane) - 1u)) == skip;
            const int s = s0 + __ffs(__ballot_sync(0xffffffffu, found)) - 1;
            int lo, hi;
            bounds(s, lo, hi);
            found_s0 = s0;
            const int rest = at_level - rank * per_seq;
            int tile = p.causal ? L : rest, piece = p.causal ? rest : 0;
            if (SPLIT && !p.causal && rest >= p.whole) {
              const int of = (rest - p.whole) / pieces;
              tile = p.whole + of;
              piece = rest - p.whole - of * pieces;
            }
            const int unit = static_cast<int>(chunk_first + in_chunk - b * chunk_units);
            it = Item{lo, hi - lo, tile * tokens, unit, 0, 0};
            if (SPLIT) {
              it.piece = piece;
              it.slot = ((lo + it.t0) / tokens + s - p.whole) * p.units + unit;  // (a whole tile has none)
            }
            return true;
          }
          skip -= n;
          found_before += n;
        }
        return false;
      };
      for (int k = 0; ok; ++k) {
        if (k >= 2) ok = __all_sync(0xffffffffu, wait_bar(at(bars.item_free[k & 1]), ((k >> 1) - 1) & 1));
        if (!ok) break;
        // Not before the item at hand nears its end: what is taken early is missing
        // where another CTA runs dry.
        if (k > 0) {
          ok = __all_sync(0xffffffffu, wait_bar(at(bars.near_end), (k - 1) & 1));
          if (!ok) break;
          more = take_next();
        }
        Item it{0, -1, 0, 0, 0, 0}, got = it;
        while (more) {
          if (zero) zero_share<T, D>(p, cu[p.S], i);
          bool has = find(got);
          if (SPLIT && has) {  // not a piece that this token block does not have
            const Range r = item_range<TILES, SPLIT>(p, got, 0);
            has = r.lo < r.hi;
          }
          if (has) {
            it = got;
            break;
          }
          more = take_next();
        }
        if (!ok) break;
        if (lane == 0) {
          items[k & 1] = it;
          mbar_arrive(at(bars.item_full[k & 1]));
        }
        __syncwarp();
        if (it.n < 0) break;  // no CTA is left that has not begun
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::tmem_dealloc(tmem, 256 * TILES);
}

// Joins the pieces of a tile: with M the largest of the pieces' maxima,
// out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p.  A CTA for 16 dims of a tile
// and head unit, a thread for a row: its loads do not wait for one another.
// Bound by the latency of a launch and two dependent loads: 10 us cold for 4000 tokens
// of 4/1 heads (17 MB of pieces).  With a CTA for all dims of a tile and head unit the
// whole call was slower (1000 tokens of 32/8 heads, split: 44 us against 33).
template <typename T, int D>
__global__ void __launch_bounds__(128) join_pieces_kernel(const __grid_constant__ Params p) {
  const int row = threadIdx.x, tokens = 128 >> p.gshift;
  const int slot = blockIdx.x / p.units, unit = blockIdx.x - slot * p.units, g = slot + p.whole;
  after_previous();
  auto bounds = [&](int s, int& lo, int& hi) {
    lo = min(max(p.cu[s], 0), p.T);
    hi = min(max(p.cu[s + 1], lo), p.T);
  };
  // The tile's number is (first packed row of it) / tokens + its sequence, which
  // grows along the batch: the last sequence whose first tile is not behind g.
  int lo = 0, hi = 0, s = 0;
  for (int below = 0, above = p.S; below < above;) {
    const int mid = (below + above) / 2;
    bounds(mid, lo, hi);
    if (lo / tokens + mid <= g) {
      s = mid;
      below = mid + 1;
    } else {
      above = mid;
    }
  }
  bounds(s, lo, hi);
  const int tile = g - (lo / tokens + s);
  Item it{lo, hi - lo, tile * tokens, unit, 0, 0};
  if (tile < 0 || static_cast<int64_t>(tile) * tokens >= it.n) return;
  const Range r = tile_range<1>(p, it, 0);
  const int pieces = pieces_of(p, tile, r.hi - r.lo);
  if (pieces <= 1) return;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * p.pieces;
  const float2* ml = p.part_ml + at * 128 + row;
  const float4* po = p.part_o + (at * (D / 4) + blockIdx.y * 4) * 128 + row;
  float m = -INFINITY, l = 0.f, w[kMaxPieces];
#pragma unroll
  for (int i = 0; i < kMaxPieces; ++i) {
    w[i] = i < pieces ? ml[i * 128].x : -INFINITY;
    m = fmaxf(m, w[i]);
  }
  float acc[16] = {};
#pragma unroll
  for (int i = 0; i < kMaxPieces; ++i) {
    if (i >= pieces) continue;
    w[i] = w[i] == -INFINITY ? 0.f : exp2f(w[i] - m);  // nothing seen in the piece: its sum is 0
    l += w[i] * ml[i * 128].y;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 o = po[(i * (D / 4) + c) * 128];
      acc[4 * c] += w[i] * o.x, acc[4 * c + 1] += w[i] * o.y;
      acc[4 * c + 2] += w[i] * o.z, acc[4 * c + 3] += w[i] * o.w;
    }
  }
  float odd = 0.f;  // becomes NaN when an element is not finite
#pragma unroll
  for (int e = 0; e < 16; ++e) odd = fmaf(acc[e], 0.f, odd);
  const int tok = it.t0 + (row >> p.gshift), h = (unit << p.gshift) + (row & ((1 << p.gshift) - 1));
  const int c = p.causal ? min(tok + 1, it.n) : it.n;
  const int ws = p.window > 0 && c > p.window ? c - p.window : 0;
  if (tok < it.n) {
    const float inv = 1.f / l;
    uint32_t out[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = pack2<T>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (static_cast<int64_t>(lo + tok) * p.H + h) * D +
                                          blockIdx.y * 16);
    dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
    dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
  }
  uint32_t redo = __ballot_sync(0xffffffffu, tok < it.n && !(odd == 0.f && l >= 0.5f && l < 1.2e30f));
  __syncwarp();
  while (redo) {
    const int from = __ffs(redo) - 1;
    redo &= redo - 1;
    const int rt = __shfl_sync(0xffffffffu, tok, from), rh = __shfl_sync(0xffffffffu, h, from);
    const int rb = __shfl_sync(0xffffffffu, ws, from), re = __shfl_sync(0xffffffffu, c, from);
    row_by_row<T, D>(p, lo + rt, rh, lo, rb, re, blockIdx.y * 16, 16);
  }
}

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [rows][heads][D] with `stride` elements between rows; a box is 64 dims x
// box_heads x box_rows, 128-byte swizzle, token-major rows.  Rows past the
// tensor read as zero.
int map_rows(CUtensorMap* map, const void* base, bool bf16, int64_t rows, int64_t stride, int heads, int D,
             int box_heads, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return fail(MEMOPT_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(stride) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(MEMOPT_ERR_CUDA, "packed_attention: cuTensorMapEncodeTiled failed: " + std::to_string(static_cast<int>(r)));
  return MEMOPT_OK;
}

// How a call is launched.
struct Plan {
  int gshift, units, tiles;
  int split, pieces;       // 0: no item is split
  int whole;               // tiles of a sequence that stay whole (not causal)
  int64_t tile_slots;      // tiles x head units that may be split
  int64_t grid, workspace;
};
Plan plan_of(int S, int64_t T, int max_seqlen, int H, int KVH, int D, int window, bool causal) {
  Plan pl{};
  const int group = H / KVH, slots = 2 * sm_count();
  while ((2 << pl.gshift) <= kMaxGp && group % (2 << pl.gshift) == 0) ++pl.gshift;
  pl.units = H >> pl.gshift;
  // At most this many items (each sequence has one partial token block at most).
  const int64_t tokens = 128 >> pl.gshift;
  auto most_items = [&](int tiles) { return (T / (tokens * tiles) + S) * pl.units; };
  // Two tiles an item halve the K/V traffic and pay where the walk over the keys is
  // long and the items are many: 2 x 8192 tokens, 32/32 heads 1.02 ms against 1.10 with
  // one tile, 32/8 heads 0.98 against 1.07, 12 x 800 with 32/8 heads of 64 dims 71.5
  // against 80.8 us.  One tile, two CTAs to an SM, hides an item's ends better and makes
  // twice the items: 32 x 512 tokens, 32/8 heads of 128 dims 114 against 118, 64 x 32
  // 13.2 against 18.4, one prompt of 1000 20.9 against 25.7.  (Just above the border it
  // would be the better form still: 12 x 800 of 128 dims 88 against 96.)
  pl.tiles = T >= 768LL * S && most_items(2) >= 2 * sm_count() ? 2 : 1;
  // Few rows with long walks: the longest item would go on alone, so items are split
  // into pieces of `split` key blocks.  With the longest sequence as hinted and the
  // others of equal length: causal walks grow along a sequence and make about
  // (all their blocks) / split + half an item per tile; other walks are alike and
  // make ceil(walk / split) each.  The split that fills `rounds` items for every CTA
  // slot is taken where `rounds` times it and an item's own time (kItemBlocks) is least.
  const int64_t longest = std::min<int64_t>(T, std::max<int64_t>(max_seqlen, (T + S - 1) / S));
  const int64_t others = S > 1 ? (T - longest) / (S - 1) : 0;
  auto walk_of = [&](int64_t n) {  // key blocks of a row's walk over a sequence of n tokens, at most
    return ((window > 0 ? std::min<int64_t>(n, int64_t(window) + 128) : n) + kBN - 1) / kBN;
  };
  auto tiles_of = [&](int64_t n) { return (n + tokens - 1) / tokens; };
  const int64_t walk = walk_of(longest);
  const double tiles = static_cast<double>(tiles_of(longest) + (S - 1) * tiles_of(others)) * pl.units;
  const double blocks = 0.5 * (tiles_of(longest) * walk + (S - 1) * tiles_of(others) * walk_of(others)) * pl.units;
  // Not causal, a little more than a whole number of items for every slot: the first
  // `whole` tiles of a sequence fill the slots, and the rest are split into another
  // round; left whole they would take as long again (0.65 of it where they have the SM
  // to themselves: 1.5 against 2.3 us a block of 128 dims).  One prompt of 2500 tokens,
  // 16/4 heads 79 -> 59 us, 10000 of 4 heads 290 -> 182, 8192 of 10 heads 384 -> 314.
  // Items of two tiles take 0.85 of the time of two items (1.95 against 2.29 us a
  // block).  Tiles of shorter sequences count by their walks.
  const double even = static_cast<double>(tiles_of(longest) * walk + (S - 1) * tiles_of(others) * walk_of(others)) *
                      pl.units / walk;
  const double filled = causal ? 0 : std::floor(even / slots);
  const bool spill = filled > 0;
  const double rest = spill ? even - filled * slots : tiles;  // tiles that may be split
  const double first = filled * (walk + kItemBlocks);
  double best = walk;
  if (spill && rest > 0)
    best = pl.tiles == 2 ? std::ceil(even / slots) * (0.85 * walk + kItemBlocks)
                         : first + (walk + kItemBlocks) * (rest <= slots / 2 ? 0.65 : 1.0);
  best -= kSplitGain;
  for (int rounds = 1; rounds <= 3; ++rounds) {
    double split;
    if (causal && window <= 0) {
      if (rounds * slots <= 0.5 * tiles) continue;
      split = std::ceil(blocks / (rounds * slots - 0.5 * tiles));
    } else {
      if (rounds * slots < rest || rest <= 0) continue;
      split = std::ceil(walk / std::floor(rounds * slots / rest));
    }
    split = std::max(3.0, split);
    const double time = first + rounds * (split + kItemBlocks) - (spill ? 0 : kItemBlocks);
    const int64_t pieces = std::min<int64_t>(kMaxPieces, static_cast<int64_t>((walk + split - 1) / split));
    const int whole = spill ? static_cast<int>(tiles_of(longest) * filled * slots / even) : 0;
    const int64_t tile_slots = (T / tokens + S - whole) * pl.units, bytes = tile_slots * pieces * 128 * (D * 4 + 8);
    if (time >= best || pieces < 2 || bytes > kMaxWorkspace) continue;
    best = time;
    pl.split = static_cast<int>(split);
    pl.pieces = static_cast<int>(pieces);
    pl.whole = whole;
    pl.tile_slots = tile_slots;
    pl.workspace = bytes;
  }
  if (pl.split) pl.tiles = 1;
  // Every tile, and the further pieces of those that are split.
  pl.grid = most_items(pl.tiles);
  if (pl.split) pl.grid += pl.tile_slots * (pl.pieces - 1);
  return pl;
}

template <typename T, int D, int TILES, bool SPLIT>
int launch(const Params& p, int KVH, const Plan& pl, cudaStream_t s) {
  using C = Cfg<D, TILES>;
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  alignas(64) CUtensorMap qm, km, vm;
  const int Gp = 1 << p.gshift;
  int st = map_rows(&qm, p.q, bf16, p.T, p.q_stride, p.H, D, Gp, 128 / Gp);
  if (st == MEMOPT_OK) st = map_rows(&km, p.k, bf16, p.T, p.k_stride, KVH, D, 1, kBN);
  if (st == MEMOPT_OK) st = map_rows(&vm, p.v, bf16, p.T, p.v_stride, KVH, D, 1, kBN);
  if (st != MEMOPT_OK) return st;
  auto kern = packed_attention_kernel<T, D, TILES, SPLIT>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(packed_attention)");
  MEMOPT_LAUNCH(launch_after(kern, static_cast<unsigned>(pl.grid), C::THREADS, C::SMEM, s, p, qm, km, vm),
                "packed_attention_kernel launch");
  if (SPLIT)
    MEMOPT_LAUNCH(launch_after(join_pieces_kernel<T, D>, dim3(static_cast<unsigned>(pl.tile_slots), D / 16), 128, 0, s, p),
                  "join_pieces_kernel launch");
  return MEMOPT_OK;
}

template <typename T, int D>
int launch(const Params& p, int KVH, const Plan& pl, cudaStream_t s) {
  if (pl.split) return launch<T, D, 1, true>(p, KVH, pl, s);
  return pl.tiles == 1 ? launch<T, D, 1, false>(p, KVH, pl, s) : launch<T, D, 2, false>(p, KVH, pl, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace packed
}  // namespace memopt

using namespace memopt;

extern "C" size_t memopt_packed_attention_workspace_size(int num_seqs, int64_t total_tokens, int max_seqlen,
                                                         int num_heads, int num_kv_heads, int head_dim,
                                                         int window_size, int causal) {
  if (num_seqs <= 0 || total_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return static_cast<size_t>(packed::plan_of(num_seqs, total_tokens, max_seqlen, num_heads, num_kv_heads, head_dim,
                                             window_size, causal != 0)
                                 .workspace);
}

extern "C" int memopt_packed_attention(const void* query, int64_t query_stride, const void* keys, int64_t key_stride,
                                       const void* values, int64_t value_stride, int dtype, const int32_t* cu_seqlens,
                                       int num_seqs, int64_t total_tokens, int max_seqlen, int num_heads,
                                       int num_kv_heads, int head_dim, int window_size, int causal, void* out,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  return memopt_packed_attention_ex(query, query_stride, keys, key_stride, values, value_stride, dtype, cu_seqlens,
                                    num_seqs, total_tokens, max_seqlen, num_heads, num_kv_heads, head_dim, window_size,
                                    causal, 0, out, workspace, workspace_bytes, stream);
}

extern "C" int memopt_packed_attention_ex(const void* query, int64_t query_stride, const void* keys,
                                          int64_t key_stride, const void* values, int64_t value_stride, int dtype,
                                          const int32_t* cu_seqlens, int num_seqs, int64_t total_tokens,
                                          int max_seqlen, int num_heads, int num_kv_heads, int head_dim,
                                          int window_size, int causal, int zero_rest, void* out, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  if (num_seqs < 0 || total_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(MEMOPT_ERR_INVALID_ARG, "packed_attention: invalid geometry");
  if (dtype != MEMOPT_DTYPE_F16 && dtype != MEMOPT_DTYPE_BF16)
    return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: dtype must be fp16 or bf16");
  if (head_dim != 64 && head_dim != 128)
    return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: head_dim must be 64 or 128");
  if (total_tokens > 0x7fffff00LL) return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: more than 2^31 tokens");
  if (total_tokens == 0 || (num_seqs == 0 && !zero_rest)) return MEMOPT_OK;
  if (num_seqs == 0) {  // no sequence: every row is behind the last one
    if (!out) return fail(MEMOPT_ERR_INVALID_ARG, "packed_attention: null pointer");
    const cudaError_t e = cudaMemsetAsync(out, 0, static_cast<size_t>(total_tokens) * num_heads * head_dim * 2,
                                          as_stream(stream));
    return e == cudaSuccess ? MEMOPT_OK : cuda_fail(e, "packed_attention");
  }
  if (!query || !keys || !values || !cu_seqlens || !out)
    return fail(MEMOPT_ERR_INVALID_ARG, "packed_attention: null pointer");
  if (!packed::aligned16(query) || !packed::aligned16(keys) || !packed::aligned16(values) ||
      !packed::aligned16(out) || (query_stride | key_stride | value_stride) % 8 != 0)
    return fail(MEMOPT_ERR_INVALID_ARG,
                "packed_attention: pointers must be 16-byte aligned and strides multiples of 8 elements");
  packed::Params p{};
  p.q = query, p.k = keys, p.v = values, p.out = out, p.cu = cu_seqlens;
  p.q_stride = query_stride, p.k_stride = key_stride, p.v_stride = value_stride;
  p.T = static_cast<int>(total_tokens), p.S = num_seqs, p.H = num_heads, p.group = num_heads / num_kv_heads;
  packed::Plan pl = packed::plan_of(num_seqs, total_tokens, max_seqlen, num_heads, num_kv_heads, head_dim, window_size,
                                    causal != 0);
  if (pl.split && (workspace == nullptr || workspace_bytes < static_cast<size_t>(pl.workspace)))
    return fail(MEMOPT_ERR_WORKSPACE, "packed_attention: workspace too small (need " + std::to_string(pl.workspace) +
                                          " bytes)");
  if (pl.split && !packed::aligned16(workspace))
    return fail(MEMOPT_ERR_INVALID_ARG, "packed_attention: workspace must be 16-byte aligned");
  p.gshift = pl.gshift, p.units = pl.units, p.split = pl.split, p.pieces = pl.pieces, p.whole = pl.whole;
  p.part_o = static_cast<float4*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + pl.tile_slots * pl.pieces * (head_dim / 4) * 128);
  p.window = window_size > 0 ? window_size : 0, p.causal = causal ? 1 : 0;
  p.zero_rest = zero_rest ? 1 : 0;
  p.qscale = (1.0f / sqrtf(static_cast<float>(head_dim))) * 1.4426950408889634f;
  // Head units per chunk: the chunk's keys and values fill about a quarter of L2.
  // Units that share a KV head stay together.
  const int per_kv = p.group >> p.gshift;
  const int64_t kv_bytes = total_tokens * head_dim * 4;
  p.chunk = static_cast<int>(std::min<int64_t>(p.units, per_kv * std::max<int64_t>(1, (int64_t(32) << 20) / kv_bytes)));
  if (pl.grid > 0x7fffffffLL) return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: too many work items");
  cudaStream_t s = as_stream(stream);
  if (dtype == MEMOPT_DTYPE_F16)
    return head_dim == 128 ? packed::launch<__half, 128>(p, num_kv_heads, pl, s)
                           : packed::launch<__half, 64>(p, num_kv_heads, pl, s);
  return head_dim == 128 ? packed::launch<__nv_bfloat16, 128>(p, num_kv_heads, pl, s)
                         : packed::launch<__nv_bfloat16, 64>(p, num_kv_heads, pl, s);
}
