// rotary.cu — rotary positions with several axes, fused with the cache write.
//
// A head of D dims has P rotary pairs (dims 2P..D-1 pass through).  Pair i
// belongs to axis a(i) (the sections share the pairs out among the axes: time,
// height, width; one axis for plain text) and turns by position[a(i)][token] *
// inv_freq[i]:
//   (x, y) -> (x cos - y sin, x sin + y cos),
// with (x, y) = dims (i, i + P), or (2i, 2i + 1) when interleaved.
//
// Angles of far positions: fp32 would lose them (2^17 rad have a spacing of
// 2^-7).  The frequency is held as a 64-bit fraction of a turn, so the integer
// product with the position wraps modulo whole turns without rounding, and its
// top 32 bits are the angle (error below 2^-24 of a half turn).  inv_freq is
// fp64, so the fraction itself is off by 2^-52 of the frequency.
//
// Everything is held in fp32 and rounded once per output.  Bound by HBM: q and
// k read and written once, v read once, the K and V rows written to the pool.
// A lane owns 16 dims of a head (two 16-byte vectors holding 8 whole pairs),
// D/16 lanes a head, a warp 512 / D heads at a time (a step).  A CTA takes a few
// tokens: its warps put their first loads in flight, the threads compute the
// (cos, sin) of the tokens' pairs once into shared memory, and every step reads
// them there.  Small CTAs of two warps, each with one batch of loads: on 32768
// tokens x 64 heads of 128 with the cache (1.88 GB) 297 to 339 us between boards
// (6.33 to 5.54 TB/s); on the fastest of them 297 against 306 to 349 us with four or eight warps, 2 to 4 steps in flight or up to four
// batches a warp; holding (cos, sin) in registers for all heads of a token and a
// grid of resident warps took 316 us (28.6 against 25.6 us on 4099 tokens).
#include <algorithm>

#include <cuda_bf16.h>

#include "common.cuh"

namespace memopt {
namespace {

constexpr int kWarps = 2;
constexpr int kMaxAxes = 4;
constexpr int kBatch = 4;  // steps whose loads a lane has in flight

struct RotaryArgs {
  const void *q, *k, *v;
  const int32_t* pos;   // [A, T]
  const double* freq;   // [P]
  const int32_t* slots;  // [T] or null: no cache write
  void *q_out, *k_out;
  __half *kc, *vc;
  int64_t T, q_stride, k_stride, v_stride;  // strides in elements
  int64_t num_slots;
  int H, KVH, P, axes;
  int steps, tokens;  // warp steps over a token's heads; tokens of a CTA
  int ends[kMaxAxes];  // axis a owns the pairs below ends[a] and from ends[a - 1] on
};

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Pair<T>::get(w[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Pair<T>::put(f[0], f[1]), Pair<T>::put(f[2], f[3]), Pair<T>::put(f[4], f[5]),
                    Pair<T>::put(f[6], f[7]));
}

// Both vectors of a lane's unit, rotated (in fp32); cs holds the (cos, sin) of
// its 8 pairs, two to a float4.
template <bool kInterleaved>
__device__ __forceinline__ void turn(float (&a)[8], float (&b)[8], const float4* cs) {
  auto one = [](float& x, float& y, float c, float s) {
    const float z = x;
    x = z * c - y * s;
    y = z * s + y * c;
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = cs[i];
    if (kInterleaved) {  // a holds pairs 0..3 of the unit, b pairs 4..7
      float(&x)[8] = i < 2 ? a : b;
      const int e = 4 * (i & 1);
      one(x[e], x[e + 1], v.x, v.y);
      one(x[e + 2], x[e + 3], v.z, v.w);
    } else {  // a holds the first dims of the 8 pairs, b the second ones
      one(a[2 * i], b[2 * i], v.x, v.y);
      one(a[2 * i + 1], b[2 * i + 1], v.z, v.w);
    }
  }
}

template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kWarps * 32) rotary_kernel(const __grid_constant__ RotaryArgs p) {
  constexpr int U = D / 16;    // units (lanes) per head
  constexpr int HPW = 32 / U;  // heads per warp step
  extern __shared__ float2 turns[];  // (cos, sin) of pair i of the CTA's k-th token at [k][i]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, u = lane % U, sub = lane / U;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.T - t0));
  const bool rotary = u < p.P / 8;
  // Dims of the unit's two vectors; units past the rotary ones cover the rest of the head.
  const int d0 = (!rotary || kInterleaved) ? 16 * u : 8 * u;
  const int d1 = (!rotary || kInterleaved) ? 16 * u + 8 : p.P + 8 * u;
  // Heads of a token: those of q, of k and, with a cache, of v (which only move).
  const int heads = p.H + p.KVH + (p.slots ? p.KVH : 0);
  const int all = tokens * p.steps;  // warp steps of the CTA

  uint4 ua[kBatch], ub[kBatch];
  auto load = [&](int st0) {  // a batch of this warp's steps: st0, st0 + kWarps, ...
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int st = st0 + i * kWarps, k = st / p.steps, h = (st - k * p.steps) * HPW + sub;
      if (st < all && h < heads) {
        const int64_t t = t0 + k;
        const T* src = h < p.H ? static_cast<const T*>(p.q) + t * p.q_stride + h * D
                       : h < p.H + p.KVH
                           ? static_cast<const T*>(p.k) + t * p.k_stride + (h - p.H) * D
                           : static_cast<const T*>(p.v) + t * p.v_stride + (h - p.H - p.KVH) * D;
        ua[i] = ld_once_v4(src + d0);
        ub[i] = ld_once_v4(src + d1);
      }
    }
  };
  begin_next();
  after_previous();
  load(warp);
  // The angles of the CTA's tokens while the first loads are in flight.
  for (int i = tid; i < tokens * p.P; i += kWarps * 32) {
    const int k = i / p.P, pair = i - k * p.P;
    int axis = 0;
    for (int a = 0; a + 1 < p.axes; ++a) axis += pair >= p.ends[a];
    const double f = p.freq[pair] * 0.15915494309189535;  // 1 / (2 pi)
    const uint64_t turn64 = static_cast<uint64_t>((f - floor(f)) * 18446744073709551616.0);
    const int64_t pos = p.pos[axis * p.T + t0 + k];
    const uint64_t w = static_cast<uint64_t>(pos) * turn64;
    float cs, sn;
    // the top 32 bits as a signed fraction of a turn, in half turns
    sincospif(static_cast<float>(static_cast<int32_t>(w >> 32)) * 4.656612873077393e-10f, &sn, &cs);
    turns[i] = make_float2(cs, sn);
  }
  __syncthreads();
  for (int st0 = warp; st0 < all; st0 += kBatch * kWarps) {
    if (st0 > warp) load(st0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int st = st0 + i * kWarps, k = st / p.steps, h = (st - k * p.steps) * HPW + sub;
      if (st >= all || h >= heads) continue;
      const int64_t t = t0 + k;
      const bool is_v = h >= p.H + p.KVH;
      float a[8], b[8];
      unpack8<T>(ua[i], a);
      unpack8<T>(ub[i], b);
      if (rotary && !is_v) turn<kInterleaved>(a, b, reinterpret_cast<const float4*>(turns + k * p.P + 8 * u));
      if (!is_v) {
        T* dst = h < p.H ? static_cast<T*>(p.q_out) + (t * p.H + h) * D
                         : static_cast<T*>(p.k_out) + (t * p.KVH + (h - p.H)) * D;
        *reinterpret_cast<uint4*>(dst + d0) = pack8<T>(a);
        *reinterpret_cast<uint4*>(dst + d1) = pack8<T>(b);
      }
      if (h >= p.H && p.slots) {
        const int64_t slot = p.slots[t];
        if (slot >= 0 && slot < p.num_slots) {
          __half* dst = is_v ? p.vc + (slot * p.KVH + (h - p.H - p.KVH)) * D : p.kc + (slot * p.KVH + (h - p.H)) * D;
          *reinterpret_cast<uint4*>(dst + d0) = pack8<__half>(a);
          *reinterpret_cast<uint4*>(dst + d1) = pack8<__half>(b);
        }
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int D>
int launch_rotary(const RotaryArgs& p, bool interleaved, int64_t ctas, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(ctas);
  const size_t smem = sizeof(float2) * p.tokens * p.P;
  auto kern = interleaved ? rotary_kernel<T, D, true> : rotary_kernel<T, D, false>;
  MEMOPT_LAUNCH(launch_after(kern, grid, kWarps * 32, smem, s, p), "rotary_kernel launch");
  return MEMOPT_OK;
}

}  // namespace
}  // namespace memopt

using namespace memopt;

extern "C" int memopt_rotary_write_cache(const void* query, int64_t query_stride, const void* keys, int64_t key_stride,
                                         const void* values, int64_t value_stride, int dtype, int64_t num_tokens,
                                         int num_heads, int num_kv_heads, int head_dim, const int32_t* positions,
                                         int num_axes, const int32_t* sections, const double* inv_freq, int num_pairs,
                                         int interleaved, void* query_out, void* keys_out,
                                         const int32_t* slot_mapping, void* key_pool, void* value_pool,
                                         int64_t num_blocks, int block_size, void* stream) {
  if (num_tokens < 0 || num_heads < 0 || num_kv_heads < 0 || num_heads + num_kv_heads <= 0)
    return fail(MEMOPT_ERR_INVALID_ARG, "rotary: invalid geometry");
  if (dtype != MEMOPT_DTYPE_F16 && dtype != MEMOPT_DTYPE_BF16)
    return fail(MEMOPT_ERR_UNSUPPORTED, "rotary: dtype must be fp16 or bf16");
  if (head_dim != 64 && head_dim != 128) return fail(MEMOPT_ERR_UNSUPPORTED, "rotary: head_dim must be 64 or 128");
  if (num_pairs <= 0 || num_pairs % 8 != 0 || 2 * num_pairs > head_dim)
    return fail(MEMOPT_ERR_UNSUPPORTED, "rotary: the number of pairs must be a multiple of 8, at most head_dim / 2");
  if (num_axes < 1 || num_axes > kMaxAxes || !sections)
    return fail(MEMOPT_ERR_UNSUPPORTED, "rotary: between 1 and 4 axes");
  RotaryArgs p{};
  int end = 0;
  for (int a = 0; a < num_axes; ++a) {
    if (sections[a] < 0 || sections[a] > num_pairs)
      return fail(MEMOPT_ERR_INVALID_ARG, "rotary: a section is negative or larger than the number of pairs");
    end += sections[a];
    p.ends[a] = end;
  }
  if (end != num_pairs) return fail(MEMOPT_ERR_INVALID_ARG, "rotary: the sections do not sum to the number of pairs");
  if (num_tokens == 0) return MEMOPT_OK;
  const bool cache = slot_mapping != nullptr;
  if (!positions || !inv_freq || (num_heads > 0 && (!query || !query_out)) ||
      (num_kv_heads > 0 && (!keys || !keys_out)) || (cache && num_kv_heads > 0 && (!values || !key_pool || !value_pool)))
    return fail(MEMOPT_ERR_INVALID_ARG, "rotary: null pointer");
  if (cache && (num_blocks < 0 || block_size <= 0)) return fail(MEMOPT_ERR_INVALID_ARG, "rotary: invalid pool geometry");
  if (!aligned16(query) || !aligned16(keys) || !aligned16(values) || !aligned16(query_out) || !aligned16(keys_out) ||
      !aligned16(key_pool) || !aligned16(value_pool) || (query_stride | key_stride | value_stride) % 8 != 0)
    return fail(MEMOPT_ERR_INVALID_ARG, "rotary: pointers must be 16-byte aligned and strides multiples of 8 elements");
  p.q = query, p.k = keys, p.v = values;
  p.q_stride = query_stride, p.k_stride = key_stride, p.v_stride = value_stride;
  p.pos = positions, p.freq = inv_freq, p.slots = slot_mapping;
  p.q_out = query_out, p.k_out = keys_out;
  p.kc = static_cast<__half*>(key_pool), p.vc = static_cast<__half*>(value_pool);
  p.T = num_tokens, p.num_slots = cache ? num_blocks * block_size : 0;
  p.H = num_heads, p.KVH = num_kv_heads, p.P = num_pairs, p.axes = num_axes;
  const int hpw = 512 / head_dim, heads = num_heads + num_kv_heads * (cache ? 2 : 1);
  p.steps = (heads + hpw - 1) / hpw;
  p.tokens = std::max(1, kBatch * kWarps / p.steps);
  const int64_t grid = (num_tokens + p.tokens - 1) / p.tokens;
  if (grid > 0x7fffffffLL) return fail(MEMOPT_ERR_UNSUPPORTED, "rotary: too many tokens");
  cudaStream_t s = as_stream(stream);
  const bool il = interleaved != 0;
  if (dtype == MEMOPT_DTYPE_F16)
    return head_dim == 128 ? launch_rotary<__half, 128>(p, il, grid, s) : launch_rotary<__half, 64>(p, il, grid, s);
  return head_dim == 128 ? launch_rotary<__nv_bfloat16, 128>(p, il, grid, s)
                         : launch_rotary<__nv_bfloat16, 64>(p, il, grid, s);
}
