// packed.cu — attention over packed prompts of different lengths, with
// grouped heads (simple form: one warp per query row and head).
#include <algorithm>
#include <cmath>

#include <cuda_bf16.h>

#include "common.cuh"

namespace memopt {
namespace {

constexpr int kWarps = 8;

struct PackedArgs {
  const void *q, *k, *v;
  void* out;
  const int32_t* cu;
  int64_t q_stride, k_stride, v_stride;
  int T, S, H, group, window, causal;
  float qscale;
};

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) packed_simple_kernel(const PackedArgs p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(item / p.H), h = static_cast<int>(item % p.H);
  if (t >= p.T) return;
  int lo = 0, hi = p.S;  // the last s with cu[s] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int first = max(p.cu[lo], 0), last = min(p.cu[lo + 1], p.T);
  if (t < first || t >= last) return;
  const int end = p.causal ? t + 1 : last;
  const int begin = p.window > 0 && end - first > p.window ? end - p.window : first;
  const T* q = static_cast<const T*>(p.q) + t * p.q_stride + h * D;
  const T* k = static_cast<const T*>(p.k) + (h / p.group) * D;
  const T* v = static_cast<const T*>(p.v) + (h / p.group) * D;
  float qr[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qr[e] = to_f(q[lane + 32 * e]) * p.qscale;
    acc[e] = 0.f;
  }
  for (int j = begin; j < end; ++j) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += qr[e] * to_f(k[j * p.k_stride + lane + 32 * e]);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float mn = fmaxf(m, s), a = exp2f(m - mn), w = exp2f(s - mn);
    l = l * a + w;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + w * to_f(v[j * p.v_stride + lane + 32 * e]);
  }
  T* o = static_cast<T*>(p.out) + (static_cast<int64_t>(t) * p.H + h) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) o[lane + 32 * e] = from_f<T>(acc[e] / l);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace memopt

using namespace memopt;

extern "C" int memopt_packed_attention(const void* query, int64_t query_stride, const void* keys, int64_t key_stride,
                                       const void* values, int64_t value_stride, int dtype, const int32_t* cu_seqlens,
                                       int num_seqs, int64_t total_tokens, int max_seqlen, int num_heads,
                                       int num_kv_heads, int head_dim, int window_size, int causal, void* out,
                                       void* stream) {
  if (num_seqs < 0 || total_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(MEMOPT_ERR_INVALID_ARG, "packed_attention: invalid geometry");
  if (dtype != MEMOPT_DTYPE_F16 && dtype != MEMOPT_DTYPE_BF16)
    return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: dtype must be fp16 or bf16");
  if (head_dim != 64 && head_dim != 128)
    return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: head_dim must be 64 or 128");
  if (total_tokens > 0x7fffff00LL) return fail(MEMOPT_ERR_UNSUPPORTED, "packed_attention: more than 2^31 tokens");
  if (num_seqs == 0 || total_tokens == 0) return MEMOPT_OK;
  if (!query || !keys || !values || !cu_seqlens || !out)
    return fail(MEMOPT_ERR_INVALID_ARG, "packed_attention: null pointer");
  if (!aligned16(query) || !aligned16(keys) || !aligned16(values) || !aligned16(out) ||
      (query_stride | key_stride | value_stride) % 8 != 0)
    return fail(MEMOPT_ERR_INVALID_ARG,
                "packed_attention: pointers must be 16-byte aligned and strides multiples of 8 elements");
  PackedArgs p{query, keys, values, out, cu_seqlens, query_stride, key_stride, value_stride,
               static_cast<int>(total_tokens), num_seqs, num_heads, num_heads / num_kv_heads, window_size, causal,
               (1.0f / sqrtf(static_cast<float>(head_dim))) * 1.4426950408889634f};
  (void)max_seqlen;
  const int64_t items = total_tokens * num_heads;
  const int grid = static_cast<int>((items + kWarps - 1) / kWarps);
  cudaStream_t s = as_stream(stream);
  if (dtype == MEMOPT_DTYPE_F16) {
    if (head_dim == 128) packed_simple_kernel<__half, 128><<<grid, kWarps * 32, 0, s>>>(p);
    else packed_simple_kernel<__half, 64><<<grid, kWarps * 32, 0, s>>>(p);
  } else {
    if (head_dim == 128) packed_simple_kernel<__nv_bfloat16, 128><<<grid, kWarps * 32, 0, s>>>(p);
    else packed_simple_kernel<__nv_bfloat16, 64><<<grid, kWarps * 32, 0, s>>>(p);
  }
  MEMOPT_LAUNCH_CHECK("packed_attention launch");
  return MEMOPT_OK;
}
