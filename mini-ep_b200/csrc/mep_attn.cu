// Attention of the new tokens over the key/value cache.
//
// Query (b, t, h) attends to every column of the shared prefix (if any) and to
// the own columns c of row b with c <= col + t and (c < lengths[b] or
// c >= prompt_cols):
//   s = scale * q.k, out = sum exp(s - m) v / sum exp(s - m), m = max s,
// in fp32, rounded once to the model dtype; zeros where nothing is visible.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "mep_device.cuh"
#include "mep_serve.cuh"

namespace mep {
namespace {

struct AttnArgs {
  int64_t batch, tokens;
  int q_heads, kv_heads, head_dim;
  HeadsView q;
  CacheView c;
  const int64_t* lengths;
  int64_t prompt_cols, col;
  const int64_t* col_dev;
  const void* kp;
  const void* vp;
  int64_t prefix_cols;
  float scale;
  void* out;
};

template <typename C>
__device__ __forceinline__ float elt(const void* p, int64_t i) {
  return Elt<C>::to_f(static_cast<const C*>(p)[i]);
}
template <>
__device__ __forceinline__ float elt<uint8_t>(const void* p, int64_t i) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(p)[i], __NV_E4M3)));
}

// one warp per query head; the lanes share the head's values
template <typename T, typename C>
__global__ void __launch_bounds__(128) k_attn(const AttnArgs a) {
  const int lane = lane_id(), D = a.head_dim;
  const int64_t i = (int64_t)blockIdx.x * 4 + warp_id();
  if (i >= a.batch * a.tokens * a.q_heads) return;
  const int h = (int)(i % a.q_heads);
  const int64_t bt = i / a.q_heads, b = bt / a.tokens, t = bt - b * a.tokens;
  const int kh = h / (a.q_heads / a.kv_heads);
  const int64_t col = a.col_dev ? *a.col_dev : a.col;
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.sb + t * a.q.st + h * a.q.sh;
  float x[4] = {}, o[4] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < D) x[e] = Elt<T>::to_f(q[lane + 32 * e]);
  auto see = [&](auto tag, const void* k, const void* v, int64_t row, float ks, float vs) {
    using E = decltype(tag);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < D) s += x[e] * elt<E>(k, row * D + lane + 32 * e);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= ks * a.scale;
    const float mn = fmaxf(m, s), keep = expf(m - mn), p = expf(s - mn);
    m = mn;
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < D) o[e] = o[e] * keep + p * vs * elt<E>(v, row * D + lane + 32 * e);
  };
  for (int64_t c = 0; c < a.prefix_cols; ++c)
    see(T{}, a.kp, a.vp, kh * a.prefix_cols + c, 1.f, 1.f);
  const int64_t end = min(col + t + 1, a.c.capacity);
  const int64_t len = a.lengths ? a.lengths[b] : end;
  for (int64_t c = 0; c < end; ++c) {
    if (c >= len && c < a.prompt_cols) continue;
    const int64_t row = (b * a.kv_heads + kh) * a.c.capacity + c;
    see(C{}, a.c.k, a.c.v, row, sizeof(C) == 1 ? a.c.ks[row] : 1.f,
        sizeof(C) == 1 ? a.c.vs[row] : 1.f);
  }
  T* out = static_cast<T*>(a.out) + i * D;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < D) out[lane + 32 * e] = Elt<T>::from_f(l > 0.f ? o[e] / l : 0.f);
}

}  // namespace
}  // namespace mep

using namespace mep;

extern "C" int mep_cache_attention_workspace(int dtype, int cache_dtype, int64_t batch,
                                             int64_t tokens, int q_heads, int kv_heads,
                                             int head_dim, int64_t capacity, int64_t col,
                                             int64_t prefix_cols, int64_t* bytes_out) {
  const char* op = "mep_cache_attention_workspace";
  if (const char* why = bad_heads(dtype, cache_dtype, batch, tokens, q_heads, kv_heads, head_dim))
    return serve_invalid(op, why);
  if (capacity < 0 || prefix_cols < 0) return serve_invalid(op, "negative columns");
  if (!bytes_out) return serve_invalid(op, "bytes_out is required");
  (void)col;
  *bytes_out = 0;
  return MEP_OK;
}

extern "C" int mep_cache_attention(int dtype, int cache_dtype, int64_t batch, int64_t tokens,
                                   int q_heads, int kv_heads, int head_dim, const void* q,
                                   int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k_cache,
                                   const void* v_cache, const float* k_scale, const float* v_scale,
                                   int64_t capacity, const int64_t* lengths, int64_t prompt_cols,
                                   int64_t col, const int64_t* col_dev, const void* k_prefix,
                                   const void* v_prefix, int64_t prefix_cols, float scale,
                                   void* out, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  const char* op = "mep_cache_attention";
  if (const char* why = bad_heads(dtype, cache_dtype, batch, tokens, q_heads, kv_heads, head_dim))
    return serve_invalid(op, why);
  if (capacity < 0 || prefix_cols < 0 || prompt_cols < 0)
    return serve_invalid(op, "negative columns");
  if (!col_dev && (col < 0 || col + tokens > capacity))
    return serve_invalid(op, "columns [col, col + tokens) do not fit the cache");
  if (batch == 0 || tokens == 0) return MEP_OK;
  AttnArgs a{batch, tokens, q_heads, kv_heads, head_dim, {q, q_sb, q_st, q_sh},
             {k_cache, v_cache, k_scale, v_scale, capacity}, lengths, prompt_cols, col, col_dev,
             k_prefix, v_prefix, prefix_cols, scale, out};
  if (!q || !k_cache || !v_cache || !out) return serve_invalid(op, "null tensor");
  if (prefix_cols > 0 && (!k_prefix || !v_prefix)) return serve_invalid(op, "null prefix");
  if (cache_dtype == MEP_E4M3 && (!k_scale || !v_scale))
    return serve_invalid(op, "a quantised cache needs k_scale and v_scale");
  if (bad_strides(a.q, dtype == MEP_BF16 ? 2 : 4) || !aligned16(k_cache) || !aligned16(v_cache) ||
      !aligned16(k_prefix) || !aligned16(v_prefix) || !aligned16(out))
    return serve_invalid(op, "tensors and row strides must be multiples of 16 bytes");
  (void)workspace, (void)workspace_bytes;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((batch * tokens * q_heads + 3) / 4);
  if (dtype == MEP_BF16) {
    if (cache_dtype == MEP_E4M3)
      k_attn<__nv_bfloat16, uint8_t><<<grid, 128, 0, st>>>(a);
    else
      k_attn<__nv_bfloat16, __nv_bfloat16><<<grid, 128, 0, st>>>(a);
  } else {
    if (cache_dtype == MEP_E4M3)
      k_attn<float, uint8_t><<<grid, 128, 0, st>>>(a);
    else
      k_attn<float, float><<<grid, 128, 0, st>>>(a);
  }
  return serve_launched(op);
}
