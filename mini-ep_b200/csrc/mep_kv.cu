// Writing new tokens into the key/value cache and reading a quantised cache
// back.
//
// k_norm_rope_store, per head row x of D values, in fp32: an optional RMS norm
// over the head, y = x * rsqrt(mean(x^2) + eps) * w, then the rotation of the
// two halves by the token's position p,
//   r[i] = y[i] cos[p][i] - y[i+D/2] sin[p][i]
//   r[i+D/2] = y[i+D/2] cos[p][i+D/2] + y[i] sin[p][i+D/2];
// q's result is rounded once to the model dtype; k's goes to its cache column,
// v unrotated to the same one. A quantised cache holds e4m3 codes of
// x * (448 / a) and the fp32 scale a / 448, a the row's largest magnitude (448
// is the largest e4m3 value), quantised from the fp32 result: one rounding.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "mep_device.cuh"
#include "mep_serve.cuh"

namespace mep {
namespace {

constexpr float kE4M3Max = 448.f;
// a row whose largest magnitude is below this is stored as zeros: 448 / a
// would come near the end of the fp32 range
constexpr float kTinyRow = 7.888609e-31f;  // 2^-100

// 8 consecutive values of a row
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(__nv_fp8_storage_t* p, const float (&x)[8]) {
  uint32_t u[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]),
                                                 __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]),
                                                 __NV_SATFINITE, __NV_E4M3);
    u[i] = lo | hi << 16;
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
}

struct StoreArgs {
  int64_t batch, tokens;
  int q_heads, kv_heads, head_dim;
  HeadsView q, k, v;
  const void* q_norm;
  const void* k_norm;
  float eps;
  const void* cos;
  const void* sin;
  int64_t table_rows;
  const int64_t* positions;
  int64_t psb, pst;
  void* q_out;
  void* kc;
  void* vc;
  float* ks;
  float* vs;
  int64_t capacity, col;
  const int64_t* col_dev;
};

// sum / maximum over the `n` lanes of a row's group (lane `j` of it), in every lane
__device__ __forceinline__ float group_sum(float x, int j, int n, int first) {
  for (int o = 1; o < n; o <<= 1) {
    const float y = __shfl_down_sync(0xffffffffu, x, o);
    if (j + o < n) x += y;
  }
  return __shfl_sync(0xffffffffu, x, first);
}
__device__ __forceinline__ float group_max(float x, int j, int n, int first) {
  for (int o = 1; o < n; o <<= 1) {
    const float y = __shfl_down_sync(0xffffffffu, x, o);
    if (j + o < n) x = fmaxf(x, y);
  }
  return __shfl_sync(0xffffffffu, x, first);
}

// D/8 lanes per head row, 32 / (D/8) rows a warp. T: model type, C: cache
// element, W: type of the rotation tables.
template <typename T, typename C, typename W>
__global__ void __launch_bounds__(256) k_norm_rope_store(const StoreArgs a) {
  const int D = a.head_dim, L = D >> 3, half = L >> 1;
  const int per_warp = 32 / L, lane = lane_id();
  const int sub = lane / L, j = lane - sub * L, first = sub * L;
  const int heads = a.q_heads + 2 * a.kv_heads;
  const int64_t rows = a.batch * a.tokens * heads;
  const int64_t row = ((int64_t)blockIdx.x * (blockDim.x >> 5) + warp_id()) * per_warp + sub;
  const bool live = sub < per_warp && row < rows;
  const int64_t tok = live ? row / heads : 0;
  const int head = live ? (int)(row - tok * heads) : 0;
  const int64_t b = tok / a.tokens, t = tok - b * a.tokens;
  const int kind = head < a.q_heads ? 0 : head < a.q_heads + a.kv_heads ? 1 : 2;
  const int h = kind == 0 ? head : kind == 1 ? head - a.q_heads : head - a.q_heads - a.kv_heads;
  const HeadsView& in = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  float x[8] = {};
  if (live) load8<T>(static_cast<const T*>(in.p) + b * in.sb + t * in.st + h * in.sh + j * 8, x);
  const void* nw = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
  if (a.q_norm || a.k_norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
    ss = group_sum(ss, j, L, first);
    if (nw && live) {
      const float r = rsqrtf(ss / (float)D + a.eps);
      float w[8];
      load8<T>(static_cast<const T*>(nw) + j * 8, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
    }
  }
  const int other = first + (j < half ? j + half : j - half);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], other & 31);
  if (live && kind < 2) {
    const int64_t p = a.positions[b * a.psb + t * a.pst];
    if (p >= 0 && p < a.table_rows) {
      float c[8], s[8];
      load8<W>(static_cast<const W*>(a.cos) + p * D + j * 8, c);
      load8<W>(static_cast<const W*>(a.sin) + p * D + j * 8, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * c[i] + (j < half ? -y[i] : y[i]) * s[i];
    } else {  // no such position: NaN rather than a read outside the tables
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fffffff);
    }
  }
  if (live && kind == 0) {
    store8(static_cast<T*>(a.q_out) + (tok * a.q_heads + h) * D + j * 8, x);
  }
  const int64_t col = (a.col_dev ? *a.col_dev : a.col) + t;
  const bool keep = live && kind > 0 && col >= 0 && col < a.capacity;
  const int64_t at = ((b * a.kv_heads + h) * a.capacity + col);
  if (sizeof(C) == 1) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
    m = group_max(m, j, L, first);
    const bool some = m >= kTinyRow;
    const float inv = some ? kE4M3Max / m : 0.f;
    if (keep) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv;
      if (j == 0) (kind == 1 ? a.ks : a.vs)[at] = some ? m / kE4M3Max : 0.f;
    }
  }
  if (keep) store8(static_cast<C*>(kind == 1 ? a.kc : a.vc) + at * D + j * 8, x);
}

template <typename T, typename C>
void launch_store(const StoreArgs& a, int table_f32, cudaStream_t st) {
  const int per_warp = 32 / (a.head_dim / 8);
  const int64_t rows = a.batch * a.tokens * (a.q_heads + 2 * a.kv_heads);
  const unsigned grid = (unsigned)((rows + 8 * per_warp - 1) / (8 * per_warp));
  if (table_f32)
    k_norm_rope_store<T, C, float><<<grid, 256, 0, st>>>(a);
  else
    k_norm_rope_store<T, C, T><<<grid, 256, 0, st>>>(a);
}

// columns [start, start + n) of a quantised layer, code * scale rounded once:
// 8 values a thread, K and V in one launch (blockIdx.y)
template <typename T>
__global__ void __launch_bounds__(256) k_kv_read(CacheView c, int64_t heads, int D, int64_t start,
                                                 int64_t n, T* k_out, T* v_out) {
  const int per_row = D >> 3;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= heads * n * per_row) return;
  const int64_t row = i / per_row;
  const int j = (int)(i - row * per_row);
  const int64_t bh = row / n;
  const int64_t at = bh * c.capacity + start + (row - bh * n);
  const uint8_t* codes = static_cast<const uint8_t*>(blockIdx.y ? c.v : c.k);
  const float scale = (blockIdx.y ? c.vs : c.ks)[at];
  const uint2 u = *reinterpret_cast<const uint2*>(codes + at * D + j * 8);
  float x[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t w = q < 2 ? u.x : u.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        (__nv_fp8x2_storage_t)(q & 1 ? w >> 16 : w & 0xffff), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    x[2 * q] = f.x * scale;
    x[2 * q + 1] = f.y * scale;
  }
  store8((blockIdx.y ? v_out : k_out) + row * D + j * 8, x);
}

}  // namespace
}  // namespace mep

using namespace mep;

extern "C" int mep_norm_rope_store(
    int dtype, int cache_dtype, int64_t batch, int64_t tokens, int q_heads, int kv_heads,
    int head_dim, const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k,
    int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st,
    int64_t v_sh, const void* q_norm, const void* k_norm, float eps, const void* cos,
    const void* sin, int table_dtype, int64_t table_rows, const int64_t* positions, int64_t p_sb,
    int64_t p_st, void* q_out, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
    int64_t capacity, int64_t col, const int64_t* col_dev, void* stream) {
  const char* op = "mep_norm_rope_store";
  if (const char* why = bad_heads(dtype, cache_dtype, batch, tokens, q_heads, kv_heads, head_dim))
    return serve_invalid(op, why);
  if (table_dtype != MEP_F32 && table_dtype != dtype)
    return serve_invalid(op, "the rotation tables must be fp32 or in the model dtype");
  if (capacity < 0) return serve_invalid(op, "negative capacity");
  if (!col_dev && (col < 0 || col + tokens > capacity))
    return serve_invalid(op, "columns [col, col + tokens) do not fit the cache");
  if (batch == 0 || tokens == 0) return MEP_OK;
  StoreArgs a{batch, tokens, q_heads, kv_heads, head_dim, {q, q_sb, q_st, q_sh},
              {k, k_sb, k_st, k_sh}, {v, v_sb, v_st, v_sh}, q_norm, k_norm, eps, cos, sin,
              table_rows, positions, p_sb, p_st, q_out, k_cache, v_cache, k_scale, v_scale,
              capacity, col, col_dev};
  if (!q || !k || !v || !cos || !sin || !positions || !q_out || !k_cache || !v_cache)
    return serve_invalid(op, "null tensor");
  if (cache_dtype == MEP_E4M3 && (!k_scale || !v_scale))
    return serve_invalid(op, "a quantised cache needs k_scale and v_scale");
  const int elt = dtype == MEP_BF16 ? 2 : 4;
  if (bad_strides(a.q, elt) || bad_strides(a.k, elt) || bad_strides(a.v, elt) || !aligned16(cos) ||
      !aligned16(sin) || !aligned16(q_norm) || !aligned16(k_norm) || !aligned16(q_out) ||
      !aligned16(k_cache) || !aligned16(v_cache))
    return serve_invalid(op, "tensors and row strides must be multiples of 16 bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int tf = table_dtype == MEP_F32;
  if (dtype == MEP_BF16) {
    if (cache_dtype == MEP_E4M3)
      launch_store<__nv_bfloat16, __nv_fp8_storage_t>(a, tf, st);
    else
      launch_store<__nv_bfloat16, __nv_bfloat16>(a, tf, st);
  } else {
    if (cache_dtype == MEP_E4M3)
      launch_store<float, __nv_fp8_storage_t>(a, tf, st);
    else
      launch_store<float, float>(a, tf, st);
  }
  return serve_launched(op);
}

extern "C" int mep_kv_read(int dtype, int64_t batch, int kv_heads, int head_dim,
                           const void* k_cache, const void* v_cache, const float* k_scale,
                           const float* v_scale, int64_t capacity, int64_t start, int64_t columns,
                           void* k_out, void* v_out, void* stream) {
  const char* op = "mep_kv_read";
  if (const char* why = bad_heads(dtype, MEP_E4M3, batch, 1, kv_heads, kv_heads, head_dim))
    return serve_invalid(op, why);
  if (start < 0 || columns < 0 || start + columns > capacity)
    return serve_invalid(op, "columns outside the cache");
  if (batch == 0 || columns == 0) return MEP_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !k_out || !v_out)
    return serve_invalid(op, "null tensor");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out))
    return serve_invalid(op, "tensors must start on a 16-byte boundary");
  const int64_t heads = batch * kv_heads, n = heads * columns * (head_dim / 8);
  const dim3 grid((unsigned)((n + 255) / 256), 2);
  const CacheView c{k_cache, v_cache, k_scale, v_scale, capacity};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MEP_BF16)
    k_kv_read<__nv_bfloat16><<<grid, 256, 0, st>>>(c, heads, head_dim, start, columns,
                                                   static_cast<__nv_bfloat16*>(k_out),
                                                   static_cast<__nv_bfloat16*>(v_out));
  else
    k_kv_read<float><<<grid, 256, 0, st>>>(c, heads, head_dim, start, columns,
                                           static_cast<float*>(k_out), static_cast<float*>(v_out));
  return serve_launched(op);
}
