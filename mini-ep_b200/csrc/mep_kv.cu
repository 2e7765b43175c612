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
//
// Measured: 16 x 1021 tokens of 32 + 8 + 8 heads of 128, bf16, normalised, into
// an e4m3 cache (370 MB): 96 us, 3.9 TB/s; issue is 0.6 busy with 43 % of the warps
// active, so what holds it is each head's chain (load, two reductions, a division,
// conversions). The same into a bf16 cache (418 MB) 94 us, 4.4 TB/s, fp32 into fp32
// (820 MB) 145 us, 5.7 TB/s. One token: 2.0 us, 64 tokens of 32 heads of 64: 3.0 us.
// Reading the same columns back (101 MB): 19 us, 5.4 TB/s.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <type_traits>

#include "mep_device.cuh"
#include "mep_serve.cuh"

namespace mep {
namespace {

constexpr float kE4M3Max = 448.f;
// a row whose largest magnitude is below this is stored as zeros: 448 / a
// would come near the end of the fp32 range
constexpr float kTinyRow = 7.888609e-31f;  // 2^-100

// 4 consecutive values of a row, as loaded and in fp32
template <typename T>
struct Raw4 {
  uint2 v;
  __device__ void load(const T* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ void get(float* x) const {
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};
template <>
struct Raw4<float> {
  float4 v;
  __device__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ void get(float* x) const { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
};
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* x) {
  Raw4<T> r;
  r.load(p);
  r.get(x);
}
__device__ __forceinline__ void store4(float* p, const float* x) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint32_t bf16x2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(bf16x2(x[0], x[1]), bf16x2(x[2], x[3]));
}
__device__ __forceinline__ void store4(__nv_fp8_storage_t* p, const float* x) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<uint32_t*>(p) = lo | hi << 16;
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  store4(p, x);
  store4(p + 4, x + 4);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16x2(x[0], x[1]), bf16x2(x[2], x[3]),
                                            bf16x2(x[4], x[5]), bf16x2(x[6], x[7]));
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

// sum / maximum over a row's group of lanes, in every lane. L: lanes of a
// group when that is a power of two, else 0 (n lanes, this one the j-th).
template <int L>
__device__ __forceinline__ float group_sum(float x, int j, int n, int first) {
  if constexpr (L != 0) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  } else {
    for (int o = 1; o < n; o <<= 1) {
      const float y = __shfl_down_sync(0xffffffffu, x, o);
      if (j + o < n) x += y;
    }
    return __shfl_sync(0xffffffffu, x, first);
  }
}
template <int L>
__device__ __forceinline__ float group_max(float x, int j, int n, int first) {
  if constexpr (L != 0) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
  } else {
    for (int o = 1; o < n; o <<= 1) {
      const float y = __shfl_down_sync(0xffffffffu, x, o);
      if (j + o < n) x = fmaxf(x, y);
    }
    return __shfl_sync(0xffffffffu, x, first);
  }
}

// A lane holds values 4j..4j+3 of a head row and the same of its other half,
// so that the rotation needs no exchange; D/8 lanes a row, 32 / (D/8) rows a
// pass of a warp, all q, all k or all v. A warp takes `share` passes of one
// token, the next pass's rows loaded while it works on this one's, the token's
// table rows in registers throughout. T: model type, C: cache element, W: type
// of the tables, LT: D/8 where that is a power of two, else 0.
template <typename T, typename C, typename W, int LT>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3)
    k_norm_rope_store(const StoreArgs a, int share, int parts) {
  const int D = a.head_dim, L = LT ? LT : D >> 3, half = D >> 1;
  const int per_warp = 32 / L, lane = lane_id();
  const int sub = lane / L, j = lane - sub * L, first = sub * L;
  const int qp = (a.q_heads + per_warp - 1) / per_warp;
  const int kp = (a.kv_heads + per_warp - 1) / per_warp;
  const int64_t item = (int64_t)blockIdx.x * (blockDim.x >> 5) + warp_id();
  const int64_t tok = item / parts;
  if (tok >= a.batch * a.tokens) return;
  const int p0 = (int)(item - tok * parts) * share, p1 = min(qp + 2 * kp, p0 + share);
  const int64_t b = tok / a.tokens, t = tok - b * a.tokens;
  const int64_t col = (a.col_dev ? *a.col_dev : a.col) + t;
  const bool stored = col >= 0 && col < a.capacity;
  float c[8], s[8];
  if (p0 < qp + kp) {
    const int64_t p = a.positions[b * a.psb + t * a.pst];
    if (p >= 0 && p < a.table_rows) {
      const W* cw = static_cast<const W*>(a.cos) + p * D + 4 * j;
      const W* sw = static_cast<const W*>(a.sin) + p * D + 4 * j;
      load4<W>(cw, c), load4<W>(cw + half, c + 4);
      load4<W>(sw, s), load4<W>(sw + half, s + 4);
    } else {  // no such position: NaN rather than a read outside the tables
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    }
  }

  // the warp's passes [p, end) over the heads of one of q, k and v (KIND 0, 1, 2)
  auto heads = [&](auto kind_tag, const HeadsView& in, int count, const void* norm, int p, int end) {
    constexpr int KIND = decltype(kind_tag)::value;
    if (p >= end) return;
    const T* x0 = static_cast<const T*>(in.p) + b * in.sb + t * in.st + 4 * j +
                  (int64_t)(p * per_warp + sub) * in.sh;
    const int64_t step = (int64_t)per_warp * in.sh;
    int h = p * per_warp + sub;  // this lane's head
    const bool lane_on = sub < per_warp;
    float w[8];
    if (KIND < 2 && norm) {
      const T* nw = static_cast<const T*>(norm) + (lane_on ? 4 * j : 0);
      load4<T>(nw, w), load4<T>(nw + half, w + 4);
    }
    // rows of this call: where they go, and how far the next pass's are
    T* q_to = nullptr;
    C* kv_to = nullptr;
    float* scale_to = nullptr;
    if (KIND == 0) {
      q_to = static_cast<T*>(a.q_out) + (tok * a.q_heads + h) * D + 4 * j;
    } else {
      const int64_t at = (b * a.kv_heads + h) * a.capacity + col;
      kv_to = static_cast<C*>(KIND == 1 ? a.kc : a.vc) + at * D + 4 * j;
      if (sizeof(C) == 1) scale_to = (KIND == 1 ? a.ks : a.vs) + at;
    }
    const int64_t kv_step = per_warp * a.capacity;
    Raw4<T> raw[2] = {};
    bool on = lane_on && h < count;
    if (on) raw[0].load(x0), raw[1].load(x0 + half);
    for (; p < end; ++p) {
      float x[8];
      raw[0].get(x);
      raw[1].get(x + 4);
      x0 += step;
      h += per_warp;
      const bool next = lane_on && h < count;
      if (p + 1 < end && next) raw[0].load(x0), raw[1].load(x0 + half);
      if (KIND < 2) {
        if (norm) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
          ss = group_sum<LT>(ss, j, L, first);
          const float r = rsqrtf(ss / (float)D + a.eps);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float lo = x[i], hi = x[i + 4];
          x[i] = lo * c[i] - hi * s[i];
          x[i + 4] = hi * c[i + 4] + lo * s[i + 4];
        }
      }
      if (KIND == 0) {
        if (on) {
          store4(q_to, x);
          store4(q_to + half, x + 4);
        }
        q_to += per_warp * D;
      } else {
        if (sizeof(C) == 1) {
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
          m = group_max<LT>(m, j, L, first);
          const bool some = m >= kTinyRow;
          // 448 / m in the row's first lane and m / 448 in its second: one
          // division an instruction for both
          const float d = (j & 1 ? m : kE4M3Max) / (j & 1 ? kE4M3Max : m);
          // every lane takes part, whatever its row holds
          const float d0 = __shfl_sync(0xffffffffu, d, first & 31);
          const float inv = some ? d0 : 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= inv;
          if (on && stored && j == 1) *scale_to = some ? d : 0.f;
          scale_to += kv_step;
        }
        if (on && stored) {
          store4(kv_to, x);
          store4(kv_to + half, x + 4);
        }
        kv_to += kv_step * D;
      }
      on = next;
    }
  };
  heads(std::integral_constant<int, 0>(), a.q, a.q_heads, a.q_norm, p0, min(p1, qp));
  heads(std::integral_constant<int, 1>(), a.k, a.kv_heads, a.k_norm, max(p0 - qp, 0),
        min(p1 - qp, kp));
  heads(std::integral_constant<int, 2>(), a.v, a.kv_heads, nullptr, max(p0 - qp - kp, 0),
        p1 - qp - kp);
}

template <typename T, typename C, typename W, int LT>
void launch_store_l(const StoreArgs& a, cudaStream_t st) {
  const int per_warp = 32 / (a.head_dim / 8);
  const int passes = (a.q_heads + per_warp - 1) / per_warp + 2 * ((a.kv_heads + per_warp - 1) / per_warp);
  const int64_t tokens = a.batch * a.tokens;
  // few tokens: one pass a warp, for the latency (64 tokens of 48 heads of 128,
  // bf16: 4.1 us against 8.1); many (32 warps on each of 148 SMs, four passes
  // each): all of a token's up to 12, else half of them, which share the table
  // rows (16 x 1021 such tokens 96 us, 197 with one pass a warp). Half against all
  // of 24 passes: 1024 tokens 8.2 us against 10.3, 8 x 1021 53.3 against 51.3; of 8
  // passes: 8 x 1021 18.5 against 16.4.
  const int share = tokens * passes < (int64_t)148 * 32 * 4 ? 1 : passes <= 12 ? passes : (passes + 1) / 2;
  const int parts = (passes + share - 1) / share;
  const int warps = share == 1 ? 4 : 8;
  k_norm_rope_store<T, C, W, LT>
      <<<(unsigned)((tokens * parts + warps - 1) / warps), warps * 32, 0, st>>>(a, share, parts);
}
template <typename T, typename C, typename W>
void launch_store_w(const StoreArgs& a, cudaStream_t st) {
  if (a.head_dim == 64)
    launch_store_l<T, C, W, 8>(a, st);
  else if (a.head_dim == 128)
    launch_store_l<T, C, W, 16>(a, st);
  else
    launch_store_l<T, C, W, 0>(a, st);
}
template <typename T, typename C>
void launch_store(const StoreArgs& a, int table_f32, cudaStream_t st) {
  if (table_f32)
    launch_store_w<T, C, float>(a, st);
  else
    launch_store_w<T, C, T>(a, st);
}

// columns [start, start + n) of a quantised layer, code * scale rounded once:
// 16 codes a thread (one 16-byte load), K and V of a head (blockIdx.y, z)
template <typename T>
__global__ void __launch_bounds__(256) k_kv_read(CacheView c, int64_t heads, int D,
                                                 int64_t start, int64_t n, T* k_out, T* v_out) {
  const unsigned per_row = (unsigned)D >> 4;
  const unsigned kv = blockIdx.y;
  const unsigned pieces = (unsigned)n * per_row;
  for (int64_t bh = blockIdx.z; bh < heads; bh += gridDim.z) {
    const uint8_t* codes =
        static_cast<const uint8_t*>(kv ? c.v : c.k) + (bh * c.capacity + start) * D;
    const float* scales = (kv ? c.vs : c.ks) + bh * c.capacity + start;
    T* out = (kv ? v_out : k_out) + bh * n * D;
    for (unsigned i = blockIdx.x * blockDim.x + threadIdx.x; i < pieces;
         i += gridDim.x * blockDim.x) {
      const float scale = scales[i / per_row];
      const uint4 u = reinterpret_cast<const uint4*>(codes)[i];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      float x[2][8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t two = q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xffff;
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        x[q >> 2][(2 * q) & 7] = f.x * scale;
        x[q >> 2][(2 * q + 1) & 7] = f.y * scale;
      }
      store8(out + (size_t)i * 16, x[0]);
      store8(out + (size_t)i * 16 + 8, x[1]);
    }
  }
}

}  // namespace
}  // namespace mep

using namespace mep;

extern "C" int mep_norm_rope_store(const mep_store_args* x, void* stream) {
  const char* op = "mep_norm_rope_store";
  if (!x) return serve_invalid(op, "null arguments");
  if (const char* why = bad_heads(x->dtype, x->cache_dtype, x->batch, x->tokens, x->q_heads,
                                  x->kv_heads, x->head_dim))
    return serve_invalid(op, why);
  if (x->table_dtype != MEP_F32 && x->table_dtype != x->dtype)
    return serve_invalid(op, "the rotation tables must be fp32 or in the model dtype");
  if (x->capacity < 0) return serve_invalid(op, "negative capacity");
  if (!x->col_dev && (x->col < 0 || x->col > x->capacity - x->tokens))
    return serve_invalid(op, "columns [col, col + tokens) do not fit the cache");
  if (x->batch == 0 || x->tokens == 0) return MEP_OK;
  const StoreArgs a{x->batch, x->tokens, (int)x->q_heads, (int)x->kv_heads, (int)x->head_dim,
                    {x->q, x->q_sb, x->q_st, x->q_sh}, {x->k, x->k_sb, x->k_st, x->k_sh},
                    {x->v, x->v_sb, x->v_st, x->v_sh}, x->q_norm, x->k_norm, (float)x->eps, x->cos,
                    x->sin, x->table_rows, x->positions, x->p_sb, x->p_st, x->q_out, x->k_cache,
                    x->v_cache, x->k_scale, x->v_scale, x->capacity, x->col, x->col_dev};
  if (!x->q || !x->k || !x->v || !x->cos || !x->sin || !x->positions || !x->q_out ||
      !x->k_cache || !x->v_cache)
    return serve_invalid(op, "null tensor");
  if (x->cache_dtype == MEP_E4M3 && (!x->k_scale || !x->v_scale))
    return serve_invalid(op, "a quantised cache needs k_scale and v_scale");
  const int elt = x->dtype == MEP_BF16 ? 2 : 4;
  if (bad_strides(a.q, elt) || bad_strides(a.k, elt) || bad_strides(a.v, elt) ||
      !aligned16(x->cos) || !aligned16(x->sin) || !aligned16(x->q_norm) || !aligned16(x->k_norm) ||
      !aligned16(x->q_out) || !aligned16(x->k_cache) || !aligned16(x->v_cache))
    return serve_invalid(op, "tensors and row strides must be multiples of 16 bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int tf = x->table_dtype == MEP_F32;
  if (x->dtype == MEP_BF16) {
    if (x->cache_dtype == MEP_E4M3)
      launch_store<__nv_bfloat16, __nv_fp8_storage_t>(a, tf, st);
    else
      launch_store<__nv_bfloat16, __nv_bfloat16>(a, tf, st);
  } else {
    if (x->cache_dtype == MEP_E4M3)
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
  if (start < 0 || columns < 0 || capacity < 0 || columns > capacity - start)
    return serve_invalid(op, "columns outside the cache");
  if (batch == 0 || columns == 0) return MEP_OK;
  if (!k_cache || !v_cache || !k_scale || !v_scale || !k_out || !v_out)
    return serve_invalid(op, "null tensor");
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_out) || !aligned16(v_out))
    return serve_invalid(op, "tensors must start on a 16-byte boundary");
  const int64_t heads = batch * kv_heads;
  if (columns * head_dim > 0xffffffffll) return serve_invalid(op, "columns * head_dim up to 2^32 - 1");
  const int64_t pieces = columns * (head_dim / 16);
  const int64_t most = 148 * 64 / heads + 1;  // CTAs of a head: some 64 an SM in all
  const int64_t want = (pieces + 255) / 256;
  const dim3 grid((unsigned)(want < most ? want : most), 2,
                  (unsigned)(heads < 65535 ? heads : 65535));
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
