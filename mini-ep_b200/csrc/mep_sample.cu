// Sampling the next token of each row from its logits.
//
// Tokens are ordered by (logit descending, id ascending), w = exp((l - lmax) /
// temperature). Kept: ranks below top_k; of those, the ranks whose preceding
// mass is below top_p times their whole mass; of those, w >= min_p. The token is
// the first id, ascending, whose running sum of kept weights exceeds u times
// their sum. The best token is always kept; temperature 0 takes it. A NaN
// logit counts as -inf; several +inf logits share the mass.
//
// Whether a token is drawn is decided at borders of running sums, so the
// weights are held as 64-bit fixed-point numbers (scaled so that a row's sum
// fits 62 bits): integer sums do not depend on their order, and the rounding
// of each weight, computed in 64 bits, is below 2^-44 of the best token's.
#include <cstdint>
#include <cuda_bf16.h>

#include "mep_device.cuh"
#include "mep_serve.cuh"

namespace mep {
namespace {

struct SampleArgs {
  const void* logits;
  int64_t vocab, stride;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s;
  int32_t top_k_s;
  float top_p_s, min_p_s;
  int64_t* tokens;
  float* logprobs;
};

using u64 = unsigned long long;

// order-preserving integer of a logit: NaN as -inf, -0 as +0
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) l = -INFINITY;
  l += 0.f;
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // key_of(-inf), the smallest

struct Row {
  float lmax, t;
  double one;  // fixed-point value of weight 1
  __device__ double weight(uint32_t key) const {
    const float l = logit_of(key);
    if (l == lmax) return 1.0;
    return t > 0.f ? exp(((double)l - (double)lmax) / (double)t) : 0.0;
  }
  __device__ u64 fixed(uint32_t key) const { return __double2ull_rn(weight(key) * one); }
};

template <int T>
__device__ u64 block_sum(u64 v, u64* buf) {
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane_id() == 0) buf[warp_id()] = v;
  __syncthreads();
  u64 s = 0;
  for (int i = 0; i < T / 32; ++i) s += buf[i];
  return s;
}

// One CTA per row. The top-k and top-p borders are found by building, bit by
// bit, the smallest key whose count (mass) above it is still below the limit.
template <typename T>
__global__ void __launch_bounds__(1024) k_sample(const SampleArgs a) {
  constexpr int NT = 1024;
  __shared__ u64 buf[32];
  __shared__ u64 scan_w[32], scan_c[32];
  const int64_t row = blockIdx.x, V = a.vocab;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const float temp = a.temperature ? a.temperature[row] : a.temperature_s;
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k_s;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_s;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_s;
  const int tid = threadIdx.x;
  auto key_at = [&](int64_t i) { return key_of(Elt<T>::to_f(x[i])); };

  // the best token: largest key, lowest id
  u64 best = 0;
  for (int64_t i = tid; i < V; i += NT) {
    const u64 c = (u64)key_at(i) << 32 | (uint32_t)~(uint32_t)i;
    best = c > best ? c : best;
  }
  __syncthreads();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if (lane_id() == 0) buf[warp_id()] = best;
  __syncthreads();
  for (int i = 0; i < NT / 32; ++i) best = buf[i] > best ? buf[i] : best;
  const uint32_t kmax = (uint32_t)(best >> 32);
  if (kmax == kKeyNegInf) {  // nothing to draw
    if (tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {
    if (tid == 0) {
      a.tokens[row] = (uint32_t)~(uint32_t)best;
      if (a.logprobs) a.logprobs[row] = 0.f;
    }
    return;
  }
  int bits = 0;
  while ((1ll << bits) < V) ++bits;
  const Row r{logit_of(kmax), temp, (double)(1ull << (62 - bits < 47 ? 62 - bits : 47))};

  // kept: keys above `edge`, and the first `ties` ids of key `edge`
  uint32_t edge = 0;
  u64 ties = ~0ull;
  if (top_k > 0 && top_k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t tryk = edge | (1u << bit);
      u64 n = 0;
      for (int64_t i = tid; i < V; i += NT) n += key_at(i) >= tryk;
      if (block_sum<NT>(n, buf) >= (u64)top_k) edge = tryk;
    }
    u64 n = 0;
    for (int64_t i = tid; i < V; i += NT) n += key_at(i) > edge;
    ties = (u64)top_k - block_sum<NT>(n, buf);
  }
  if (top_p < 1.f) {
    u64 w = 0, same = 0;
    for (int64_t i = tid; i < V; i += NT) {
      const uint32_t k = key_at(i);
      if (k > edge) w += r.fixed(k);
      same += k == edge;
    }
    const u64 above = block_sum<NT>(w, buf), eq = block_sum<NT>(same, buf);
    const u64 total = above + (eq < ties ? eq : ties) * r.fixed(edge);
    const double limit = (double)top_p * (double)total;
    // the smallest key at least one of whose tokens is kept: mass above it < limit
    uint32_t low = edge;
    if (!((double)above < limit)) {
      // largest key whose mass at or above it reaches the limit
      uint32_t k2 = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t tryk = k2 | (1u << bit);
        u64 s = 0;
        for (int64_t i = tid; i < V; i += NT) {
          const uint32_t k = key_at(i);
          if (k >= tryk) s += r.fixed(k);
        }
        if ((double)block_sum<NT>(s, buf) >= limit) k2 = tryk;
      }
      low = k2 > kmax ? kmax : k2;  // limit <= 0 or NaN: the best key alone
      ties = ~0ull;
    }
    u64 s = 0;
    for (int64_t i = tid; i < V; i += NT) {
      const uint32_t k = key_at(i);
      if (k > low) s += r.fixed(k);
    }
    const u64 mass = block_sum<NT>(s, buf), w1 = r.fixed(low);
    if (w1 > 0) {
      const double n = ceil((limit - (double)mass) / (double)w1);
      const u64 m = n < 1.0 ? 1 : (u64)n;
      if (m < ties) ties = m;
    }
    edge = low;
  }
  // draw: running sums in id order, one tile of NT ids at a time
  u64 target = 0, total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    u64 run_w = 0, run_c = 0;
    for (int64_t base = 0; base < V; base += NT) {
      const int64_t i = base + tid;
      const uint32_t k = i < V ? key_at(i) : 0;
      u64 eq = k == edge && i < V, c = eq;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, c, o);
        if (lane_id() >= o) c += y;
      }
      __syncthreads();
      if (lane_id() == 31) scan_c[warp_id()] = c;
      __syncthreads();
      u64 before = run_c;
      for (int w = 0; w < warp_id(); ++w) before += scan_c[w];
      for (int w = 0; w < 32; ++w) run_c += scan_c[w];
      const bool in = i < V && (k > edge || (eq && before + c <= ties)) &&
                      (k == kmax || r.weight(k) >= (double)min_p);
      const u64 w1 = in ? r.fixed(k) : 0;
      u64 w = w1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane_id() >= o) w += y;
      }
      if (lane_id() == 31) scan_w[warp_id()] = w;
      __syncthreads();
      u64 sum = run_w + w;
      for (int q = 0; q < warp_id(); ++q) sum += scan_w[q];
      for (int q = 0; q < 32; ++q) run_w += scan_w[q];
      if (pass == 1 && w1 > 0 && sum > target && sum - w1 <= target) {
        a.tokens[row] = i;
        if (a.logprobs) a.logprobs[row] = (float)log((double)w1 / (double)total);
      }
    }
    if (pass == 0) {
      total = run_w;
      const double u = a.u[row];
      const double g = (u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0) * (double)total;
      target = (u64)g;
      if (target >= total) target = total - 1;  // u = 1: the last kept token
    }
  }
}

}  // namespace
}  // namespace mep

using namespace mep;

extern "C" int mep_sample(int dtype, const void* logits, int64_t rows, int64_t vocab,
                          int64_t stride, const float* u, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p,
                          float temperature_all, int32_t top_k_all, float top_p_all,
                          float min_p_all, int64_t* tokens, float* logprobs, void* stream) {
  const char* op = "mep_sample";
  if (dtype != MEP_F32 && dtype != MEP_BF16)
    return serve_invalid(op, "dtype must be MEP_F32 or MEP_BF16");
  if (rows < 0 || rows > 0x7fffffff) return serve_invalid(op, "rows out of range");
  if (vocab < 1 || vocab > (1 << 24)) return serve_invalid(op, "vocab must be 1..2^24");
  if (stride < 0) return serve_invalid(op, "negative row stride");
  if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY))
    return serve_invalid(op, "temperature must be finite and not negative");
  if (!top_k && top_k_all < 0) return serve_invalid(op, "top_k must not be negative");
  if (!top_p && !(top_p_all > 0.f)) return serve_invalid(op, "top_p must be positive");
  if (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f))
    return serve_invalid(op, "min_p must be in [0, 1]");
  if (rows == 0) return MEP_OK;
  if (!logits || !u || !tokens) return serve_invalid(op, "null tensor");
  const SampleArgs a{logits, vocab, stride, u, temperature, top_k, top_p, min_p, temperature_all,
                     top_k_all, top_p_all, min_p_all, tokens, logprobs};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MEP_BF16)
    k_sample<__nv_bfloat16><<<(unsigned)rows, 1024, 0, st>>>(a);
  else
    k_sample<float><<<(unsigned)rows, 1024, 0, st>>>(a);
  return serve_launched(op);
}
