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
// weights are held as 64-bit fixed-point numbers (the best token's is 2^46, or
// less where the row's sum would pass 62 bits): integer sums do not depend on
// their order, and a weight, computed in 64 bits, is off by half a unit.
//
// Measured, bf16 / fp32 logits: 256 rows of 100,003 with top_p 0.95 72 / 208
// us, unfiltered 53 / 104 us, with top_k 50 70 / 86 us, greedy 21 / 36 us; one
// row of 49,155 with top_k and top_p 16.4 us, greedy 6.2 us. Reading the logits
// would take 8 / 16 us at 256 rows: what bounds it is the work on every token
// (bf16, top_p: 51 warp instructions for 32 tokens, a shared-memory addition
// and a read among them) and 256 CTAs on 148 SMs, for a few rows the chain of
// passes between cluster barriers.
#include <cstdint>
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "mep_device.cuh"
#include "mep_serve.cuh"

namespace mep {
namespace {

namespace cg = cooperative_groups;

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

// ---- weights
// exp2 by table and polynomial (P. T. P. Tang, "Table-driven implementation of
// the exponential function in IEEE floating-point arithmetic", ACM TOMS 15(2),
// 1989): with (l - lmax) * 256 log2(e) / T = k + r, |r| <= 1/2, the weight is
// 2^(k >> 8) * 2^((k & 255) / 256) * e^(r ln2 / 256), the last factor to the
// fourth power of r ln2 / 256 <= 0.00136 (4e-17 left).
struct Weights {
  float lmax, lcut;   // logits below lcut weigh less than half a unit
  double top, c;      // lmax; 256 log2(e) / temperature
  int scale;          // weight 1 is 2^scale
  const double* tab;  // 2^(j / 256)
  // a call where a copy at every use would only fill the instruction cache
  __device__ u64 operator()(float l) const;
  __device__ __forceinline__ u64 inlined(float l) const {
    if (l == lmax) return 1ull << scale;
    if (!(l >= lcut)) return 0;
    constexpr double kMagic = 6755399441055744.0;        // 1.5 * 2^52: rounds to an integer
    constexpr double a1 = 0.693147180559945309417 / 256;  // ln 2 / 256
    const double d = (double)l - top;
    const double z = fma(d, c, kMagic);
    const int k = __double2loint(z);
    const double r = fma(d, c, kMagic - z);
    const double q = r * fma(r, fma(r, fma(r, a1 * a1 * a1 * a1 / 24, a1 * a1 * a1 / 6),
                                    a1 * a1 / 2), a1);
    const double t = tab[k & 255];
    const double w = fma(t, q, t);
    // times 2^((k >> 8) + scale) in the exponent field, then to an integer by
    // adding 2^52 (weights stay below 2^47)
    const double y = __hiloint2double(__double2hiint(w) + (((k >> 8) + scale) << 20),
                                      __double2loint(w));
    return (u64)__double_as_longlong(y + 4503599627370496.0) & 0xfffffffffffffull;
  }
};

__device__ __noinline__ u64 weight_call(float l, float lmax, float lcut, double top, double c,
                                        int scale, const double* tab) {
  return Weights{lmax, lcut, top, c, scale, tab}.inlined(l);
}
__device__ __forceinline__ u64 Weights::operator()(float l) const {
  return weight_call(l, lmax, lcut, top, c, scale, tab);
}

constexpr int kNT = 512;        // threads of a CTA
constexpr int kNW = kNT / 32;
constexpr int kBins = 1024;
constexpr int kList = 2048;     // candidates the leading CTA can finish alone
constexpr int kPer = kList / kNT;  // of them a thread
constexpr int kMaxCtas = 8;     // CTAs of a row

constexpr int kCodes = 4096;    // 16-bit logits told apart by the table

struct Shared {
  double tab[256];
  union {
    struct {
      uint32_t cnt[kBins], lo[kBins], hi[kBins];  // this CTA's histogram
      u64 tmass[kBins];                           // the row's
      uint32_t tcnt[kBins];
      alignas(16) u64 item[kList];
      u64 w[kList];
    };
    struct {
      uint32_t total[kCodes];  // tokens of each code in the row
      union {
        uint32_t mine[kCodes];  // in this CTA, until they are summed
        u64 weight[kCodes];     // a kept token's weight, by code
      };
    };
  };
  u64 wmass[kMaxCtas * kNW];     // of every warp of the row
  uint32_t wties[kMaxCtas * kNW];
  u64 best[kMaxCtas], zero[kMaxCtas];
  float lmax[kMaxCtas], lmin[kMaxCtas];
  u64 red[kNW], red2[kNW];
  uint32_t n_items;
  // results that one thread finds for all
  uint32_t r_bin, r_cnt, r_hi;
  u64 r_above, r_mass;
};

// 16 bytes of a row: ids from `id` on, NaN (which counts as -inf and is no
// minimum) outside [0, vocab)
template <typename T>
struct Vec {
  static constexpr int E = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z),
  x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ uint4 fetch(const T* row, int id, int vocab) {
  constexpr int E = Vec<T>::E;
  if (id >= 0 && id + E <= vocab) return *reinterpret_cast<const uint4*>(row + id);
  __align__(16) T x[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    x[i] = id + i >= 0 && id + i < vocab ? row[id + i] : Elt<T>::from_f(__int_as_float(0x7fffffff));
  return *reinterpret_cast<const uint4*>(x);
}

// largest and smallest of a piece into hi and lo; NaN is neither
__device__ __forceinline__ void extremes(const uint4& v, float (&hi)[1], float (&lo)[1]) {
  float x[4];
  unpack(v, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) hi[0] = fmaxf(hi[0], x[i]), lo[0] = fminf(lo[0], x[i]);
}
__device__ __forceinline__ void extremes(const uint4& v, __nv_bfloat162& hi, __nv_bfloat162& lo) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&u[i]);
    hi = __hmax2(hi, x), lo = __hmin2(lo, x);
  }
}
template <typename T>
struct Extremes {
  float hi[1] = {-INFINITY}, lo[1] = {INFINITY};
  __device__ float high() const { return hi[0]; }
  __device__ float low() const { return lo[0]; }
};
template <>
struct Extremes<__nv_bfloat16> {
  __nv_bfloat162 hi = __float2bfloat162_rn(-INFINITY), lo = __float2bfloat162_rn(INFINITY);
  __device__ float high() const { return fmaxf(__low2float(hi), __high2float(hi)); }
  __device__ float low() const { return fminf(__low2float(lo), __high2float(lo)); }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane_id() >= o) v += y;
  }
  return v;
}
// exclusive prefix over the CTA's threads, and the whole sum
__device__ __forceinline__ u64 block_scan(u64 v, u64* buf, u64& total) {
  const u64 inc = warp_scan(v);
  __syncthreads();
  if (lane_id() == 31) buf[warp_id()] = inc;
  __syncthreads();
  const u64 own = lane_id() < kNW ? buf[lane_id()] : 0;
  const u64 sums = warp_scan(own);
  total = __shfl_sync(0xffffffffu, sums, 31);
  return __shfl_sync(0xffffffffu, sums - own, warp_id()) + inc - v;
}

// descending sort of x[0..n), n a power of two from 32 on: by counting the
// larger ones where each thread has one value at most, else bitonic (64
// barriers, 6 us at 2048)
__device__ __noinline__ void sort_desc(u64* x, int n) {
  __syncthreads();
  if (n <= kNT) {
    const int i = threadIdx.x;
    u64 v = 0;
    int rank = 0;
    if (i < n) {
      v = x[i];
#pragma unroll 4
      for (int j = 0; j < n; j += 2) {
        const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(x + j);
        rank += (y.x > v || (y.x == v && j < i)) + (y.y > v || (y.y == v && j + 1 < i));
      }
    }
    __syncthreads();
    if (i < n) x[rank] = v;
    __syncthreads();
    return;
  }
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kNT) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const u64 p = x[a], q = x[b];
        if ((p < q) == ((a & k) == 0)) x[a] = q, x[b] = p;
      }
    }
  __syncthreads();
}

// A cluster of CTAs takes a row, each a run of its ids, each warp a run of
// that, so that sums over ids stay in order. The passes after the first read a
// short run from shared memory and a long one from L2 (a whole row in shared
// memory would take an SM for itself).
// Without a filter the weights are summed per warp, and the warp
// whose share holds the target finds the token. With top_k or top_p a
// histogram over the logits (counts, or masses) tells which bins can hold kept
// tokens. When those are few the leading CTA sorts and finishes them alone. Else it sorts the bin of the border, and the kept weights are summed
// per warp as without a filter. A bin too large for that, and a second border
// behind a wide top_k, are found by histograms over ever narrower key ranges.
// All sums are of integers: their order is free.
//
// 16-bit logits have few values: where those from lcut to lmax are at most
// kCodes (with all below 2^-9 in magnitude taken as one), the row's tokens are
// counted by value, one addition a token; the borders follow from the counts
// and a weight for each value, and the sums over ids read a table of the kept
// values' weights instead of computing 100,000 exponentials.
template <typename T>
__global__ void __launch_bounds__(kNT, 2) k_sample(const SampleArgs a, int cached) {
  constexpr int E = Vec<T>::E;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& S = *reinterpret_cast<Shared*>(smem_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int nc = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  // others' shared memory may be touched once they run: waited for behind the
  // first pass
  if (nc > 1) cluster.barrier_arrive();
  const int64_t row = blockIdx.x / nc;
  const int V = (int)a.vocab;
  const int tid = threadIdx.x, lane = lane_id(), warp = warp_id();
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const float temp = a.temperature ? a.temperature[row] : a.temperature_s;
  const int64_t top_k = a.top_k ? a.top_k[row] : a.top_k_s;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_s;
  const float min_p_given = a.min_p ? a.min_p[row] : a.min_p_s;
  const float min_p = min_p_given > 1.f ? 1.f : min_p_given;

  // 16-byte pieces of the row on the grid of its addresses; piece p holds the
  // ids from p * E - shift on. This CTA has [p0, p1), this warp [w0, w1).
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int pieces = (shift + V + E - 1) / E;
  const int per = (pieces + nc - 1) / nc;
  const int p0 = min(pieces, per * rank), p1 = min(pieces, p0 + per);
  const int per_w = ((p1 - p0 + kNW - 1) / kNW + 31) / 32 * 32;
  const int w0 = min(p1, p0 + per_w * warp), w1 = min(p1, w0 + per_w);

  uint4* kept = reinterpret_cast<uint4*>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);
  auto piece = [&](int p) { return cached ? kept[p - p0] : fetch<T>(x, p * E - shift, V); };
  // f(piece, first id) for this lane's pieces, two loads under way
  auto each_piece = [&](auto f) {
    for (int p = w0 + lane; p < w1; p += 64) {
      const uint4 a0 = piece(p);
      const uint4 a1 = p + 32 < w1 ? piece(p + 32) : make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN
      f(a0, p * E - shift);
      f(a1, (p + 32) * E - shift);
    }
  };
  // f(l, id) for this warp's ids
  auto each = [&](auto f) {
    each_piece([&](const uint4& v, int id0) {
      float l[E];
      unpack(v, l);
#pragma unroll
      for (int i = 0; i < E; ++i) f(l[i], id0 + i);
    });
  };

  // ---- the largest and the smallest logit
  constexpr bool kTable = sizeof(T) == 2;
  if (tid < 256) S.tab[tid] = exp2(tid / 256.0);
  if (kTable)
    for (int i = tid; i < kCodes; i += kNT) S.mine[i] = 0;
  if (tid == 0) S.n_items = 0;
  Extremes<T> ex;
  for (int p = w0 + lane; p < w1; p += 128) {  // four loads under way
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = p + 32 * i < w1 ? fetch<T>(x, (p + 32 * i) * E - shift, V)
                             : make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (cached && p + 32 * i < w1) kept[p + 32 * i - p0] = v[i];
      extremes(v[i], ex.hi, ex.lo);
    }
  }
  float lmax = ex.high(), lmin = ex.low();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lmax = fmaxf(lmax, __shfl_xor_sync(0xffffffffu, lmax, o));
    lmin = fminf(lmin, __shfl_xor_sync(0xffffffffu, lmin, o));
  }
  if (lane == 0) S.red[warp] = __float_as_uint(lmax), S.red2[warp] = __float_as_uint(lmin);
  __syncthreads();
  if (nc > 1) cluster.barrier_wait();  // every CTA of the row has begun
  if (tid < nc) {
    for (int i = 0; i < kNW; ++i) {
      lmax = fmaxf(lmax, __uint_as_float((uint32_t)S.red[i]));
      lmin = fminf(lmin, __uint_as_float((uint32_t)S.red2[i]));
    }
    Shared* to = cluster.map_shared_rank(&S, tid);
    to->lmax[rank] = lmax;
    to->lmin[rank] = lmin;
  }
  cluster.sync();
  for (int i = 0; i < nc; ++i) {
    lmax = fmaxf(lmax, S.lmax[i]);
    lmin = fminf(lmin, S.lmin[i]);
  }
  lmax += 0.f;
  const uint32_t kmax = key_of(lmax);
  if (kmax == kKeyNegInf) {  // nothing to draw
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {  // the best token of the lowest id
    int id0 = 0x7fffffff;
    each([&](float l, int id) {
      if (l == lmax) id0 = min(id0, id);
    });
    id0 = __reduce_min_sync(0xffffffffu, id0);
    if (lane == 0) S.red[warp] = (uint32_t)id0;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < kNW; ++i) id0 = min(id0, (int)S.red[i]);
      cluster.map_shared_rank(&S, 0)->best[rank] = (uint32_t)id0;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < nc; ++i) id0 = min(id0, (int)S.best[i]);
      a.tokens[row] = id0;
      if (a.logprobs) a.logprobs[row] = 0.f;
    }
    return;
  }
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  Weights W;
  W.lmax = lmax;
  // 34 temperatures below the best a weight is 2^-49; lmax = inf leaves only
  // its equals, -inf never weighs
  W.lcut = W.lmax == INFINITY ? W.lmax : fmaxf(W.lmax - 34.f * temp, -3.402823466e38f);
  W.top = W.lmax;
  W.c = 369.329930467574632284 / (double)temp;  // 256 log2(e)
  W.scale = min(46, 62 - bits);
  W.tab = S.tab;
  const double one = (double)(1ull << W.scale);
  // integer borders: w >= min_p * one, and mass < top_p * total, are w >= and <
  // their next integers
  auto ceiling = [&](double v) { return v > 0.0 ? (u64)ceil(v) : 0ull; };
  const u64 floor_p = ceiling((double)min_p * one);
  const bool by_k = top_k > 0 && top_k < V, by_p = top_p < 1.f;
  const double u = a.u[row];
  auto target_of = [&](u64 total) {
    const u64 t = (u64)((u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0) * (double)total);
    return t < total ? t : total - 1;  // u = 1: the last kept token
  };
  auto answer = [&](int64_t id, u64 w, u64 total) {
    a.tokens[row] = id;
    if (a.logprobs) a.logprobs[row] = (float)log((double)w / (double)total);
  };
  auto add_mass = [&](int b, u64 w) {  // 64-bit sum in two 32-bit halves, carry by hand
    const uint32_t lo = (uint32_t)w;
    const uint32_t old = atomicAdd(&S.lo[b], lo);
    atomicAdd(&S.hi[b], (uint32_t)(w >> 32) + (old + lo < old));
  };
  // the CTAs' histograms summed into everyone's tcnt / tmass
  auto join = [&] {
    cluster.sync();
    const int share = kBins / nc;
    for (int i = tid; i < share; i += kNT) {
      const int b = rank * share + i;
      uint32_t c = 0;
      u64 m = 0;
      for (int r = 0; r < nc; ++r) {
        const Shared* from = cluster.map_shared_rank(&S, r);
        c += from->cnt[b];
        m += (u64)from->hi[b] << 32 | 0ull;
        m += from->lo[b];
      }
      for (int r = 0; r < nc; ++r) {
        Shared* to = cluster.map_shared_rank(&S, r);
        to->tcnt[b] = c;
        to->tmass[b] = m;
      }
    }
    cluster.sync();
  };

  // weights below min_p's border weigh nothing (the best token's is 2^scale)
  auto floored = [&](u64 w) {
    return w < floor_p && w < 1ull << W.scale ? 0ull : w;
  };
  // ---- the draw: weigh(l) is a token's kept weight; of the tokens with
  // on_edge(l) the first `ties` ids weigh `wedge` each; mass and n_edge are
  // this thread's sums of them
  auto finish = [&](u64 mass, uint32_t n_edge, auto weigh, auto on_edge, u64 ties, u64 wedge) {
    mass = warp_sum(mass);
    n_edge = __reduce_add_sync(0xffffffffu, n_edge);
    if (lane < nc) {
      Shared* to = cluster.map_shared_rank(&S, lane);
      to->wmass[rank * kNW + warp] = mass;
      to->wties[rank * kNW + warp] = n_edge;
    }
    cluster.sync();
    // of every warp's run its share of the row's kept mass, `total`, and the ids
    // on the edge before it; the run that the target falls in is `owner`'s
    constexpr int PW = kMaxCtas * kNW / 32;
    u64 share[PW], sum = 0, start = 0;
    uint32_t t[PW], seen = 0, before = 0;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int j = lane * PW + i;
      share[i] = j < nc * kNW ? S.wmass[j] : 0;
      t[i] = j < nc * kNW ? S.wties[j] : 0;
      seen += t[i];
    }
    const uint32_t at0 = (uint32_t)warp_scan(seen) - seen;
    uint32_t at = at0;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      share[i] += min((u64)t[i], ties > at ? ties - at : 0) * wedge;
      at += t[i];
      sum += share[i];
    }
    const u64 inc = warp_scan(sum), total = __shfl_sync(0xffffffffu, inc, 31);
    const u64 target = target_of(total);
    u64 run0 = inc - sum;
    int owner = -1;
    at = at0;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      if (target >= run0 && target - run0 < share[i])
        owner = lane * PW + i, start = run0, before = at;
      run0 += share[i];
      at += t[i];
    }
    const uint32_t found = __ballot_sync(0xffffffffu, owner >= 0);
    if (!found) return;
    int src = __ffs(found) - 1;
    owner = __shfl_sync(0xffffffffu, owner, src);
    start = __shfl_sync(0xffffffffu, start, src);
    before = __shfl_sync(0xffffffffu, before, src);
    if (owner / kNW != rank) return;  // all warps of the CTA alike
    int r0 = min(p1, p0 + per_w * (owner % kNW)), r1 = min(p1, r0 + per_w);
    if (r1 - r0 > 64) {
      // a long run is dealt to all warps first: one warp alone took up to 50 us
      // for its 800 pieces, some 2 us for 32 of them
      const int part = ((r1 - r0 + kNW - 1) / kNW + 31) / 32 * 32;
      const int q0 = min(r1, r0 + part * warp), q1 = min(r1, q0 + part);
      u64 m = 0;
      uint32_t eq = 0;
      for (int p = q0 + lane; p < q1; p += 32) {
        float l[E];
        unpack(piece(p), l);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          m += weigh(l[i]);  // 0 on the edge
          eq += on_edge(l[i]);
        }
      }
      m = warp_sum(m);
      eq = __reduce_add_sync(0xffffffffu, eq);
      if (lane == 0) S.red[warp] = m, S.red2[warp] = eq;
      __syncthreads();
      m = lane < kNW ? S.red[lane] : 0;
      eq = lane < kNW ? (uint32_t)S.red2[lane] : 0;
      before += (uint32_t)warp_scan(eq) - eq;
      m += min((u64)eq, ties > before ? ties - before : 0) * wedge;
      start += warp_scan(m) - m;
      src = __ffs(__ballot_sync(0xffffffffu, target >= start && target - start < m)) - 1;
      if (warp != src) return;
      start = __shfl_sync(0xffffffffu, start, src);
      before = __shfl_sync(0xffffffffu, before, src);
      r0 = q0, r1 = q1;
    } else if (warp != owner % kNW) {
      return;
    }
    for (int p = r0; p < r1; p += 32) {
      float l[E];
      const bool have = p + lane < r1;
      if (have) unpack(piece(p + lane), l);
      u64 w[E], sum = 0;
      uint32_t eq = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) eq += have && on_edge(l[i]);
      u64 nth = before + warp_scan(eq) - eq;  // ids on the edge before this lane's
      before += __reduce_add_sync(0xffffffffu, eq);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        w[i] = have ? weigh(l[i]) : 0;
        if (have && on_edge(l[i])) w[i] = nth++ < ties ? wedge : 0;
        sum += w[i];
      }
      u64 run = warp_scan(sum);
      const u64 step = __shfl_sync(0xffffffffu, run, 31);
      run += start - sum;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (run <= target && run + w[i] > target)
          answer((p + lane) * E - shift + i, w[i], total);
        run += w[i];
      }
      start += step;
      if (start > target) return;
    }
  };

  if constexpr (kTable) {
    // ---- a slot for each 16-bit value from 2^-9 to 2^7 in magnitude: kHalf of
    // either sign in the order of their bits. The last of each sign takes all
    // that has none (what the table is used for leaves no positive one there,
    // and negative ones there weigh nothing). By rank, best first: positive
    // ones from lmax down, all smaller ones as one, negative ones.
    constexpr int kSmall = (127 - 9) << 7, kHalf = kCodes / 2;
    const int top_mag = __float_as_int(W.lmax) >> 16 & 0x7fff;
    const bool neg = W.lmax < 0.f && top_mag >= kSmall;  // all negative, none small
    const int n_pos = W.lmax < 0.f ? 0 : max(top_mag - kSmall + 1, 0);
    const int cut_mag = __float_as_int(W.lcut) >> 16 & 0x7fff;
    const bool fits = top_mag < kSmall + kHalf - 1 &&
                      (W.lcut >= 0.f || cut_mag < kSmall + kHalf - 1);
    // a few tokens by top_k are sooner on one CTA's list (15 us against 20 for a
    // row of 49,155, 22 against 29 for 64; alike at 256 x 100003), short runs
    // without a border by their exponentials (11.9 against 12.3 us at 2000 ids a
    // CTA, 15.8 against 14.5 at 6000). The row's CTAs have to choose alike, as
    // the two ways meet at different barriers: `per` is the same in all of them,
    // the last one's own run may be shorter.
    const bool brief = by_k ? top_k <= 128 : !by_p && per * E < 4096;
    if (fits && !brief) {
      auto slot_of = [&](uint32_t u, int high) {  // of a pair's low or high half
        const uint32_t c = min((high ? u >> 16 & 0x7fff : u & 0x7fff) - kSmall, kHalf - 1u);
        return c | ((high ? u >> 20 : u >> 4) & kHalf);
      };
      auto value = [&](const uint4& v, int i) {
        const uint32_t u = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
        return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
      };
      // f(value) for a piece's values below 2^-9 in magnitude
      auto each_small = [&](const uint4& v, auto f) {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        const uint32_t m = __vminu2(__vminu2(v.x & 0x7fff7fff, v.y & 0x7fff7fff),
                                    __vminu2(v.z & 0x7fff7fff, v.w & 0x7fff7fff));
        if (min(m & 0xffff, m >> 16) >= (uint32_t)kSmall) return;
        uint32_t rest = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          rest |= (uint32_t)((i & 1 ? u[i >> 1] >> 16 & 0x7fff : u[i >> 1] & 0x7fff) < kSmall) << i;
        for (; rest; rest &= rest - 1) f(value(v, __ffs(rest) - 1));
      };
      auto slot_at = [&](int rank) {  // n_pos (if not negative): the small ones' rank
        return rank < n_pos ? n_pos - 1 - rank : kHalf + rank - n_pos - 1;
      };
      auto logit = [&](int slot) {
        const int mag = kSmall + (slot < kHalf ? slot : slot - kHalf);
        return __int_as_float((slot < kHalf ? 0u : 0x80000000u) | (uint32_t)mag << 16);
      };
      auto small = [&](float l) { return fabsf(l) < 0x1p-9f; };
      u64 zall = 0, mass_p = 0;  // the small ones' mass, the mass top_p is of
      uint32_t zcnt = 0;
      if (by_k || by_p) {
        each_piece([&](const uint4& v, int) {
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) atomicAdd(&S.mine[slot_of(u[i >> 1], i & 1)], 1u);
          each_small(v, [&](float l) { zall += W(l), ++zcnt; });
        });
        u64 all, nz;
        block_scan(zall, S.red, all);
        block_scan(zcnt, S.red2, nz);
        if (tid < nc) {
          Shared* to = cluster.map_shared_rank(&S, tid);
          to->zero[rank] = all;
          to->best[rank] = nz;
        }
        cluster.sync();
        if (nc > 1) {
          const int share = kCodes / nc;
          for (int i = tid; i < share; i += kNT) {
            const int c = rank * share + i;
            uint32_t n = 0;
            for (int r = 0; r < nc; ++r) n += cluster.map_shared_rank(&S, r)->mine[c];
            for (int r = 0; r < nc; ++r) cluster.map_shared_rank(&S, r)->total[c] = n;
          }
          cluster.sync();
        }
        zall = 0, zcnt = 0;
        for (int i = 0; i < nc; ++i) zall += S.zero[i], zcnt += (uint32_t)S.best[i];
      }
      const uint32_t* total = nc > 1 ? S.total : S.mine;
      // ---- PER ranks a thread: weights, then the borders
      constexpr int PER = kCodes / kNT;
      const int c0 = tid * PER, z = neg ? -1 : n_pos;  // z: the small ones' rank
      // all negative and large: ranks start behind slot kHalf
      auto at = [&](int rank) { return neg ? kHalf + top_mag - kSmall + rank : slot_at(rank); };
      const int ranks = neg ? kHalf - (top_mag - kSmall) : n_pos + 1 + kHalf;
      int erank = 1 << 20;  // ranks before it are kept, and `ties` tokens of it
      u64 ties = 0, w[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i)
        w[i] = c0 + i < ranks && c0 + i != z ? W(logit(at(c0 + i))) : 0;
      if (by_k || by_p) {
        uint32_t t[PER];
        u64 n = 0, m = 0, all;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          t[i] = c0 + i >= ranks ? 0 : c0 + i == z ? zcnt : total[at(c0 + i)];
          n += t[i];
          m += c0 + i == z ? zall : t[i] * w[i];
        }
        const u64 m0 = block_scan(m, S.red2, mass_p);
        if (by_k) {
          u64 nb = block_scan(n, S.red, all), mb = m0;
          if ((u64)top_k < all) {
            if (nb < (u64)top_k && nb + n >= (u64)top_k) {  // among this thread's
#pragma unroll
              for (int i = 0; i < PER; ++i) {
                if (nb < (u64)top_k && nb + t[i] >= (u64)top_k) {
                  S.r_bin = c0 + i;
                  S.r_above = (u64)top_k - nb;
                  S.r_mass = mb + S.r_above * w[i];
                }
                nb += t[i];
                mb += c0 + i == z ? zall : t[i] * w[i];
              }
            }
            __syncthreads();
            erank = S.r_bin, ties = S.r_above, mass_p = S.r_mass;
            __syncthreads();
          }
        }
        if (by_p && erank != z) {
          const u64 limit = ceiling((double)top_p * (double)mass_p);
          if (tid == 0) S.r_bin = 0, S.r_above = 1;  // top_p <= 0: the best token
          __syncthreads();
          if (m0 < limit && m0 + m >= limit) {
            u64 mb = m0, left = 0, each_w = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const u64 here = c0 + i == z ? zall : t[i] * w[i];
              if (mb < limit && mb + here >= limit) S.r_bin = c0 + i, left = limit - mb, each_w = w[i];
              mb += here;
            }
            S.r_above = each_w > 0 ? (left + each_w - 1) / each_w : 0;
          }
          __syncthreads();
          if ((int)S.r_bin < erank || S.r_above < ties) erank = S.r_bin, ties = S.r_above;
        }
      }
      // a border among the small ones is left to the search below
      if (erank != z) {
        __syncthreads();  // `mine` becomes `weight`
        for (int i = tid; i < kCodes; i += kNT) S.weight[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (c0 + i < ranks && c0 + i != z && c0 + i < erank)
            S.weight[at(c0 + i)] = floored(w[i]);
        // a border in the last slot leaves nothing out that weighs
        const int eslot = erank < ranks && at(erank) != kCodes - 1 ? at(erank) : -1;
        u64 wedge = eslot >= 0 ? floored(W(logit(eslot))) : 0;
        if (eslot >= 0 && tid == 0) S.weight[eslot] = 0;
        __syncthreads();
        const bool some_small = z >= 0 && z < erank;
        auto weigh = [&](float l) -> u64 {
          if (small(l)) return some_small ? floored(W(l)) : 0;
          return S.weight[slot_of(__float_as_uint(l), 1)];
        };
        u64 mass = 0;
        uint32_t n_edge = 0;
        // a table read for every token, without a branch: tokens behind the border
        // weigh 0 in it (72 us at 256 x 100003 against 81 with a comparison first)
        const float border = eslot >= 0 ? logit(eslot) : -INFINITY;
        each_piece([&](const uint4& v, int) {
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float l = value(v, i);
            mass += S.weight[slot_of(u[i >> 1], i & 1)];
            n_edge += wedge && l == border;
          }
          if (some_small) each_small(v, [&](float l) { mass += floored(W(l)); });
        });
        finish(mass, n_edge, weigh,
               [&](float l) {
                 return !small(l) && (int)slot_of(__float_as_uint(l), 1) == eslot;
               },
               ties, wedge);
        return;
      }
    }
    cluster.sync();  // the counts have been read everywhere
  }
  for (int i = tid; i < kBins; i += kNT) S.cnt[i] = S.lo[i] = S.hi[i] = 0;
  __syncthreads();

  uint32_t edge = 0;  // kept: keys above `edge`, and the first `ties` ids of key `edge`
  u64 ties = ~0ull;
  if (by_k || by_p) {
    // ---- bins of equal width in the logit, best first
    const float range = fminf(W.lmax - W.lcut, W.lmax - lmin);
    const float bscale = range > 0.f && range < INFINITY ? (float)(kBins - 1) / range : 0.f;
    // rounded to an integer in the low bits of 2^23 + x: x up to kBins - 1
    auto bin_of = [&](float l) {
      const float x = l == W.lmax ? 0.f : fminf((W.lmax - l) * bscale, (float)(kBins - 1));
      return __float_as_int(x + 8388608.f) & (kBins - 1);
    };
    each([&](float l, int) {
      if (l >= W.lcut) {
        const int b = bin_of(l);
        atomicAdd(&S.cnt[b], 1u);
        if (!by_k) add_mass(b, W.inlined(l));
      }
    });
    join();
    // exclusive sums over the bins, two a thread
    const uint32_t c0 = S.tcnt[2 * tid], c1 = S.tcnt[2 * tid + 1];
    const u64 m0 = S.tmass[2 * tid], m1 = S.tmass[2 * tid + 1];
    u64 nall, mall;
    const u64 cb = block_scan(c0 + c1, S.red, nall);
    const u64 mb = block_scan(m0 + m1, S.red2, mall);
    const double limit = (double)top_p * (double)mall;
    // the bin of the border: the last that begins before it
    if (tid == 0) S.r_bin = 0;
    __syncthreads();
#pragma unroll
    for (int e = 1; e >= 0; --e) {
      const u64 cx = cb + (e ? c0 : 0), mx = mb + (e ? m0 : 0);
      const bool in = (e ? c1 : c0) && (by_k ? cx < (u64)top_k : (double)mx < limit);
      if (in) {
        atomicMax(&S.r_bin, (uint32_t)(2 * tid + e));
        break;
      }
    }
    __syncthreads();
    const uint32_t last = S.r_bin;
    if (last / 2 == tid) {  // candidates up to it, its own, and what lies above it
      S.r_cnt = (uint32_t)(cb + c0 + (last & 1 ? c1 : 0));
      S.r_hi = last & 1 ? c1 : c0;
      S.r_above = by_k ? cb + (last & 1 ? c0 : 0) : mb + (last & 1 ? m0 : 0);
    }
    __syncthreads();
    const uint32_t n = S.r_cnt, n_bin = S.r_hi;
    const u64 above0 = S.r_above;
    // all candidates to the leading CTA if it finishes them sooner than all
    // CTAs the row, else the border's bin alone, if it can sort that. Behind one
    // border 2048 candidates on one CTA cost more than 256 (one row of 49,155, fp32,
    // top_p: 53 us against 22.6), behind two they save (64 mixed rows: 64 us with 256)
    const bool whole = n <= (by_k && by_p ? kList : kNT / 2);
    if (whole || n_bin <= kList) {
      Shared* lead = cluster.map_shared_rank(&S, 0);
      const uint32_t from = whole ? 0 : last;
      each([&](float l, int id) {
        if (l >= W.lcut) {
          const uint32_t b = bin_of(l);
          if (b <= last && b >= from)
            lead->item[atomicAdd(&lead->n_items, 1u)] =
                (u64)key_of(l) << 32 | (uint32_t)~(uint32_t)id;
        }
      });
      cluster.sync();
    }
    if (whole) {
      if (rank != 0) return;
      int n2 = 32;
      while (n2 < (int)n) n2 <<= 1;
      for (int i = (int)n + tid; i < n2; i += kNT) S.item[i] = 0;
      sort_desc(S.item, n2);
      // kPer neighbours a thread: their weights, and the mass before them
      u64 w[kPer], sum = 0, before, mass;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = kPer * tid + e;
        w[e] = i < (int)n && !(by_k && i >= top_k) ? W(logit_of((uint32_t)(S.item[i] >> 32))) : 0;
        sum += w[e];
      }
      before = block_scan(sum, S.red, mass);
      const double lim = by_k ? (double)top_p * (double)mass : limit;
      bool keep[kPer];
      u64 kept = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        keep[e] = w[e] > 0 && (kPer * tid + e == 0 ||
                               ((!by_p || (double)before < lim) && w[e] >= floor_p));
        kept += keep[e];
        before += w[e];
      }
      u64 nkept;
      block_scan(kept, S.red2, nkept);  // the kept are the first nkept of the list
      // the kept by id: ~id in the upper half, descending
      n2 = 32;
      while (n2 < (int)nkept) n2 <<= 1;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = kPer * tid + e;
        S.w[i] = w[e];
        if (i < n2) S.item[i] = keep[e] ? S.item[i] << 32 | (uint32_t)i : 0;
      }
      sort_desc(S.item, n2);
      sum = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = kPer * tid + e;
        w[e] = i < (int)nkept ? S.w[(uint32_t)S.item[i]] : 0;
        sum += w[e];
      }
      u64 total;
      u64 run = block_scan(sum, S.red, total);
      const u64 target = target_of(total);
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (run <= target && run + w[e] > target)
          answer((uint32_t)~(uint32_t)(S.item[kPer * tid + e] >> 32), w[e], total);
        run += w[e];
      }
      return;
    }
    // the key at the border of its sorted bin, and how many tokens of that key are kept
    auto border_of_bin = [&](bool mass, double want) {
      if (rank == 0) {
        const int m = (int)S.n_items;
        int n2 = 32;
        while (n2 < m) n2 <<= 1;
        for (int i = m + tid; i < n2; i += kNT) S.item[i] = 0;
        sort_desc(S.item, n2);
        u64 v[kPer], sum = 0, all;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int i = kPer * tid + e;
          v[e] = i >= m ? 0 : mass ? W(logit_of((uint32_t)(S.item[i] >> 32))) : 1;
          sum += v[e];
        }
        u64 run = above0 + block_scan(sum, S.red, all);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          // the last token that begins before the border (the first there is, if none does)
          const int i = kPer * tid + e;
          const u64 next = run + v[e];
          if (i < m && ((double)run < want || i == 0) && (!((double)next < want) || i == m - 1)) {
            const uint32_t k = (uint32_t)(S.item[i] >> 32);
            int first = 0;  // the first of its key
            for (int up = i; first < up;) {
              const int mid = (first + up) / 2;
              if ((uint32_t)(S.item[mid] >> 32) > k)
                first = mid + 1;
              else
                up = mid;
            }
            for (int r = 0; r < nc; ++r) {
              Shared* to = cluster.map_shared_rank(&S, r);
              to->r_bin = k;
              to->r_cnt = i + 1 - first;
            }
          }
          run = next;
        }
        if (tid == 0) S.n_items = 0;
      }
      cluster.sync();
    };
    // ---- too many candidates: borders by histograms over key ranges.
    // largest key whose count (mass) at or above it reaches `want`, and what is above it
    auto border = [&](bool mass, double want, u64& above_out) {
      uint32_t lo = edge, hi = kmax;
      const uint32_t kcut = key_of(W.lcut);
      if (lo < kcut) lo = kcut;
      u64 above = 0;
      for (;;) {
        const uint32_t span = hi - lo;
        const int sh = max(0, 32 - __clz(span) - 10);
        cluster.sync();  // nobody still reads the last histogram
        for (int i = tid; i < kBins; i += kNT) S.cnt[i] = S.lo[i] = S.hi[i] = 0;
        __syncthreads();
        each([&](float l, int id) {
          const uint32_t k = key_of(l);
          if (id >= 0 && id < V && k >= lo && k <= hi) {
            const int b = kBins - 1 - (int)((k - lo) >> sh);  // best first
            if (mass)
              add_mass(b, W(l));
            else
              atomicAdd(&S.cnt[b], 1u);
          }
        });
        join();
        u64 v[2], all;
#pragma unroll
        for (int e = 0; e < 2; ++e) v[e] = mass ? S.tmass[2 * tid + e] : S.tcnt[2 * tid + e];
        u64 run = above + block_scan(v[0] + v[1], S.red, all);
        // where nothing reaches it: the last bin
        if (tid == 0) S.r_bin = kBins - 1 - (span >> sh), S.r_above = above;
        __syncthreads();
        const bool none = !((double)(above + all) >= want);
        if (none) {
          if (tid == kNT - 1) S.r_bin = kBins - 1, S.r_above = run + v[0];
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if ((double)run < want && (double)(run + v[e]) >= want)
              S.r_bin = 2 * tid + e, S.r_above = run;
            run += v[e];
          }
        }
        __syncthreads();
        const uint32_t b = kBins - 1 - S.r_bin;
        above = S.r_above;
        __syncthreads();
        const uint32_t nlo = lo + (b << sh);
        hi = min(hi, nlo + ((1u << sh) - 1));
        lo = nlo;
        if (sh == 0) break;
      }
      above_out = above;
      return lo;
    };
    u64 above;
    // sums over the whole row of what f gives for each id
    auto row_sum = [&](auto f) {
      u64 s = 0, all;
      each([&](float l, int id) { s += f(l, id); });
      block_scan(s, S.red, all);
      if (tid < nc) cluster.map_shared_rank(&S, tid)->best[rank] = all;
      cluster.sync();
      all = 0;
      for (int i = 0; i < nc; ++i) all += S.best[i];
      cluster.sync();
      return all;
    };
    double lim = limit;
    bool found = !by_p;
    if (n_bin <= kList) {
      border_of_bin(!by_k, by_k ? (double)top_k : limit);
      edge = S.r_bin;
      ties = S.r_cnt;
      found = !by_k || !by_p;
    } else if (by_k) {
      edge = border(false, (double)top_k, above);
      ties = (u64)top_k - above;
    }
    if (by_k && by_p) {
      const uint32_t ed = edge;
      const u64 m = row_sum([&](float l, int) { return key_of(l) > ed ? W(l) : 0ull; });
      const u64 eq = row_sum([&](float l, int id) {
        return (u64)(id >= 0 && id < V && key_of(l) == ed);
      });
      lim = (double)top_p * (double)(m + min(ties, eq) * W(logit_of(edge)));
      if ((double)m < lim) {  // the border lies among the edge's own ties, or behind them
        const u64 w1 = W(logit_of(edge));
        if (w1 > 0) ties = min(ties, (u64)ceil((lim - (double)m) / (double)w1));
        found = true;
      }
    }
    if (!found) {
      edge = border(true, lim, above);
      const u64 w1 = W(logit_of(edge));
      ties = w1 > 0 ? (u64)fmax(1.0, ceil((lim - (double)above) / (double)w1)) : ~0ull;
    }
  }

  u64 mass = 0;
  uint32_t n_edge = 0;
  each([&](float l, int) {
    const uint32_t k = key_of(l);
    if (k > edge) mass += floored(W.inlined(l));
    n_edge += k == edge;
  });
  finish(mass, n_edge, [&](float l) { return key_of(l) > edge ? floored(W(l)) : 0ull; },
         [&](float l) { return key_of(l) == edge; }, ties,
         edge ? floored(W(logit_of(edge))) : 0ull);
}

constexpr int64_t kRunBytes = 52 << 10;

template <typename T>
int launch_sample(const SampleArgs& a, int64_t rows, cudaStream_t st) {
  // CTAs of a row: one from 148 rows on (a table of weights in each costs more
  // than it saves: 148 rows of 49,155, bf16, top_p 33 us, with four 70; fp32 rows of
  // mixed filters would gain, 80 and 68), else up to 8 so that every SM has work
  // (one row, top_p, 22.6 us, on one CTA 33; fp32 22.6 and 70), 512 ids each or more
  int nc = 1;
  while (nc < kMaxCtas && rows * nc < 148 && a.vocab >= nc * 1024) nc *= 2;
  // a CTA's run in shared memory if two CTAs still fit an SM (64 rows of 49,155,
  // fp32, top_p: 43 us against 46 from L2; most others alike)
  const int64_t run = (a.vocab * (int64_t)sizeof(T) / 16 + 2 + nc) / nc * 16;
  const int cached = run <= kRunBytes;
  const int smem = (int)((sizeof(Shared) + 15) / 16 * 16 + (cached ? run : 0));
  auto* k = k_sample<T>;
  static SmemLimit limit;
  if (const int e = limit.raise(reinterpret_cast<const void*>(k),
                                (int)((sizeof(Shared) + 15) / 16 * 16 + kRunBytes)))
    return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * nc));
  cfg.blockDim = dim3(kNT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = nc, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, k, a, cached);
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
  if (rows < 0 || rows > 0x7fffffff / kMaxCtas) return serve_invalid(op, "rows out of range");
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
  const int rc = dtype == MEP_BF16 ? launch_sample<__nv_bfloat16>(a, rows, st)
                                   : launch_sample<float>(a, rows, st);
  if (rc) return serve_cuda(op, (cudaError_t)rc);
  return serve_launched(op);
}
