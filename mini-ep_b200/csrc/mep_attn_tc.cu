// Attention over the shared prefix on the tcgen05 tensor cores, for bf16 models
// and batches of many rows: the queries of the whole batch that share a
// key/value head are the rows of one matrix product, so a prefix tile is read
// once for 256 of them and the work is bound by the products and the
// exponentials, not by the prefix's bytes.
//
// A CTA has 256 rows (two halves of 128, the MMA's M) and walks tiles of 128
// keys in steps of 64: S = Q K^T into TMEM, a thread a row takes the running
// maximum and the exponentials, P goes back to TMEM over S as bf16 and is the A
// operand of O += P V, which stays in TMEM. Each half has two S buffers, so
// that the next step's scores are there when a step's exponentials are done:
// with one buffer of 128 keys the products' latency (1900 of 4100 clocks a
// tile) lay open, 128 us where this takes 109, although a product of 64 columns
// holds the tensor cores as long as one of 128. Q lies in shared memory, K and V come by TMA through rings (a 3D
// tensor map, so that the last tile's missing keys read as zeros). O is
// rescaled only when a row's maximum has grown by more than 2^8 since it was
// last fixed: weights up to 2^8 are as exact in bf16 and fp32 as weights up to 1.
//
// Persistent: the (head, 256-row tile, key tile) units are dealt to the CTAs in
// equal runs, so a tile's keys may be cut between CTAs. A run's result is a
// partial one (fp32 sums, maximum in base 2) in the tile's next slot.
//
// 6144 rows on each of 8 heads of 128 behind 4099 keys: 109 us, 950 TFLOP/s,
// 0.59 of the measured bf16 rate (on warp-level products the call took 477 us).
// A tile of 128 keys takes the two halves 2 x 2 x (4 + 8) products of some 64
// clocks each, about three quarters of its time; the exponentials (2048 clocks
// of the unit that does 16 a clock) run beside them. 128 rows on each of 8 heads
// of 64 behind 4096 keys: 10.7 us, latency.
#include <atomic>
#include <cstdint>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include "mep_attn.cuh"
#include "mep_device.cuh"
#include "mep_tc.cuh"

namespace mep {
namespace {
namespace px {
using namespace ::mep::tc;

// the driver's cuTensorMapEncodeTiled, looked up once (no device state)
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q);
    return e == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f) : nullptr;
  }();
  return fn;
}
// bf16 (z, y, x) with 128-byte swizzle, zeros outside; 0 ok
int encode_3d(CUtensorMap* m, const void* base, const cuuint64_t (&dims)[3],
              const cuuint32_t (&box)[3]) {
  if (!encoder()) return -1;
  const cuuint64_t strides[2] = {dims[0] * 2, dims[0] * dims[1] * 2};
  const cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = encoder()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base),
                               dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -100 - (int)r;
}

constexpr int kRows = 128;   // rows of a half
constexpr int kKeys = 128;   // keys of a tile
constexpr int kStep = 64;    // keys of a step
constexpr int kThreads = 352;  // two softmax warpgroups, an MMA warp for each, a TMA warp
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr float kGrow = 8.f;

template <int DP>
struct Cfg {
  static constexpr int SUB = kKeys * 128;           // 128 rows of 64 bf16: one swizzled block
  static constexpr int TILE = DP / 64 * SUB;        // Q half, K tile or V tile
  static constexpr int STAGES = DP == 64 ? 4 : 2;   // of K, and of V
  static constexpr int DATA = (2 + 2 * STAGES) * TILE;
  static constexpr int SMEM = DATA + 1024 + 1024;   // data | barriers | alignment slack
  // kind::f16, fp32 accumulators, bf16 operands, M = 128
  static constexpr uint32_t BASE = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kRows >> 4) << 24);
  static constexpr uint32_t IDESC_S = BASE | ((uint32_t)(kStep >> 3) << 17);
  static constexpr uint32_t IDESC_O = BASE | ((uint32_t)(DP >> 3) << 17) | (1u << 16);  // V: N-major
};

struct Smem {
  uint64_t kfull[4], kempty[4], vfull[4], vempty[4];
  uint64_t qready[2], qfree[2], sfull[2][2], pfull[2][2], odone[2], ofull[2], drained[2];
  uint32_t tmem_base;
  int abort;
};

struct Args {
  AttnArgs a;
  int group, rows, row_tiles, key_tiles, slots;
  int last_load;  // a CTA's loads stop at this one of K, as if a wait ran out (-1: never)
  int64_t units, out_rows;
  float* part_o;
  float2* part_ml;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* tm, int x, int y, int z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// V as the B operand: the 64 values of a swizzled row run along N, rows along
// K. Blocks of 64 values are SUB bytes apart, groups of 8 keys 1024.
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr, uint32_t block_bytes) {
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(block_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
// Products from ready descriptors. ACC: 0 overwrite, 1 accumulate, 2 as `acc` says.
template <int ACC>
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "n"(ACC));
}
// A operand from TMEM
template <int ACC>
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b,
                                       uint32_t idesc, uint32_t acc) {
  if (ACC == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "n"(ACC));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// two fp32 values an instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  return (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
}
__device__ __forceinline__ void unpair(uint64_t v, float& x, float& y) {
  x = __uint_as_float((uint32_t)v), y = __uint_as_float((uint32_t)(v >> 32));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    k_attn_prefix_tc(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const Args p) {
  using C = Cfg<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sq = smem;                        // two halves of queries
  uint8_t* sk = smem + 2 * C::TILE;          // ring of K tiles
  uint8_t* sv = sk + C::STAGES * C::TILE;    // ring of V tiles
  Smem* S = reinterpret_cast<Smem*>(smem + C::DATA);
  const int wp = warp_id(), lane = lane_id();
  const AttnArgs& a = p.a;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&S->kfull[s], 1), mbar_init(&S->kempty[s], 2);
      mbar_init(&S->vfull[s], 1), mbar_init(&S->vempty[s], 2);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&S->qready[w], 4), mbar_init(&S->qfree[w], 4), mbar_init(&S->odone[w], 1);
      mbar_init(&S->ofull[w], 1), mbar_init(&S->drained[w], 1);
      for (int i = 0; i < 2; ++i) mbar_init(&S->sfull[w][i], 1), mbar_init(&S->pfull[w][i], kRows);
    }
    S->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (wp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&S->tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  // S of half w, buffer i: columns 128 w + 64 i; O: 256 + DP w
  const uint32_t tmem = S->tmem_base;
  // bounded; the clock is first read after 256 tries, well past any wait of a
  // healthy run (reading it at the first miss held up every wait)
  auto wait = [&](uint64_t* b, uint32_t parity) {
    unsigned long long t0 = 0;
    for (uint32_t it = 1; !mbar_try(b, parity); ++it) {
      if (it & 255u) continue;
      if (*reinterpret_cast<volatile int*>(&S->abort)) return false;
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kWaitNs) {
        *reinterpret_cast<volatile int*>(&S->abort) = 1;
        return false;
      }
    }
    return true;
  };
  // this CTA's run of units; f(tile, first key tile, last + 1) for each tile in it
  const int64_t u0 = p.units * blockIdx.x / gridDim.x, u1 = p.units * (blockIdx.x + 1) / gridDim.x;
  auto each_tile = [&](auto f) {
    for (int64_t u = u0; u < u1;) {
      const int tile = (int)(u / p.key_tiles), k0 = (int)(u - (int64_t)tile * p.key_tiles);
      const int k1 = (int)min((int64_t)p.key_tiles, k0 + (u1 - u));
      if (!f(tile, k0, k1)) return;
      u += k1 - k0;
    }
  };
  // steps of key tiles [k0, k1): the last tile's second one may hold no key
  auto steps_of = [&](int k0, int k1) {
    return min(2 * (k1 - k0), ((int)a.prefix_cols - k0 * kKeys + kStep - 1) / kStep);
  };
  auto halves_of = [&](int tile) {
    return p.rows - (tile % p.row_tiles) * 2 * kRows > kRows ? 2 : 1;
  };

  if (wp == 10) {
    // ------------------------------------------------------------ TMA loads
    if (lane == 0) {
      int s = 0, k_loads = 0, v_loads = 0;
      uint32_t ph = 0;
      each_tile([&](int tile, int k0, int k1) {
        const int kh = tile / p.row_tiles;
        for (int k = k0; k < k1; ++k) {
          if (!wait(&S->kempty[s], ph ^ 1u)) return false;
          mbar_expect_tx(&S->kfull[s], C::TILE);
          for (int d = 0; d < DP / 64; ++d)
            tma_load_3d(sk + s * C::TILE + d * C::SUB, &tmK, d * 64, k * kKeys, kh, &S->kfull[s]);
          if (k_loads++ == p.last_load) {
            *reinterpret_cast<volatile int*>(&S->abort) = 1;
            return false;
          }
          if (!wait(&S->vempty[s], ph ^ 1u)) return false;
          mbar_expect_tx(&S->vfull[s], C::TILE);
          for (int d = 0; d < DP / 64; ++d)
            tma_load_3d(sv + s * C::TILE + d * C::SUB, &tmV, d * 64, k * kKeys, kh, &S->vfull[s]);
          ++v_loads;
          if (++s == C::STAGES) s = 0, ph ^= 1u;
        }
        return true;
      });
      // leave no copy in flight, whoever gave up: load n fills stage n % STAGES
      for (int n = max(0, k_loads - C::STAGES); n < k_loads; ++n)
        mbar_wait_for(&S->kfull[n % C::STAGES], n / C::STAGES & 1, kWaitNs, nullptr);
      for (int n = max(0, v_loads - C::STAGES); n < v_loads; ++n)
        mbar_wait_for(&S->vfull[n % C::STAGES], n / C::STAGES & 1, kWaitNs, nullptr);
    }
  } else if (wp >= 8) {
    // ------------------------------------------------------------ MMA issue
    // A warp for each half, so that one's waits do not hold up the other's
    // products. The whole warp walks the steps, its elected lane issues: with
    // operands that are the same in every lane an instruction takes the issuer
    // some 50 clocks; from a branch of one lane it took 80, more than it ran.
    const int w = wp - 8;
    int ks = 0, vs = 0;
    uint32_t kph = 0, vph = 0, qph = 0, pph[2] = {0, 0};
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    // descriptors of the first block of each buffer; addresses count 16 bytes
    const uint64_t qw = sw128_desc(smem_u32(sq + w * C::TILE)), kd = sw128_desc(smem_u32(sk));
    const uint64_t vd = v_desc(smem_u32(sv), C::SUB);
    auto wait_all = [&](uint64_t* b, uint32_t parity) {
      return __all_sync(0xffffffffu, wait(b, parity)) != 0;
    };
    each_tile([&](int tile, int k0, int k1) {
      const bool idle = w >= halves_of(tile);
      const int steps = steps_of(k0, k1);
      auto next_k = [&] { if (++ks == C::STAGES) ks = 0, kph ^= 1u; };
      auto next_v = [&] { if (++vs == C::STAGES) vs = 0, vph ^= 1u; };
      if (idle) {  // no such rows: only release the tiles
        for (int k = k0; k < k1; ++k) {
          if (!wait_all(&S->kfull[ks], kph)) return false;
          if (lane == 0) mbar_arrive(&S->kempty[ks]);
          next_k();
          if (!wait_all(&S->vfull[vs], vph)) return false;
          if (lane == 0) mbar_arrive(&S->vempty[vs]);
          next_v();
        }
        return true;
      }
      // the scores of step t, from the K tile in stage ks
      auto scores = [&](int t) {
        const uint64_t kw = kd + (uint32_t)(ks * (C::TILE >> 4) + (t & 1) * (kStep * 128 >> 4));
        const uint32_t to = tm + 128 * w + 64 * (t & 1);
        const bool k_used = (t & 1) || t + 1 == steps;
        if (elect_one()) {
          mma_ss<0>(to, qw, kw, C::IDESC_S);
#pragma unroll
          for (int kk = 1; kk < DP / 16; ++kk) {
            const uint32_t off = (kk >> 2) * (C::SUB >> 4) + (kk & 3) * 2;
            mma_ss<1>(to, qw + off, kw + off, C::IDESC_S);
          }
          mma_commit<false>(&S->sfull[w][t & 1]);
          if (k_used) mma_commit<false>(&S->kempty[ks]);
        }
        __syncwarp();
        if (k_used) next_k();
      };
      if (!wait_all(&S->kfull[ks], kph) || !wait_all(&S->qready[w], qph)) return false;
      qph ^= 1u;
      fence_after();
      scores(0);
      if (steps > 1) scores(1);
      for (int t = 0; t < steps; ++t) {
        const int i = t & 1;
        if (i == 0 && !wait_all(&S->vfull[vs], vph)) return false;
        if (i == 0 && t + 2 < steps && !wait_all(&S->kfull[ks], kph)) return false;
        if (!wait_all(&S->pfull[w][i], pph[i])) return false;
        pph[i] ^= 1u;
        fence_after();
        const uint32_t po = tm + 256 + DP * w, pt = tm + 128 * w + 64 * i;
        const uint64_t vw = vd + (uint32_t)(vs * (C::TILE >> 4) + i * (kStep * 128 >> 4));
        const bool v_used = i || t + 1 == steps;
        if (elect_one()) {
          mma_ts<2>(po, pt, vw, C::IDESC_O, t != 0);
#pragma unroll
          for (int kk = 1; kk < kStep / 16; ++kk)
            mma_ts<1>(po, pt + kk * 8, vw + kk * (2048 >> 4), C::IDESC_O, 1);
          // before ofull: the tile's last arrival is the one waited for
          if (v_used) mma_commit<false>(&S->vempty[vs]);
          mma_commit<false>(&S->odone[w]);
          if (t + 1 == steps) mma_commit<false>(&S->ofull[w]);
        }
        __syncwarp();
        if (v_used) next_v();
        if (t + 2 < steps) scores(t + 2);
      }
      return true;
    });
    // leave no product in flight either
    if (elect_one()) mma_commit<false>(&S->drained[w]);
    __syncwarp();
    mbar_wait_for(&S->drained[w], 0, kWaitNs, nullptr);
  } else {
    // ------------------------------------------------------------ softmax
    const int w = wp >> 2, quad = wp & 3, tr = quad * 32 + lane;  // half, lane quadrant, row
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + lanes + 128 * w, to = tmem + lanes + 256 + DP * w;
    const float turn = a.scale < 0.f ? -1.f : 1.f;
    const float rs = fmaxf(a.scale * turn * kLog2e, kLeastScale);
    const uint32_t flip = turn < 0.f ? 0x80008000u : 0u;
    // dph: parity of the last step's product. Its wait in step t may lag by one
    // phase only: the scores of step t came behind the product of step t - 2.
    uint32_t sph[2] = {0, 0}, dph = 1, oph = 0, fph = 1;
    const int D = a.head_dim;
    // Once a wait has run out the rest of the run is only marked: sums of NaN,
    // which the join carries into every value of those rows.
    int ok = 1;
    each_tile([&](int tile, int k0, int k1) {
      if (w >= halves_of(tile)) return true;
      const int kh = tile / p.row_tiles, r = (tile % p.row_tiles) * 2 * kRows + w * kRows + tr;
      const bool real = r < p.rows;
      const int bt = real ? r / p.group : 0, h = kh * p.group + (real ? r - bt * p.group : 0);
      const int b = bt / (int)a.tokens, t = bt - b * (int)a.tokens;
      // ---- this thread's query row, K-major with the 128-byte swizzle, once the
      // half's four warps have written the last tile's results out of the buffer
      if (ok) ok = __all_sync(0xffffffffu, wait(&S->qfree[w], fph));
      fph ^= 1u;
      if (ok) {
        const __nv_bfloat16* q =
            static_cast<const __nv_bfloat16*>(a.q.p) + b * a.q.sb + t * a.q.st + h * a.q.sh;
        uint8_t* row = sq + w * C::TILE + tr * 128;
        uint4 v[DP / 8];  // all loads before the first store
#pragma unroll
        for (int c = 0; c < DP / 8; ++c)
          v[c] = real && c * 8 < D ? *reinterpret_cast<const uint4*>(q + c * 8)
                                   : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
          v[c].x ^= flip, v[c].y ^= flip, v[c].z ^= flip, v[c].w ^= flip;
          *reinterpret_cast<uint4*>(row + (c >> 3) * C::SUB + (((c & 7) ^ (tr & 7)) << 4)) = v[c];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&S->qready[w]);
      }
      float m = -INFINITY, l = 0.f;  // fixed maximum (before rs), sum
      const int steps = steps_of(k0, k1);
      for (int t = 0; ok && t < steps; ++t) {
        const int i = t & 1;
        ok = __all_sync(0xffffffffu, wait(&S->sfull[w][i], sph[i]));
        if (!ok) break;
        sph[i] ^= 1u;
        fence_after();
        uint32_t s[2][32];
        tmem_ld32(ts + 64 * i, s[0]);
        tmem_ld32(ts + 64 * i + 32, s[1]);
        tmem_wait_ld();
        const int left = (int)a.prefix_cols - k0 * kKeys - t * kStep;  // keys of this step
        if (left < kStep) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (c * 32 + e >= left) s[c][e] = 0xff800000u;  // -inf
        }
        float mx4[4] = {m, m, m, m};  // four chains of maxima at a time
#pragma unroll
        for (int e = 0; e < 32; e += 2)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            mx4[c] = fmaxf(mx4[c], __uint_as_float(s[c >> 1][e + (c & 1)]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        const bool grow = t == 0 || (mx - m) * rs > kGrow;
        if (t == 0) {
          m = mx;
        } else if (__any_sync(0xffffffffu, grow)) {
          // the last step's product has to be done before O is touched
          ok = __all_sync(0xffffffffu, wait(&S->odone[w], dph));
          if (!ok) break;
          fence_after();
          const float f = grow ? ex2((m - mx) * rs) : 1.f;
          if (grow) m = mx;
          l *= f;
#pragma unroll 1
          for (int c = 0; c < DP; c += 8) {
            uint32_t o[8];
            tmem_ld8(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st8(to + c, o);
          }
        }
        const float base = m == -INFINITY ? 0.f : m * rs;
        const uint64_t rs2 = pair(rs, rs), nb2 = pair(-base, -base);
        uint64_t sum[2] = {0, 0};  // (0.f, 0.f)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x, y;
            unpair(fma2((uint64_t)s[c][2 * e + 1] << 32 | s[c][2 * e], rs2, nb2), x, y);
            x = ex2(x), y = ex2(y);
            sum[e & 1] = add2(sum[e & 1], pair(x, y));
            pk[e] = pack_bf16x2(x, y);
          }
          tmem_st16(ts + 64 * i + 16 * c, pk);
        }
        tmem_wait_st();
        fence_before();
        mbar_arrive(&S->pfull[w][i]);
        dph ^= 1u;
        float x, y;
        unpair(add2(sum[0], sum[1]), x, y);
        l += x + y;
      }
      // ---- the run's result to its slot; slots behind the tile's last are empty
      if (ok) {
        ok = __all_sync(0xffffffffu, wait(&S->ofull[w], oph));
        oph ^= 1u;
      }
      fence_after();
      const int64_t x0 = (int64_t)tile * p.key_tiles;
      const int slot = (int)blockIdx.x - (int)(((x0 + 1) * gridDim.x - 1) / p.units);
      const int64_t orow = ((int64_t)b * a.tokens + t) * a.q_heads + h;
      if (real) {
        const float mb = m == -INFINITY ? m : m * rs;
        p.part_ml[slot * p.out_rows + orow] =
            ok ? make_float2(mb, l) : make_float2(0.f, __int_as_float(0x7fffffff));
        if (k1 == p.key_tiles)
          for (int e = slot + 1; e < p.slots; ++e)
            p.part_ml[e * p.out_rows + orow] = make_float2(-INFINITY, 0.f);
      }
      if (!ok) return true;
      // O through the half's query buffer, which no product reads any more: W
      // values of the warp's 32 rows at a time, written out a row at a time
      constexpr int W = DP / 4, STRIDE = W * 4 + 16, PER = W / 4;  // 16: rows in other banks
      static_assert(kRows * STRIDE <= C::TILE, "O passes fit the query buffer");
      uint8_t* mine = sq + w * C::TILE + quad * 32 * STRIDE;
      const int at = real ? (int)orow : -1;
#pragma unroll 1
      for (int c = 0; c < DP; c += W) {
        uint32_t o[W];
        if constexpr (W == 32)
          tmem_ld32(to + c, o);
        else
          tmem_ld16(to + c, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < W; e += 4)
          *reinterpret_cast<uint4*>(mine + lane * STRIDE + e * 4) =
              make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        __syncwarp();
        const int piece = lane % PER, d = c + piece * 4;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int r = e * (32 / PER) + lane / PER;
          const int to_row = __shfl_sync(0xffffffffu, at, r);
          const uint4 v = *reinterpret_cast<const uint4*>(mine + r * STRIDE + piece * 16);
          if (to_row >= 0 && d < D)
            *reinterpret_cast<uint4*>(p.part_o + (slot * p.out_rows + to_row) * D + d) = v;
        }
        __syncwarp();
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&S->qfree[w]);
      return true;
    });
  }
  // every warp arrives, so no copy, product or TMEM access is left when TMEM goes
  fence_before();
  __syncthreads();
  fence_after();
  if (wp == 8)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <int DP>
int launch(const Args& p, int ctas, cudaStream_t st) {
  const AttnArgs& a = p.a;
  CUtensorMap tk, tv;
  const cuuint64_t dims[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.prefix_cols,
                              (cuuint64_t)a.kv_heads};
  const cuuint32_t box[3] = {64, kKeys, 1};
  if (const int rc = encode_3d(&tk, a.kp, dims, box)) return rc;
  if (const int rc = encode_3d(&tv, a.vp, dims, box)) return rc;
  static SmemLimit limit;
  if (const int e = limit.raise(reinterpret_cast<const void*>(k_attn_prefix_tc<DP>), Cfg<DP>::SMEM))
    return e;
  k_attn_prefix_tc<DP><<<ctas, kThreads, Cfg<DP>::SMEM, st>>>(tk, tv, p);
  return 0;
}

}  // namespace px
}  // namespace

std::atomic<int> g_last_load{-1};

// Units of a CTA, at least (while the others suffice): fewer CTAs leave fewer
// partial results. 512 rows on each of 8 heads of 64 behind 4096 keys: 53.4 us,
// with 2 58.1, with 8 57.5; 128 rows behind 1024: 22.6, 20.5, 26.7.
constexpr int kMinUnits = 4;

PrefixTcPlan plan_prefix_tc(int64_t rows, int kv_heads, int64_t prefix_cols) {
  const int64_t key_tiles = (prefix_cols + px::kKeys - 1) / px::kKeys;
  const int64_t units = kv_heads * ((rows + 2 * px::kRows - 1) / (2 * px::kRows)) * key_tiles;
  PrefixTcPlan p;
  const int64_t most = (units + kMinUnits - 1) / kMinUnits;
  p.ctas = (int)(most < 148 ? most : 148);
  // a tile's key tiles lie in at most so many runs of units / ctas or more
  const int64_t run = units / p.ctas;
  const int64_t slots = (key_tiles - 1 + run - 1) / run + 1;
  p.slots = (int)(slots < key_tiles ? slots : key_tiles);
  return p;
}

int launch_prefix_tc(const AttnArgs& a, const PrefixTcPlan& plan, int64_t out_rows, float* part_o,
                     float2* part_ml, cudaStream_t st) {
  px::Args p{a, a.q_heads / a.kv_heads, 0, 0, 0, plan.slots,
             g_last_load.load(std::memory_order_relaxed), 0, out_rows, part_o, part_ml};
  p.rows = (int)(a.batch * a.tokens * p.group);
  p.row_tiles = (p.rows + 2 * px::kRows - 1) / (2 * px::kRows);
  p.key_tiles = (int)((a.prefix_cols + px::kKeys - 1) / px::kKeys);
  p.units = (int64_t)a.kv_heads * p.row_tiles * p.key_tiles;
  return a.head_dim <= 64 ? px::launch<64>(p, plan.ctas, st) : px::launch<128>(p, plan.ctas, st);
}

}  // namespace mep

extern "C" int mep_debug_prefix_loads(int loads) {
  mep::g_last_load.store(loads < 0 ? -1 : loads, std::memory_order_relaxed);
  return MEP_OK;
}
