// Attention of the new tokens over the key/value cache.
//
// Query (b, t, h) attends to every column of the shared prefix (if any) and to
// the own columns c of row b with c <= col + t and (c < lengths[b] or
// c >= prompt_cols):
//   s = scale * q.k, out = sum exp(s - m) v / sum exp(s - m), m = max s,
// in fp32, rounded once to the model dtype; zeros where nothing is visible.
//
// One pass over the keys with a running maximum and sum. The queries that
// share a key/value head are the rows of one matrix: for the own columns the
// T * (q_heads / kv_heads) queries of a batch row, for the prefix those of the
// whole batch, so that each key is read once for all of them. The keys are cut
// into splits that run on different SMs; their partial results (fp32 sums, the
// maximum in base 2) meet in k_attn_join.
//
// Measured, device time. One token a row: 8 rows over 32,768 columns, 32 / 8
// heads of 128, bf16: 158 us, the bytes at the measured copy rate; in e4m3 92 us
// for 81 of bytes. 64 ragged rows of 577 to 1089 columns, 16 / 8 heads of 64,
// e4m3: 16.6 us for 8.9 (the chain of a row's 9 tiles, and issue at 0.46). One row
// of 257 columns: 8.2 us, launch and latency. Whole prompts over their own columns
// go by the warp-level products, which bound them with the exponentials beside
// (tensor pipe 0.42, issue 0.44 busy): 16 x 1021 tokens, 32 / 8 heads of 128, bf16
// 591 us, 212 TFLOP/s of the visible products (78 us at the measured rate), e4m3
// 730, fp32 4.7 ms (three tf32 products for one, spills at 255 registers).
#include <cstdint>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "mep_attn.cuh"
#include "mep_device.cuh"

namespace mep {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 128;  // four warps a CTA

__device__ __forceinline__ void cp16(void* dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(real ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp4(void* dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(real ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p)));
}
// an 8 x 8 block of 16-bit values, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// x = hi + lo, each with the 11 bits a tf32 operand holds: products of split
// operands leave out only lo * lo, 2^-22 of the product
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = tf32(x);
  lo = tf32(x - __uint_as_float(hi));
}
__device__ __forceinline__ float two_to(int e) {  // 2^e, e in [-126, 127]
  return __uint_as_float((uint32_t)(127 + e) << 23);
}
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
  return r;
}
__device__ __forceinline__ float half_lo(uint32_t h2) {
  return __half2float(__ushort_as_half((unsigned short)(h2 & 0xffff)));
}
__device__ __forceinline__ float half_hi(uint32_t h2) {
  return __half2float(__ushort_as_half((unsigned short)(h2 >> 16)));
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

// The columns that rows of one matrix see, as one run of indices j in [0, n):
// columns [0, n1), then those from `skip` columns further on.
struct Span {
  int n, n1, skip;
  __device__ int column(int j) const { return j < n1 ? j : j + skip; }
};

// Geometry of a launch. Rows of a matrix: own columns, the tokens * group
// queries of one batch row (matrix index = batch row); prefix, those of the
// whole batch (one matrix). A partial result is slot [split][output row].
struct PartArgs {
  AttnArgs a;
  int group;             // query heads of a key/value head
  int rows;              // rows of a matrix
  int row_tiles, splits;
  int joined;            // the splits are a cluster, which joins them and writes `out`
  int extra;             // partial results of others that are joined with these
  int64_t out_rows;      // batch * tokens * q_heads
  float* part_o;         // [extra + splits][out_rows][head_dim]
  float2* part_ml;       // [extra + splits][out_rows]: maximum (base 2), sum
};

// How a CTA's four warps share its work.
enum Mode { kByRows = 0, kByKeys = 1, kFewRows = 2 };

// The kernel for one (element types, padded head width, warp layout).
// kByRows: each warp has 16 of 64 rows and every key of the tile. kByKeys: the
// four warps share 16 rows and take a quarter of each tile of keys each, for matrices of few rows, where the keys' bytes bound it: a
// warp streams its own keys and meets the others only at the end; a cluster of
// up to 8 CTAs, one a split, then joins its sums over distributed shared
// memory. kFewRows (16-bit queries): the same for up to 8 rows, with the keys
// along the products' 16 and the rows along their 8, S^T = K Q^T and
// O^T = V^T P^T: half the products and half the exponentials of rows that are
// not there.
template <typename QT, typename CT, int DP, int MODE>
struct Tile {
  static constexpr bool KS = MODE != kByRows;
  static constexpr int kElt = sizeof(CT);
  static constexpr int kRow = DP * kElt;  // bytes of a staged row
  // keys a warp works on at a time: 8 KB of keys and values a warp when the
  // keys are split (4 KB of codes)
  static constexpr int kN = KS ? (kRow >= 256 ? 16 : 32) : (kRow >= 512 ? 32 : 64);
  static constexpr int kKeys = KS ? 4 * kN : kN;  // keys of a CTA's tile
  static constexpr int kStages = KS ? 3 : 2;
  static constexpr int kRows = MODE == kFewRows ? 8 : KS ? 16 : 64;
  static constexpr bool kScaled = sizeof(CT) == 1;
  static constexpr int kScaleBytes = kScaled ? kKeys * 8 : 0;
  static constexpr int kStageBytes = 2 * kKeys * kRow + kScaleBytes;
  static constexpr bool kF32 = sizeof(QT) == 4;
  // fp32 queries stay in shared memory (their split halves do not fit the
  // registers), rows 4 floats apart in the banks
  static constexpr int kQRow = DP + 4;
  static constexpr int kQBytes = kF32 ? kRows * kQRow * 4 : 0;
  static constexpr int kJoin = KS ? 5 * 16 * (DP * 4 + 8) : 64 * ((DP + 4) * 4 + 8);
  static constexpr int kBody = kStages * kStageBytes + kQBytes;
  static constexpr int kSmem = kBody > kJoin ? kBody : kJoin;
  // place of 16-byte chunk c of staged row r, so that the accesses of a warp
  // fall into different banks
  __device__ static int k_chunk(int r, int c) {
    if (sizeof(CT) == 2) return c ^ (r & 7);
    return kRow >= 128 ? c ^ ((r & 1) << 2) : c;
  }
  __device__ static int v_chunk(int r, int c) {
    if (sizeof(CT) == 4) return c ^ (((r >> 1) & 3) << 1);
    return kRow >= 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
  }
};

// x += y's values, in units of 2^base, times `times`. The load does not wait for
// ml: an empty slot's values are unwritten and left out.
// kGlobal: from an earlier launch, through the read-only path, so that the
// loads of several values need not wait for the stores between them.
template <bool kGlobal>
__device__ __forceinline__ void add_part(float4& x, float2 ml, float base, float times,
                                         const float* values) {
  const float4 y = kGlobal ? __ldg(reinterpret_cast<const float4*>(values))
                           : *reinterpret_cast<const float4*>(values);
  if (ml.y != 0.f) {
    const float f = ex2(ml.x - base) * times;
    x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
  }
}

template <typename QT, typename CT, int DP, int MODE, bool PREFIX>
__global__ void __launch_bounds__(kThreads, MODE == kByRows && sizeof(QT) == 2 ? 3 : 1)
    k_attn_part(const PartArgs p) {
  using X = Tile<QT, CT, DP, MODE>;
  constexpr bool KS = X::KS, kFew = MODE == kFewRows;
  // accumulator tiles of the scores (8 keys, or 16) and of the values (8, or 16)
  constexpr int N = X::kN, NT = N / (kFew ? 16 : 8), OT = DP / (kFew ? 16 : 8);
  constexpr bool kF32 = X::kF32, kScaled = X::kScaled;
  extern __shared__ __align__(128) unsigned char smem[];
  const AttnArgs& a = p.a;
  const int lane = lane_id(), warp = warp_id(), g = lane >> 2, t4 = lane & 3;
  const int D = a.head_dim, tokens = (int)a.tokens;
  const int kh = blockIdx.y;
  const int split = blockIdx.x % p.splits;
  const int tile_id = blockIdx.x / p.splits;
  const int rt = tile_id % p.row_tiles;
  const int mat = tile_id / p.row_tiles;  // batch row (own columns)
  const int r0 = rt * X::kRows;
  const int rN = min(r0 + X::kRows, p.rows);  // rows of this CTA: [r0, rN)

  // row r of the matrix: its query, and its output row
  auto query_of = [&](int r, int& b, int& t, int& h) {
    const int bt = r / p.group;
    h = kh * p.group + (r - bt * p.group);
    b = PREFIX ? bt / tokens : mat;
    t = PREFIX ? bt - b * tokens : bt;
  };
  auto query_ptr = [&](int r) {
    int b, t, h;
    query_of(r, b, t, h);
    return static_cast<const QT*>(a.q.p) + b * a.q.sb + t * a.q.st + h * a.q.sh;
  };
  auto out_row = [&](int r) {
    int b, t, h;
    query_of(r, b, t, h);
    return ((int64_t)b * tokens + t) * a.q_heads + h;
  };

  // ---- the columns these rows see
  Span span;
  const int64_t col = PREFIX ? 0 : a.col_dev ? *a.col_dev : a.col;
  if (PREFIX) {
    span = {(int)a.prefix_cols, (int)a.prefix_cols, 0};
  } else {
    const int tmax = (rN - 1) / p.group;
    const int64_t end = max((int64_t)0, min(col + tmax + 1, a.c.capacity));
    int64_t len = a.lengths ? max((int64_t)0, a.lengths[mat]) : end;
    if (len >= a.prompt_cols) len = end;
    const int64_t n1 = min(len, end);
    const int64_t more = end - max(a.prompt_cols, n1);
    span.n1 = (int)n1;
    span.skip = n1 < end && more > 0 ? (int)(a.prompt_cols - n1) : 0;
    span.n = (int)(n1 + (n1 < end && more > 0 ? more : 0));
  }
  // this split's share of them, in whole tiles
  const int tiles = (span.n + X::kKeys - 1) / X::kKeys;
  const int tile0 = (int)((int64_t)tiles * split / p.splits);
  const int tile1 = (int)((int64_t)tiles * (split + 1) / p.splits);

  const int64_t head_row = PREFIX ? (int64_t)kh * a.prefix_cols
                                  : ((int64_t)mat * a.kv_heads + kh) * a.c.capacity;
  const int row_bytes = D * X::kElt;
  // ---- staging: 16-byte copies of the tile's rows, zeros past the span
  // (rows that nobody sees are never read, whatever they hold). A thread
  // copies piece `pc` of every kSweep-th row.
  constexpr int kPieces = DP * X::kElt / 16, kWho = KS ? 32 : kThreads;
  constexpr int kSweep = kWho / kPieces;
  const int who = KS ? lane : threadIdx.x;
  const int pc = who % kPieces, pr = (KS ? warp * N : 0) + who / kPieces;
  const bool has_piece = pc * 16 < row_bytes;
  const unsigned char* kbase =
      static_cast<const unsigned char*>(PREFIX ? a.kp : a.c.k) + head_row * row_bytes + pc * 16;
  const unsigned char* vbase =
      static_cast<const unsigned char*>(PREFIX ? a.vp : a.c.v) + head_row * row_bytes + pc * 16;
  auto stage = [&](int tile, int buf) {
    unsigned char* s = smem + buf * X::kStageBytes;
    if (has_piece) {
#pragma unroll
      for (int it = 0; it < N / kSweep; ++it) {
        const int r = pr + it * kSweep;
        const int j = tile * X::kKeys + r;
        const bool real = j < span.n;
        const int64_t at = (int64_t)(real ? span.column(j) : 0) * row_bytes;
        cp16(s + r * X::kRow + X::k_chunk(r, pc) * 16, kbase + at, real);
        cp16(s + X::kKeys * X::kRow + r * X::kRow + X::v_chunk(r, pc) * 16, vbase + at, real);
      }
    }
    if (kScaled) {
      float* sc = reinterpret_cast<float*>(s + 2 * X::kKeys * X::kRow);
      for (int i = who; i < N; i += kWho) {
        const int r = (KS ? warp * N : 0) + i;
        const int j = tile * X::kKeys + r;
        const bool real = j < span.n;
        const int64_t at = head_row + (real ? span.column(j) : 0);
        cp4(sc + r, a.c.ks + at, real);
        cp4(sc + X::kKeys + r, a.c.vs + at, real);
      }
    }
  };
  auto sync = [&] {
    if (KS)
      __syncwarp();
    else
      __syncthreads();
  };
  // padding between D and DP holds zeros from the start
  if (D < DP) {
    for (int i = threadIdx.x; i < X::kStages * 2 * X::kKeys * kPieces; i += kThreads) {
      const int c = i % kPieces, r = (i / kPieces) % X::kKeys, kv = (i / kPieces / X::kKeys) % 2;
      const int st = i / kPieces / X::kKeys / 2;
      if (c * 16 >= row_bytes)
        *reinterpret_cast<uint4*>(smem + st * X::kStageBytes + kv * X::kKeys * X::kRow +
                                  r * X::kRow + (kv ? X::v_chunk(r, c) : X::k_chunk(r, c)) * 16) =
            make_uint4(0, 0, 0, 0);
    }
  }
  // a negative scale turns the queries' sign, so that a larger score is always
  // a larger product
  const float turn = a.scale < 0.f ? -1.f : 1.f;
  float* qs = reinterpret_cast<float*>(smem + X::kStages * X::kStageBytes);
  if (kF32) {
    for (int i = threadIdx.x; i < X::kRows * DP; i += kThreads) {
      const int r = i / DP, d = i % DP;
      float x = 0.f;
      if (r0 + r < rN && d < D) x = Elt<QT>::to_f(query_ptr(r0 + r)[d]) * turn;
      qs[r * X::kQRow + d] = x;
    }
  }
  if (D < DP || kF32) __syncthreads();
#pragma unroll
  for (int i = 0; i < X::kStages - 1; ++i) {
    if (tile0 + i < tile1) stage(tile0 + i, i);
    cp_commit();
  }

  // ---- this thread's rows: row[0] and row[1] = row[0] + 8, or neighbours
  const int wrow = KS ? 0 : warp * 16;
  int row[2];
  int64_t tq[2];  // last column that the row sees
  float rscale[2];
  uint32_t qf[kF32 ? 1 : DP / 16][kFew ? 2 : 4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    row[u] = kFew ? r0 + 2 * t4 + u : r0 + wrow + g + 8 * u;
    tq[u] = col + (row[u] < rN ? row[u] / p.group : 0);
    rscale[u] = a.scale * turn * kLog2e;
  }
  if constexpr (!kF32) {
    const uint32_t flip = turn < 0.f ? 0x80008000u : 0u;
    // rows whose queries this thread holds: its own, or the one of its group
    constexpr int QR = kFew ? 1 : 2;
    const __nv_bfloat16* qp[2] = {nullptr, nullptr};
#pragma unroll
    for (int u = 0; u < QR; ++u) {
      const int r = kFew ? r0 + g : row[u];
      if (r < rN) qp[u] = query_ptr(r);
    }
    if constexpr (!kScaled) {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int i = 0; i < 2 * QR; ++i) {
          const int u = kFew ? 0 : i & 1, d = k * 16 + t4 * 2 + (kFew ? i : i >> 1) * 8;
          qf[k][i] = qp[u] && d < D ? *reinterpret_cast<const uint32_t*>(qp[u] + d) ^ flip : 0u;
        }
    } else {
      // Codes are exact in fp16, so the products are fp16 ones. A query row is
      // scaled by a power of two to a largest magnitude in [2^14, 2^15): its bf16
      // values stay exact down to 2^-31 of it, and below that are off by 2^-39
      // of it at most.
      uint4 raw[QR][DP / 32];
#pragma unroll
      for (int u = 0; u < QR; ++u)
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const int d = (i / 2) * 64 + t4 * 16 + (i % 2) * 8;
          raw[u][i] = qp[u] && d < D ? *reinterpret_cast<const uint4*>(qp[u] + d)
                                     : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int u = 0; u < QR; ++u) {
        float qv[DP / 4], m = 0.f;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const uint32_t w[4] = {raw[u][i].x, raw[u][i].y, raw[u][i].z, raw[u][i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            qv[i * 8 + 2 * e] = __uint_as_float((w[e] ^ flip) << 16);
            qv[i * 8 + 2 * e + 1] = __uint_as_float((w[e] ^ flip) & 0xffff0000u);
          }
        }
#pragma unroll
        for (int i = 0; i < DP / 4; ++i) m = fmaxf(m, fabsf(qv[i]));
        m = quad_max(m);
        const int ex = (int)(__float_as_uint(m) >> 23) - 127;
        const int e = m > 0.f && ex < 128 ? max(ex - 14, -126) : 0;
        const float down = two_to(-e), up = two_to(e);
        if (kFew) {
          rscale[0] *= __shfl_sync(0xffffffffu, up, 8 * t4);
          rscale[1] *= __shfl_sync(0xffffffffu, up, 8 * t4 + 4);
        } else {
          rscale[u] *= up;
        }
        // k-step k of a 64-wide block takes values 4k..4k+3 of each thread's 16
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          qf[k][u] = pack_f16x2(qv[k * 4] * down, qv[k * 4 + 1] * down);
          qf[k][u + QR] = pack_f16x2(qv[k * 4 + 2] * down, qv[k * 4 + 3] * down);
        }
      }
    }
  }

#pragma unroll
  for (int u = 0; u < 2; ++u) rscale[u] = fmaxf(rscale[u], kLeastScale);

  float o[OT][4];
#pragma unroll
  for (int i = 0; i < OT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // m before rscale
  // Codes are weighed by p times their row's scale, in fp16 for 16-bit queries:
  // times 2^wexp, which takes the row's largest such weight so far, wtop (before
  // it, in units of the running maximum), to about 2^12. Weights then keep fp16's
  // 11 bits down to 2^-26 of the largest, whatever p and scale are by themselves.
  float wtop[2] = {0.f, 0.f};
  int wexp[2] = {0, 0};

  int buf = 0, ahead = X::kStages - 1;
  for (int tile = tile0; tile < tile1; ++tile) {
    cp_wait<X::kStages - 2>();
    sync();
    if (tile + X::kStages - 1 < tile1) stage(tile + X::kStages - 1, ahead);
    cp_commit();
    const unsigned char* ks = smem + buf * X::kStageBytes;
    const unsigned char* vs = ks + X::kKeys * X::kRow;
    const float* sc = reinterpret_cast<const float*>(vs + X::kKeys * X::kRow);
    buf = buf + 1 == X::kStages ? 0 : buf + 1;
    ahead = ahead + 1 == X::kStages ? 0 : ahead + 1;
    const int kr0 = KS ? warp * N : 0;  // first staged row of this warp's keys
    const int j0 = tile * X::kKeys + kr0;
    if (KS && j0 >= span.n) continue;

    // ---- scores
    float s[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    if constexpr (kFew) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if constexpr (!kScaled) {
          const int r = kr0 + i * 16 + (lane & 15);
#pragma unroll
          for (int k = 0; k < DP / 16; ++k) {
            uint32_t ka[4];
            ldsm4(ka, ks + r * X::kRow + X::k_chunk(r, k * 2 + (lane >> 4)) * 16);
            mma_bf16(s[i], ka, qf[k][0], qf[k][1]);
          }
        } else {
          const int r = kr0 + i * 16 + g;
#pragma unroll
          for (int w = 0; w < DP / 64; ++w) {
            const uint4 v0 = *reinterpret_cast<const uint4*>(ks + r * X::kRow + X::k_chunk(r, w * 4 + t4) * 16);
            const uint4 v1 = *reinterpret_cast<const uint4*>(ks + (r + 8) * X::kRow + X::k_chunk(r + 8, w * 4 + t4) * 16);
            const uint32_t a0[4] = {v0.x, v0.y, v0.z, v0.w}, a1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t ka[4] = {e4m3x2_f16x2(a0[k] & 0xffff), e4m3x2_f16x2(a1[k] & 0xffff),
                                      e4m3x2_f16x2(a0[k] >> 16), e4m3x2_f16x2(a1[k] >> 16)};
              mma_f16(s[i], ka, qf[w * 4 + k][0], qf[w * 4 + k][1]);
            }
          }
        }
      }
    } else if constexpr (!kF32 && !kScaled) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int r = kr0 + i * 8 + (lane & 7);
#pragma unroll
        for (int k = 0; k < DP / 16; k += 2) {
          uint32_t b[4];
          ldsm4(b, ks + r * X::kRow + X::k_chunk(r, k * 2 + (lane >> 3)) * 16);
          mma_bf16(s[i], qf[k], b[0], b[1]);
          mma_bf16(s[i], qf[k + 1], b[2], b[3]);
        }
      }
    } else if constexpr (!kF32) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int r = kr0 + i * 8 + g;
#pragma unroll
        for (int w = 0; w < DP / 64; ++w) {
          const uint4 v = *reinterpret_cast<const uint4*>(ks + r * X::kRow + X::k_chunk(r, w * 4 + t4) * 16);
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_f16(s[i], qf[w * 4 + k], e4m3x2_f16x2(u[k] & 0xffff), e4m3x2_f16x2(u[k] >> 16));
        }
      }
    } else {
      const float* q0 = qs + (wrow + g) * X::kQRow;
      const float* q1 = q0 + 8 * X::kQRow;
      constexpr int kBlocks = DP / 16;  // 16 values of a row: two k-steps, 4 a thread
#pragma unroll
      for (int w = 0; w < kBlocks; ++w) {
        // scaled: chunk of 16 codes a thread, 4 of them here
        const int d = kScaled ? (w / 4) * 64 + t4 * 16 + (w % 4) * 4 : w * 16 + t4 * 4;
        const float4 x0 = *reinterpret_cast<const float4*>(q0 + d);
        const float4 x1 = *reinterpret_cast<const float4*>(q1 + d);
        uint32_t h[2][4], e[2][4];
        split_tf32(x0.x, h[0][0], e[0][0]), split_tf32(x1.x, h[0][1], e[0][1]);
        split_tf32(x0.y, h[0][2], e[0][2]), split_tf32(x1.y, h[0][3], e[0][3]);
        split_tf32(x0.z, h[1][0], e[1][0]), split_tf32(x1.z, h[1][1], e[1][1]);
        split_tf32(x0.w, h[1][2], e[1][2]), split_tf32(x1.w, h[1][3], e[1][3]);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int r = kr0 + i * 8 + g;
          float d4[4] = {0.f, 0.f, 0.f, 0.f};  // added to s in fp32, see `fresh` below
          if constexpr (kScaled) {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(
                ks + r * X::kRow + X::k_chunk(r, (w / 4) * 4 + t4) * 16 + (w % 4) * 4);
            const uint32_t lo = e4m3x2_f16x2(v & 0xffff), hi = e4m3x2_f16x2(v >> 16);
            const uint32_t b[4] = {__float_as_uint(half_lo(lo)), __float_as_uint(half_hi(lo)),
                                   __float_as_uint(half_lo(hi)), __float_as_uint(half_hi(hi))};
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              mma_tf32(d4, e[k], b[2 * k], b[2 * k + 1]);
              mma_tf32(d4, h[k], b[2 * k], b[2 * k + 1]);
            }
          } else {
            const float4 v = *reinterpret_cast<const float4*>(ks + r * X::kRow +
                                                              X::k_chunk(r, w * 4 + t4) * 16);
            uint32_t bh[4], bl[4];
            split_tf32(v.x, bh[0], bl[0]), split_tf32(v.y, bh[1], bl[1]);
            split_tf32(v.z, bh[2], bl[2]), split_tf32(v.w, bh[3], bl[3]);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              mma_tf32(d4, h[k], bl[2 * k], bl[2 * k + 1]);
              mma_tf32(d4, e[k], bh[2 * k], bh[2 * k + 1]);
              mma_tf32(d4, h[k], bh[2 * k], bh[2 * k + 1]);
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][j] += d4[j];
        }
      }
    }

    // ---- scale, mask, running maximum. Of accumulator element j of tile i:
    // its row (u: the thread's first or second), its key
    auto row_of = [](int j) { return kFew ? j & 1 : j >> 1; };
    auto key_of = [&](int i, int j) {
      return kFew ? i * 16 + g + 8 * (j >> 1) : i * 8 + t4 * 2 + (j & 1);
    };
    // over the lanes that hold other keys of the same rows
    auto all_max = [](float x) {
      if constexpr (kFew) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
        return x;
      } else {
        return quad_max(x);
      }
    };
    const bool edge = j0 + N > span.n || (!PREFIX && tokens > 1);
    float mx[2] = {m[0], m[1]};
    float vv[kScaled ? NT : 1][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (kScaled) {
        const int k0 = kr0 + key_of(i, 0), k1 = kr0 + key_of(i, kFew ? 2 : 1);
        const float f0 = sc[k0], f1 = sc[k1];
        vv[i][0] = sc[X::kKeys + k0], vv[i][1] = sc[X::kKeys + k1];
        s[i][0] *= f0, s[i][1] *= kFew ? f0 : f1, s[i][2] *= kFew ? f1 : f0, s[i][3] *= f1;
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int jj = j0 + key_of(i, j);
          const bool see = jj < span.n && (PREFIX || span.column(jj) <= tq[row_of(j)]);
          if (!see) s[i][j] = -INFINITY;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) mx[row_of(j)] = fmaxf(mx[row_of(j)], s[i][j]);
    }
    float keep[2], base[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      mx[u] = all_max(mx[u]);
      base[u] = mx[u] == -INFINITY ? 0.f : mx[u] * rscale[u];
      keep[u] = m[u] == -INFINITY ? 0.f : ex2((m[u] - mx[u]) * rscale[u]);
      m[u] = mx[u];
      l[u] *= keep[u];
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = ex2(fmaf(s[i][j], rscale[row_of(j)], -base[row_of(j)]));
        l[row_of(j)] += s[i][j];
      }
    if (kScaled) {
      float top[2] = {0.f, 0.f}, times[2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        s[i][0] *= vv[i][0], s[i][1] *= vv[i][kFew ? 0 : 1];
        s[i][2] *= vv[i][kFew ? 1 : 0], s[i][3] *= vv[i][1];
#pragma unroll
        for (int j = 0; j < 4; ++j) top[row_of(j)] = fmaxf(top[row_of(j)], s[i][j]);
      }
      bool renew = false;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        wtop[u] *= keep[u];
        times[u] = two_to(wexp[u]);
        renew |= keep[u] != 1.f || top[u] * times[u] > 32768.f;
      }
      if (__any_sync(0xffffffffu, renew)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          wtop[u] = fmaxf(wtop[u], all_max(top[u]));
          const int e = wtop[u] > 0.f ? 12 + 127 - (int)(__float_as_uint(wtop[u]) >> 23) : 0;
          const int was = wexp[u];
          wexp[u] = min(max(e, -126), 126);
          keep[u] *= two_to(min(max(wexp[u] - was, -126), 127));
          times[u] = two_to(wexp[u]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] *= times[row_of(j)];
    }
    // most tiles change neither maximum nor wexp: nothing to rescale
    if (!kF32 && __any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] *= keep[row_of(j)];
    }

    // ---- o += p v
    if constexpr (kFew) {
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        // the 8 x 8 blocks (keys, rows) turned into (rows, keys)
        uint32_t p0 = kScaled ? pack_f16x2(s[k][0], s[k][1]) : pack_bf16(s[k][0], s[k][1]);
        uint32_t p1 = kScaled ? pack_f16x2(s[k][2], s[k][3]) : pack_bf16(s[k][2], s[k][3]);
        p0 = transposed(p0), p1 = transposed(p1);
        if constexpr (!kScaled) {
          const int r = kr0 + k * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
          for (int n = 0; n < OT; ++n) {
            uint32_t va[4];
            ldsm4t(va, vs + r * X::kRow + X::v_chunk(r, n * 2 + (lane >> 3 & 1)) * 16);
            mma_bf16(o[n], va, p0, p1);
          }
        } else {
          // of the byte pair of a key, the first is value 16 n + 2 g, the
          // second 16 n + 2 g + 1: the tile's rows g and g + 8
          const int r = kr0 + k * 16 + (lane & 15);
#pragma unroll
          for (int n = 0; n < OT; n += 2) {
            uint32_t b[4];
            ldsm4t(b, vs + r * X::kRow + X::v_chunk(r, n + (lane >> 4)) * 16);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t c0 = __byte_perm(b[2 * e], 0, 0x3120);
              const uint32_t c1 = __byte_perm(b[2 * e + 1], 0, 0x3120);
              const uint32_t va[4] = {e4m3x2_f16x2(c0 & 0xffff), e4m3x2_f16x2(c0 >> 16),
                                      e4m3x2_f16x2(c1 & 0xffff), e4m3x2_f16x2(c1 >> 16)};
              mma_f16(o[n + e], va, p0, p1);
            }
          }
        }
      }
    } else if constexpr (!kF32 && !kScaled) {
#pragma unroll
      for (int k = 0; k < N / 16; ++k) {
        const uint32_t pa[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]),
                                pack_bf16(s[2 * k][2], s[2 * k][3]),
                                pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]),
                                pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
        const int r = kr0 + k * 16 + (lane & 15);
#pragma unroll
        for (int n = 0; n < OT; n += 2) {
          uint32_t b[4];
          ldsm4t(b, vs + r * X::kRow + X::v_chunk(r, n + (lane >> 4)) * 16);
          mma_bf16(o[n], pa, b[0], b[1]);
          mma_bf16(o[n + 1], pa, b[2], b[3]);
        }
      }
    } else if constexpr (!kF32) {
      // 16 keys by 32 values a load; of the byte pair a thread gets for a key,
      // the first goes to an even output tile and the second to an odd one:
      // accumulator (2n + e, column c) is value 16 n + 2 c + e
#pragma unroll
      for (int k = 0; k < N / 16; ++k) {
        const uint32_t pa[4] = {pack_f16x2(s[2 * k][0], s[2 * k][1]),
                                pack_f16x2(s[2 * k][2], s[2 * k][3]),
                                pack_f16x2(s[2 * k + 1][0], s[2 * k + 1][1]),
                                pack_f16x2(s[2 * k + 1][2], s[2 * k + 1][3])};
        const int r = kr0 + k * 16 + (lane & 15);
#pragma unroll
        for (int n = 0; n < OT / 2; n += 2) {
          uint32_t b[4];
          ldsm4t(b, vs + r * X::kRow + X::v_chunk(r, n + (lane >> 4)) * 16);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t c0 = __byte_perm(b[2 * e], 0, 0x3120);
            const uint32_t c1 = __byte_perm(b[2 * e + 1], 0, 0x3120);
            mma_f16(o[2 * (n + e)], pa, e4m3x2_f16x2(c0 & 0xffff), e4m3x2_f16x2(c1 & 0xffff));
            mma_f16(o[2 * (n + e) + 1], pa, e4m3x2_f16x2(c0 >> 16), e4m3x2_f16x2(c1 >> 16));
          }
        }
      }
    } else {
      // The tensor cores cut the low bits of a product that joins a larger sum.
      // fp32 results keep their precision with a fresh accumulator for each
      // tile of keys (each 16 values of a score), added to the sum in fp32.
      float fresh[OT][4];
#pragma unroll
      for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) fresh[i][j] = 0.f;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        // keys 2 t4 and 2 t4 + 1 of each 8 are this thread's k indices
        uint32_t h[4], e[4];
        split_tf32(s[k][0], h[0], e[0]), split_tf32(s[k][2], h[1], e[1]);
        split_tf32(s[k][1], h[2], e[2]), split_tf32(s[k][3], h[3], e[3]);
        if constexpr (kScaled) {
          const int r = kr0 + k * 8 + (lane & 7);
#pragma unroll
          for (int n = 0; n < OT / 2; n += 4) {
            uint32_t b[4];
            ldsm4t(b, vs + r * X::kRow + X::v_chunk(r, n + (lane >> 3)) * 16);
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) {
              const uint32_t c0 = e4m3x2_f16x2(b[e2] & 0xffff), c1 = e4m3x2_f16x2(b[e2] >> 16);
              mma_tf32(fresh[2 * (n + e2)], e, __float_as_uint(half_lo(c0)), __float_as_uint(half_lo(c1)));
              mma_tf32(fresh[2 * (n + e2)], h, __float_as_uint(half_lo(c0)), __float_as_uint(half_lo(c1)));
              mma_tf32(fresh[2 * (n + e2) + 1], e, __float_as_uint(half_hi(c0)), __float_as_uint(half_hi(c1)));
              mma_tf32(fresh[2 * (n + e2) + 1], h, __float_as_uint(half_hi(c0)), __float_as_uint(half_hi(c1)));
            }
          }
        } else {
          const int ra = kr0 + k * 8 + 2 * t4, rb = ra + 1;
#pragma unroll
          for (int n = 0; n < OT; ++n) {
            const int d = n * 8 + g;
            const float va = *reinterpret_cast<const float*>(vs + ra * X::kRow + X::v_chunk(ra, d >> 2) * 16 + (d & 3) * 4);
            const float vb = *reinterpret_cast<const float*>(vs + rb * X::kRow + X::v_chunk(rb, d >> 2) * 16 + (d & 3) * 4);
            uint32_t ah, al, bh, bl;
            split_tf32(va, ah, al), split_tf32(vb, bh, bl);
            mma_tf32(fresh[n], h, al, bl);
            mma_tf32(fresh[n], e, ah, bh);
            mma_tf32(fresh[n], h, ah, bh);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = o[i][j] * keep[j >> 1] + fresh[i][j];
    }
  }
  cp_wait<0>();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (kFew) {
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l[u] += __shfl_xor_sync(0xffffffffu, l[u], w);
    } else {
      l[u] = quad_sum(l[u]);
    }
  }
  if (kScaled)
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] *= two_to(-wexp[kFew ? j & 1 : j >> 1]);

  // maxima in base 2 from here on
#pragma unroll
  for (int u = 0; u < 2; ++u) m[u] = m[u] == -INFINITY ? m[u] : m[u] * rscale[u];

  // value index of accumulator element (tile n, j)
  auto value_of = [&](int n, int j) {
    if (kFew) return kScaled ? n * 16 + 2 * g + (j >> 1) : n * 16 + g + 8 * (j >> 1);
    return kScaled ? (n >> 1) * 16 + (t4 * 2 + (j & 1)) * 2 + (n & 1) : n * 8 + t4 * 2 + (j & 1);
  };
  const int nrow = rN - r0;
  if constexpr (KS) {
    // ---- the four warps' sums meet in shared memory
    __syncthreads();
    float* jo = reinterpret_cast<float*>(smem);  // [4][16][DP], then the CTA's own [16][DP]
    float2* jm = reinterpret_cast<float2*>(smem + 5 * 16 * DP * 4);  // [4][16], then [16]
    float* co = jo + 4 * 16 * DP;
    float2* cm = jm + 4 * 16;
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        jo[(warp * 16 + (kFew ? 2 * t4 + (j & 1) : g + 8 * (j >> 1))) * DP + value_of(i, j)] =
            o[i][j];
    if (kFew ? g == 0 : t4 == 0) {
      jm[warp * 16 + (kFew ? 2 * t4 : g)] = make_float2(m[0], l[0]);
      jm[warp * 16 + (kFew ? 2 * t4 + 1 : g + 8)] = make_float2(m[1], l[1]);
    }
    __syncthreads();
    const int quads = D >> 2;
    // four values of a row at a time, joined in the order of warps and splits
    for (int i = threadIdx.x; i < nrow * quads; i += kThreads) {
      const int r = i / quads, d = (i - r * quads) * 4;
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, jm[w * 16 + r].x);
      const float base = mm == -INFINITY ? 0.f : mm;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = ex2(jm[w * 16 + r].x - base);
        const float4 y = *reinterpret_cast<const float4*>(jo + (w * 16 + r) * DP + d);
        ll += jm[w * 16 + r].y * f;
        x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
      }
      if (!p.joined) {
        const int64_t slot = (p.extra + split) * p.out_rows + out_row(r0 + r);
        *reinterpret_cast<float4*>(p.part_o + slot * D + d) = x;
        if (d == 0) p.part_ml[slot] = make_float2(mm, ll);
      } else {
        *reinterpret_cast<float4*>(co + r * DP + d) = x;
        if (d == 0) cm[r] = make_float2(mm, ll);
      }
    }
    if (!p.joined) return;
    // ---- the splits' sums, and the extra ones, in this split's share of the rows
    cg::cluster_group cluster = cg::this_cluster();
    if (p.splits > 1)
      cluster.sync();
    else
      __syncthreads();
    for (int i = split * kThreads + threadIdx.x; i < nrow * quads; i += p.splits * kThreads) {
      const int r = i / quads, d = (i - r * quads) * 4;
      const int64_t orow = out_row(r0 + r);
      float mm = -INFINITY, ll = 0.f;
      for (int c = 0; c < p.splits; ++c)
        mm = fmaxf(mm, (p.splits > 1 ? cluster.map_shared_rank(cm, c) : cm)[r].x);
      for (int c = 0; c < p.extra; ++c) mm = fmaxf(mm, __ldg(p.part_ml + c * p.out_rows + orow).x);
      const float base = mm == -INFINITY ? 0.f : mm;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int c = 0; c < p.extra; ++c) {
        const int64_t slot = c * p.out_rows + orow;
        const float2 ml = __ldg(p.part_ml + slot);
        add_part<true>(x, ml, base, 1.f, p.part_o + slot * D + d);
        ll += ml.y * ex2(ml.x - base);
      }
      for (int c = 0; c < p.splits; ++c) {
        const float2 ml = (p.splits > 1 ? cluster.map_shared_rank(cm, c) : cm)[r];
        add_part<false>(x, ml, base, 1.f, (p.splits > 1 ? cluster.map_shared_rank(co, c) : co) + r * DP + d);
        ll += ml.y * ex2(ml.x - base);
      }
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      store4(static_cast<QT*>(a.out) + orow * D + d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    }
    if (p.splits > 1) cluster.sync();  // nobody leaves while its sums are read
  } else if (!p.joined) {  // kByRows
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (row[u] >= rN) continue;
      const int64_t slot = (p.extra + split) * p.out_rows + out_row(row[u]);
#pragma unroll
      for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (value_of(i, j) < D) p.part_o[slot * D + value_of(i, j)] = o[i][2 * u + j];
      if (t4 == 0) p.part_ml[slot] = make_float2(m[u], l[u]);
    }
  } else {
    // ---- 64 rows to shared memory, then joined with the extra partial
    // results and written four values a thread
    __syncthreads();
    float* co = reinterpret_cast<float*>(smem);  // [64][DP + 4]
    float2* cm = reinterpret_cast<float2*>(smem + 64 * (DP + 4) * 4);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = wrow + g + 8 * u;
#pragma unroll
      for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) co[r * (DP + 4) + value_of(i, j)] = o[i][2 * u + j];
      if (t4 == 0) cm[r] = make_float2(m[u], l[u]);
    }
    __syncthreads();
    // a row's joint maximum and the inverse of its sum
    if (threadIdx.x < nrow) {
      const float2 own = cm[threadIdx.x];
      const int64_t orow = out_row(r0 + threadIdx.x);
      float mm = own.x;
      for (int c = 0; c < p.extra; ++c) mm = fmaxf(mm, __ldg(p.part_ml + c * p.out_rows + orow).x);
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = own.y * ex2(own.x - base);
      for (int c = 0; c < p.extra; ++c) {
        const float2 ml = __ldg(p.part_ml + c * p.out_rows + orow);
        ll += ml.y * ex2(ml.x - base);
      }
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      cm[threadIdx.x] = make_float2(base, inv);
      co[threadIdx.x * (DP + 4) + DP] = ex2(own.x - base) * inv;
      *reinterpret_cast<int*>(&co[threadIdx.x * (DP + 4) + DP + 1]) = (int)orow;
    }
    __syncthreads();
    // kBatch pieces of four values a thread at a time, their loads together
    const int quads = D >> 2;
    constexpr int kBatch = 8;
    for (int i0 = threadIdx.x; i0 < nrow * quads; i0 += kBatch * kThreads) {
      float4 x[kBatch];
      int64_t orow[kBatch];
      int mrow[kBatch];
      float2 bi[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int i = min(i0 + e * kThreads, nrow * quads - 1), r = i / quads;
        const float* own = co + r * (DP + 4);
        bi[e] = cm[r];
        orow[e] = *reinterpret_cast<const int*>(own + DP + 1);
        mrow[e] = (int)orow[e];
        x[e] = *reinterpret_cast<const float4*>(own + (i - r * quads) * 4);
        x[e].x *= own[DP], x[e].y *= own[DP], x[e].z *= own[DP], x[e].w *= own[DP];
        orow[e] = orow[e] * D + (i - r * quads) * 4;
      }
      for (int c = 0; c < p.extra; ++c) {
        const float* po = p.part_o + c * p.out_rows * D;
        const float2* pm = p.part_ml + c * p.out_rows;
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
          add_part<true>(x[e], __ldg(pm + mrow[e]), bi[e].x, bi[e].y, po + orow[e]);
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e)
        if (i0 + e * kThreads < nrow * quads)
          store4(static_cast<QT*>(a.out) + orow[e], x[e].x, x[e].y, x[e].z, x[e].w);
    }
  }
}

// joins the partial results of an output row, in the order of the splits
template <typename T>
__global__ void __launch_bounds__(128) k_attn_join(const float* part_o, const float2* part_ml,
                                                   int splits, int64_t out_rows, int D, T* out) {
  const int per = D >> 2;  // 4 values a thread
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= out_rows * per) return;
  const int64_t r = i / per;
  const int d = (int)(i - r * per) * 4;
  float m = -INFINITY, l = 0.f, x[4] = {};
  for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[s * out_rows + r].x);
  const float base = m == -INFINITY ? 0.f : m;
  for (int s = 0; s < splits; ++s) {
    const float2 ml = part_ml[s * out_rows + r];
    if (ml.y == 0.f) continue;  // empty: its values may be unwritten
    const float f = ex2(ml.x - base);
    const float4 v = *reinterpret_cast<const float4*>(part_o + (s * out_rows + r) * D + d);
    l += ml.y * f;
    x[0] += v.x * f, x[1] += v.y * f, x[2] += v.z * f, x[3] += v.w * f;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[r * D + d + e] = Elt<T>::from_f(l == 0.f ? 0.f : x[e] / l);
}

// How a call is cut: splits of the own columns and of the prefix, and whether
// the own part's clusters join everything (else k_attn_join does).
struct Plan {
  Mode own, prefix;
  bool joined, prefix_tc;
  int own_splits, prefix_splits;
  PrefixTcPlan tc;
  int64_t out_rows, bytes;
};

// CTAs counted as resident at a time (148 SMs, two each): calls of as many are
// not split, smaller ones to about twice as many. Both sides, 16 / 8 heads of 64:
// with 148 in its place 20 rows of 8192 columns in e4m3 take 53.8 us against 39.0
// (160 CTAs, then whole), but 8 rows of 2100 in bf16 10.3 against 16.4 and one of
// 32,768 22.6 against 36.8 (fewer partial results to join); with 592 they take
// 22.6 and 63.2.
constexpr int kSlots = 296;
// Keys of a split, at least. With 64 one row of 1089 columns takes 10.3 us against
// 8.2; with 256 one of 2100 8.2 against 12.0, but 4 rows behind a prefix of 509 in
// fp32 20.3 against 16.4.
constexpr int64_t kMinKeys = 128;
constexpr int kMaxCluster = 8;

int splits_for(int64_t keys, int64_t ctas) {
  if (keys <= kMinKeys || ctas >= kSlots) return 1;
  const int64_t want = (2 * kSlots) / ctas;
  const int64_t most = (keys + kMinKeys - 1) / kMinKeys;
  return (int)(want < most ? want : most);
}

// Up to 8 rows transposed took 64 rows in e4m3 from 20.5 to 16.9 us, 16-bit
// queries only: split tf32 operands have no transposed form here.
Mode mode_for(int dtype, int64_t rows) {
  return rows <= 8 && dtype == MEP_BF16 ? kFewRows : rows <= 16 ? kByKeys : kByRows;
}
int rows_of(Mode m) { return m == kFewRows ? 8 : m == kByKeys ? 16 : 64; }

// Rows of a key/value head from which the prefix is tcgen05's. Both sides at 128
// rows on each of 8 heads of 64, tcgen05 against warp-level products: 4096 columns
// 24.6 us against 31.3, 16,384 36.9 against 49.7, but 300 columns 25.0 against 18.5
// and 1024 22.6 against 18.5 (too few units for the SMs); 6144 rows on each of 8
// heads of 128 behind 4099, the whole call, 136 against 477. At 64 rows: 4096 columns 18.5 both, 16,384 28.7 against
// 34.9, 1024 18.5 against 14.4.
constexpr int64_t kTcRows = 128;

Plan plan_for(int dtype, int64_t batch, int64_t tokens, int q_heads, int kv_heads, int head_dim,
              int64_t capacity, int64_t col, int64_t prefix_cols) {
  Plan p{};
  const int group = q_heads / kv_heads;
  const int64_t keys = col < 0 ? capacity : col + tokens;
  const int64_t own_rows = tokens * group, pre_rows = batch * own_rows;
  p.own = mode_for(dtype, own_rows);
  p.prefix = mode_for(dtype, pre_rows);
  const int ot = rows_of(p.own), pt = rows_of(p.prefix);
  p.own_splits = splits_for(keys, batch * kv_heads * ((own_rows + ot - 1) / ot));
  p.prefix_splits =
      prefix_cols > 0 ? splits_for(prefix_cols, kv_heads * ((pre_rows + pt - 1) / pt)) : 0;
  p.prefix_tc = dtype == MEP_BF16 && prefix_cols > 0 && pre_rows >= kTcRows;
  if (p.prefix_tc) {
    p.tc = plan_prefix_tc(pre_rows, kv_heads, prefix_cols);
    p.prefix_splits = p.tc.slots;
  }
  // up to twice as many splits as a cluster holds cost more, with another launch
  // to join them, than the cluster's 8: one row of 1089 columns 10.3 us against
  // 8.2, 8 rows of 2100 in e4m3 14.4 against 11.9
  if (p.own != kByRows && p.own_splits <= 2 * kMaxCluster && p.own_splits > kMaxCluster)
    p.own_splits = kMaxCluster;
  p.joined = p.own != kByRows ? p.own_splits <= kMaxCluster : p.own_splits == 1;
  p.out_rows = batch * tokens * q_heads;
  const int parts = p.prefix_splits + (p.joined ? 0 : p.own_splits);
  p.bytes = parts * p.out_rows * (head_dim * 4 + 8);
  return p;
}

template <typename QT, typename CT, int DP, int MODE, bool PREFIX>
int run_part(const PartArgs& p, int64_t mats, cudaStream_t st) {
  using X = Tile<QT, CT, DP, MODE>;
  auto* k = k_attn_part<QT, CT, DP, MODE, PREFIX>;
  static SmemLimit limit;
  if (const int e = limit.raise(reinterpret_cast<const void*>(k), X::kSmem)) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(mats * p.row_tiles * p.splits), (unsigned)p.a.kv_heads);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = X::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = X::KS && p.joined ? p.splits : 1, at.val.clusterDim.y = 1,
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, k, p);
}
template <typename QT, typename CT, int MODE, bool PREFIX>
int run_dp(const PartArgs& p, int64_t mats, cudaStream_t st) {
  return p.a.head_dim <= 64 ? run_part<QT, CT, 64, MODE, PREFIX>(p, mats, st)
                            : run_part<QT, CT, 128, MODE, PREFIX>(p, mats, st);
}
template <typename QT, typename CT, bool PREFIX>
int run_mode(Mode m, PartArgs& p, int64_t mats, cudaStream_t st) {
  p.row_tiles = (p.rows + rows_of(m) - 1) / rows_of(m);
  if constexpr (sizeof(QT) == 2)
    if (m == kFewRows) return run_dp<QT, CT, kFewRows, PREFIX>(p, mats, st);
  return m == kByKeys ? run_dp<QT, CT, kByKeys, PREFIX>(p, mats, st)
                      : run_dp<QT, CT, kByRows, PREFIX>(p, mats, st);
}

template <typename QT, typename CT>
int run_attention(const AttnArgs& a, const Plan& pl, void* workspace, cudaStream_t st) {
  const int group = a.q_heads / a.kv_heads;
  const int parts = pl.prefix_splits + (pl.joined ? 0 : pl.own_splits);
  float* po = parts ? static_cast<float*>(workspace) : nullptr;
  float2* pm = parts ? reinterpret_cast<float2*>(po + parts * pl.out_rows * a.head_dim) : nullptr;
  if (pl.prefix_tc) {
    if (const int rc = launch_prefix_tc(a, pl.tc, pl.out_rows, po, pm, st)) return rc;
  } else if (pl.prefix_splits) {
    PartArgs x{a, group, (int)(a.batch * a.tokens * group), 0, pl.prefix_splits, 0, 0, pl.out_rows,
               po, pm};
    if (const int rc = run_mode<QT, QT, true>(pl.prefix, x, 1, st)) return rc;
  }
  PartArgs p{a, group, (int)(a.tokens * group), 0, pl.own_splits, pl.joined, pl.prefix_splits,
             pl.out_rows, po, pm};
  if (const int rc = run_mode<QT, CT, false>(pl.own, p, a.batch, st)) return rc;
  if (!pl.joined) {
    const int64_t n = pl.out_rows * (a.head_dim / 4);
    k_attn_join<QT><<<(unsigned)((n + 127) / 128), 128, 0, st>>>(po, pm, parts, pl.out_rows,
                                                                  a.head_dim,
                                                                  static_cast<QT*>(a.out));
  }
  return 0;
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
  *bytes_out = batch && tokens ? plan_for(dtype, batch, tokens, q_heads, kv_heads, head_dim, capacity, col,
                                          prefix_cols)
                                     .bytes
                               : 0;
  return MEP_OK;
}

extern "C" int mep_cache_attention(const mep_attention_args* x, void* stream) {
  const char* op = "mep_cache_attention";
  if (!x) return serve_invalid(op, "null arguments");
  if (const char* why = bad_heads(x->dtype, x->cache_dtype, x->batch, x->tokens, x->q_heads,
                                  x->kv_heads, x->head_dim))
    return serve_invalid(op, why);
  if (x->capacity < 0 || x->prefix_cols < 0 || x->prompt_cols < 0)
    return serve_invalid(op, "negative columns");
  if (x->capacity > 0x7fffffff - 1024 || x->prefix_cols > 0x7fffffff - 1024)
    return serve_invalid(op, "columns up to 2^31 - 1025");
  if (!x->col_dev && (x->col < 0 || x->col > x->capacity - x->tokens))
    return serve_invalid(op, "columns [col, col + tokens) do not fit the cache");
  if (!(x->scale >= -0x1p127 && x->scale <= 0x1p127))  // times log2 e it still has to fit fp32
    return serve_invalid(op, "scale must be finite, up to 2^127");
  if (x->batch == 0 || x->tokens == 0) return MEP_OK;
  const AttnArgs a{x->batch, x->tokens, (int)x->q_heads, (int)x->kv_heads, (int)x->head_dim,
                   {x->q, x->q_sb, x->q_st, x->q_sh},
                   {x->k_cache, x->v_cache, x->k_scale, x->v_scale, x->capacity}, x->lengths,
                   x->prompt_cols, x->col, x->col_dev, x->k_prefix, x->v_prefix, x->prefix_cols,
                   (float)x->scale, x->out};
  if (!x->q || !x->k_cache || !x->v_cache || !x->out) return serve_invalid(op, "null tensor");
  if (x->prefix_cols > 0 && (!x->k_prefix || !x->v_prefix))
    return serve_invalid(op, "null prefix");
  if (x->cache_dtype == MEP_E4M3 && (!x->k_scale || !x->v_scale))
    return serve_invalid(op, "a quantised cache needs k_scale and v_scale");
  if (bad_strides(a.q, x->dtype == MEP_BF16 ? 2 : 4) || !aligned16(x->k_cache) ||
      !aligned16(x->v_cache) || !aligned16(x->k_prefix) || !aligned16(x->v_prefix) ||
      !aligned16(x->out))
    return serve_invalid(op, "tensors and row strides must be multiples of 16 bytes");
  const Plan pl = plan_for((int)x->dtype, x->batch, x->tokens, a.q_heads, a.kv_heads, a.head_dim,
                           x->capacity, x->col_dev ? -1 : x->col, x->prefix_cols);
  if (pl.bytes > 0 &&
      (!x->workspace || x->workspace_bytes < pl.bytes || !aligned16(x->workspace)))
    return serve_invalid(op, "workspace of " + std::to_string(pl.bytes) + " bytes needed");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool e4m3 = x->cache_dtype == MEP_E4M3;
  int rc;
  if (x->dtype == MEP_BF16)
    rc = e4m3 ? run_attention<__nv_bfloat16, uint8_t>(a, pl, x->workspace, st)
              : run_attention<__nv_bfloat16, __nv_bfloat16>(a, pl, x->workspace, st);
  else
    rc = e4m3 ? run_attention<float, uint8_t>(a, pl, x->workspace, st)
              : run_attention<float, float>(a, pl, x->workspace, st);
  if (rc < 0) return serve_invalid(op, "tensor map error " + std::to_string(rc));
  if (rc) return serve_cuda(op, (cudaError_t)rc);
  return serve_launched(op);
}
