// Arguments of cache_attention's kernels (mep_attn.cu: CUDA-core staging and
// warp-level products; mep_attn_tc.cu: the shared prefix on tcgen05).
#pragma once

#include <cstdint>
#include "mep_serve.cuh"

namespace mep {

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

constexpr float kLog2e = 1.4426950408889634f;
// Least factor of the scores: a masked score is -inf and has to stay that, which
// it would not times 0. Scores below 2^100 all weigh alike under it, as under 0.
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Partial results of the prefix on tcgen05: slots [0, slots) of part_o
// (slots, out_rows, head_dim) and part_ml (slots, out_rows). Empty slots have
// the sum 0 and unwritten values.
struct PrefixTcPlan {
  int ctas, slots;
};
PrefixTcPlan plan_prefix_tc(int64_t rows, int kv_heads, int64_t prefix_cols);
// 0, a cudaError_t, or a negative tensor-map error
int launch_prefix_tc(const AttnArgs& a, const PrefixTcPlan& plan, int64_t out_rows, float* part_o,
                     float2* part_ml, cudaStream_t st);

}  // namespace mep
