// Shared by the decode-step operators (mep_kv.cu, mep_attn.cu, mep_sample.cu):
// the layout of a layer's key/value cache, argument errors and launch checks.
#pragma once

#include <atomic>
#include <cstdint>
#include <string>

#include <cuda_runtime.h>
#include "mep_internal.h"

namespace mep {
void set_global_error(const std::string& msg);  // mep_api.cu: read by mep_last_error(NULL)

// head widths the decode-step operators take: multiples of 16 up to this
constexpr int kMaxHeadDim = 128;

inline int serve_invalid(const char* op, const std::string& msg) {
  set_global_error(std::string(op) + ": " + msg);
  return MEP_ERR_INVALID;
}
inline int serve_cuda(const char* op, cudaError_t e) {
  set_global_error(std::string(op) + ": " + cudaGetErrorString(e));
  return MEP_ERR_CUDA;
}
// status of the launches just enqueued
inline int serve_launched(const char* op) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return MEP_OK;
  set_global_error(std::string(op) + ": kernel launch: " + cudaGetErrorString(e));
  return MEP_ERR_CUDA;
}
// Dynamic shared memory limit of a kernel, raised once on each device.
class SmemLimit {
 public:
  int raise(const void* kernel, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done_.load(std::memory_order_acquire) & bit) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int)e;
    done_.fetch_or(bit, std::memory_order_release);
    return 0;
  }

 private:
  std::atomic<uint64_t> done_{0};
};
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// One layer of a key/value cache: (batch, kv_heads, capacity, head_dim), rows
// contiguous; quantised rows carry one fp32 scale each, (batch, kv_heads,
// capacity).
struct CacheView {
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  int64_t capacity;
};

// q, k or v of the new tokens: element strides of (batch, token, head), the
// head's values contiguous
struct HeadsView {
  const void* p;
  int64_t sb, st, sh;
};

// Checks shared by the entry points that take heads; null when they hold.
inline const char* bad_heads(int64_t dtype, int64_t cache_dtype, int64_t batch, int64_t tokens,
                             int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
  if (dtype != MEP_F32 && dtype != MEP_BF16) return "dtype must be MEP_F32 or MEP_BF16";
  if (cache_dtype != dtype && cache_dtype != MEP_E4M3)
    return "the cache must be in the model dtype or in MEP_E4M3";
  if (batch < 0 || tokens < 0) return "negative batch or token count";
  if (batch > 65535 || tokens > (1 << 24)) return "batch up to 65535, tokens up to 2^24";
  if (kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0 || q_heads > 1024)
    return "q_heads must be a multiple of kv_heads, up to 1024";
  // rows are counted in 32 bits, and up to whole tiles of 256
  if (batch * tokens * q_heads > 0x7fffffff - 1024)
    return "batch * tokens * q_heads up to 2^31 - 1025";
  if (head_dim < 16 || head_dim > kMaxHeadDim || head_dim % 16 != 0)
    return "head_dim must be a multiple of 16 up to 128";
  return nullptr;
}
inline bool bad_strides(const HeadsView& h, int elt) {
  const int64_t unit = 16 / elt;
  return !aligned16(h.p) || h.sb % unit || h.st % unit || h.sh % unit;
}

}  // namespace mep
