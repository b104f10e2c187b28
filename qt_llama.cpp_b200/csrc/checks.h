// checks.h — argument checks shared by the C-ABI entry points (internal), so
// that every entry point that takes the same shapes accepts the same ones.
#pragma once
#include <stdint.h>

#include "../../include/mrml_moe.h"
#include "kernels.h"

#define MRML_TRY(expr)                 \
  do {                                 \
    const int _st = (expr);            \
    if (_st != MRML_OK) return _st;    \
  } while (0)

#define MRML_LAUNCH(expr)              \
  do {                                 \
    mrml::LaunchMark _mark(s);         \
    MRML_TRY(mrml::cuda_status(expr)); \
  } while (0)

namespace mrml {

// MRML_OK if the current device is an sm_100 part (mrml_moe.cu).
int check_device();

// Records the profiling events of mrml_moe_profile_events around a launch
// (mrml_moe.cu).
struct LaunchMark {
  cudaStream_t s;
  explicit LaunchMark(cudaStream_t st);
  ~LaunchMark();
};

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline int cuda_status(cudaError_t e) { return e == cudaSuccess ? MRML_OK : MRML_ERR_CUDA; }
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Router shapes and pointers (mrml_moe_router, mrml_moe_router_noalloc,
// the router half of mrml_moe_forward).
inline int check_router_args(const float* W, const float* x, const float* logits, const int32_t* ids,
                             const float* probs, int H, int E, int K, int T) {
  if (H <= 0 || E <= 0 || K <= 0 || T < 0) return MRML_ERR_INVALID_ARGUMENT;
  if (K > E) return MRML_ERR_INVALID_ARGUMENT;
  if (E > kMaxExperts || K > kMaxTopK) return MRML_ERR_UNSUPPORTED;
  if (T > 0 && (!W || !x || !logits || !ids || !probs)) return MRML_ERR_INVALID_ARGUMENT;
  return MRML_OK;
}

}  // namespace mrml
