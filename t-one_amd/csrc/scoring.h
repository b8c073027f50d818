// The phrase operators: frame pages and slot maps (frames.hip), scores of given tokens per row (scores.hip) and CTC
// alignment (align.hip).  They are stateless: every buffer is the caller's, the C entry points stand at the end of each file.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include <exception>
#include <string>

#include "../../include/tonehip.h"

namespace tone {

// records the message tone_last_error() returns; returns `code`
int set_error(int code, const std::string& msg);

using Bf16 = __bf16;

__device__ __forceinline__ float load_elem(const float* p) { return *p; }
__device__ __forceinline__ float load_elem(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_elem(const Bf16* p) { return static_cast<float>(*p); }
// one rounding to nearest even; an infinity or a NaN stays one
__device__ __forceinline__ void store_elem(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_elem(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_elem(Bf16* p, float v) { *p = static_cast<Bf16>(v); }

inline bool known_type(int t) { return t == TONE_TYPE_FP32 || t == TONE_TYPE_FP16 || t == TONE_TYPE_BF16; }

// A launch's threads are counted in 32 bits, and loops over a row's frames run in 32-bit integers with room for a stride.
constexpr int64_t kMaxThreads = UINT32_MAX;
constexpr int kMaxFrames = 1 << 29;

// whether a pointer lies on a whole element of its type
inline bool aligned(const void* p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type == TONE_TYPE_FP32 ? 3 : 1)) == 0; }

// The calling thread's device for the life of an entry point, the former one afterwards.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    err_ = hipGetDevice(&before_);
    if (err_ == hipSuccess && before_ != device) {
      err_ = hipSetDevice(device);
      moved_ = err_ == hipSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  hipError_t error() const { return err_; }

 private:
  int before_ = 0;
  bool moved_ = false;
  hipError_t err_ = hipSuccess;
};

// Runs an entry point's launch on `device`: no exception crosses the C boundary, HIP errors become TONE_E_HIP.
template <typename F>
int launch_on(int device, const char* what, F&& launch) noexcept {
  try {
    OnDevice on(device);
    hipError_t e = on.error();
    if (e == hipSuccess) e = launch();
    if (e != hipSuccess) return set_error(TONE_E_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return TONE_OK;
  } catch (const std::exception&) {
    return TONE_E_HIP;
  }
}

inline int refuse(const char* what, const char* why) noexcept {
  try {
    return set_error(TONE_E_INVALID, std::string(what) + ": " + why);
  } catch (const std::exception&) {
    return TONE_E_INVALID;
  }
}

}  // namespace tone
