// What every C entry point goes through: exceptions become return codes and a message, work runs on the operands' GPU.
#pragma once
#include "rpu_host.h"

#include <hip/hip_runtime.h>

#include <string>

namespace rpu_amd {

#define RPU_HIP_CHECK(expr)                                                                         \
  do {                                                                                              \
    hipError_t _e = (expr);                                                                         \
    if (_e != hipSuccess) {                                                                         \
      throw RpuError(std::string("HIP error: ") + hipGetErrorString(_e) + " in " #expr);            \
    }                                                                                               \
  } while (0)

class DeviceGuard {
public:
  explicit DeviceGuard(int device) {
    RPU_HIP_CHECK(hipGetDevice(&prev_));
    if (device != prev_) {
      RPU_HIP_CHECK(hipSetDevice(device));
      changed_ = true;
    }
  }
  ~DeviceGuard() {
    if (changed_) (void)hipSetDevice(prev_);
  }

private:
  int prev_ = 0;
  bool changed_ = false;
};

// message of the last failure on the calling thread (rpu_last_error)
std::string &last_error();

template <typename F> int guarded(F &&f) {
  try {
    f();
    return 0;
  } catch (const std::exception &e) {
    last_error() = e.what();
    return 1;
  } catch (...) {
    last_error() = "unknown error";
    return 2;
  }
}

} // namespace rpu_amd
