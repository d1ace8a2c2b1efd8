// What the C ABI's files share: the thread's error message and the device
// switch of a launch.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

namespace shk {

// Sets amd_strix_halo_kernels_last_error of this thread and returns 1 (capi.hip).
int capi_fail(const std::string& msg);
int capi_fail_hip(const char* what, hipError_t err);
void capi_clear_error();

// Makes `device` current for the duration of a launch and restores the
// caller's device afterwards.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device) {
    if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
    if (prev_ != device) {
      err_ = hipSetDevice(device);
      switched_ = err_ == hipSuccess;
    }
  }
  ~DeviceGuard() {
    if (switched_ && prev_ >= 0) (void)hipSetDevice(prev_);
  }
  hipError_t error() const { return err_; }

 private:
  int prev_ = -1;
  bool switched_ = false;
  hipError_t err_ = hipSuccess;
};

// Runs a C entry's body; an exception (out of host memory) ends as rc 1.
template <class F>
int capi_entry(F&& body) {
  try {
    capi_clear_error();
    return body();
  } catch (const std::exception& e) {
    try {
      return capi_fail(e.what());
    } catch (...) {
      return 1;
    }
  } catch (...) {
    return 1;
  }
}

}  // namespace shk
