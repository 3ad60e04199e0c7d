// Host helpers shared by the C entry points: the calling thread's error message,
// device properties, the device switch of a call.  Defined in cvs_capi.hip.
#pragma once

#include <hip/hip_runtime.h>

namespace cvs {

// Sets the calling thread's message (cvs_last_error) and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int hip_fail(hipError_t e, const char* what);

struct DevInfo {
  bool ready = false;
  bool gfx950 = false;
  int cus = 0;
  char arch[64] = {0};
};

int dev_info(int device, DevInfo* out);

// Switches to `device` for the lifetime of the guard (the reference's CUDAGuard).
struct DeviceGuard {
  int prev = -1;
  bool switched = false;
  hipError_t err = hipSuccess;
  explicit DeviceGuard(int device) {
    err = hipGetDevice(&prev);
    if (err == hipSuccess && prev != device) {
      err = hipSetDevice(device);
      switched = (err == hipSuccess);
    }
  }
  ~DeviceGuard() {
    if (switched) (void)hipSetDevice(prev);
  }
};

}  // namespace cvs
