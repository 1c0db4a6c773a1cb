// What kernels report to the host: two words of device memory, a wait that gave up and a bad argument (0: neither).  They are apart
// since kernels whose waits gave up look at the first on their way out, for copies that may still be in flight, and since an index
// that the device found to be bad must not take the place of a wait's code.
#pragma once

#include <cuda_runtime.h>

namespace axb {

enum : int {
  kStatusOk = 0,
  kStatusWaitTimeoutProducer = 1,
  kStatusWaitTimeoutMma = 2,
  kStatusWaitTimeoutEpilogue = 3,
  kStatusWaitTimeoutPeer = 4,
  kStatusBadArgument = 5,
};

__device__ __forceinline__ void report_bad_argument(int* status) { *reinterpret_cast<volatile int*>(status + 1) = kStatusBadArgument; }

}  // namespace axb
