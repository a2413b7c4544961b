// cbk_host.hpp -- what the files of C entry points share: error messages, the device of a call, and the
// arrival counters of in-dispatch combines (abi.cpp has them).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cbk {

// Sets the calling thread's message (cbk_last_error) and returns `code`.
int fail(int code, const char* fmt, ...);
int hip_fail(hipError_t e, const char* what);

// Switches to `device` for the duration of a call (the reference's CUDAGuard).
struct DeviceGuard {
    int prev = -1;
    hipError_t err = hipSuccess;
    explicit DeviceGuard(int device) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != device) err = hipSetDevice(device);
        else if (err != hipSuccess) prev = -1;
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
    }
};

// Windows of arrival counters: kinds of calls, and the counters of a window.
enum { WIN_DECODE = 0, WIN_GEMM = 1, WIN_ATTN = 2, WIN_KINDS = 3 };
constexpr int SPLIT_COUNTERS = 4096;

// The counter window of a cache attention call on `device` (made current by the caller), or nullptr.
uint32_t* attn_window(int device, hipStream_t stream);

}  // namespace cbk
