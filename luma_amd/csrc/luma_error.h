// The library's last-error text (luma_last_error), which every source sets:
// defined in luma_step.hip.
#pragma once
#include <hip/hip_runtime.h>

namespace luma {

// Records `msg` (and the HIP error's text); returns the status to return.
int fail(const char *msg, hipError_t e = hipSuccess);

// 0, or fail() with the error that the launch before left.
int check_launch(const char *what);

}  // namespace luma
