// What the library's translation units share on the host side.
#pragma once
#include <hip/hip_runtime.h>

// Records the message erf_last_error() returns and gives back 1.
__attribute__((visibility("hidden"))) int host_fail(const char *fmt, ...) __attribute__((format(printf, 1, 2)));
// 0 when the launch just made was accepted (it is counted), else host_fail().
__attribute__((visibility("hidden"))) int host_launched(const char *kernel);
