// What the files that hold C entry points share: the calling thread's error
// message (tilec_last_error) and the limits of an argument.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace tilec {

// Record a message for tilec_last_error() and return `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// Forget the last message (every entry point begins with it).
void clear_error();

constexpr int64_t kMaxDim = (int64_t(1) << 31) - 1024;  // kernels index rows/cols in int32

}  // namespace tilec
