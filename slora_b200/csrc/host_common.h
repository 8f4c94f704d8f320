// Host-side helpers shared by the library's source files: the error string of a failing call, the launch counters and
// pointer checks.  Defined in lora_kernels.cu.
#pragma once

#include <atomic>
#include <cstdint>

#include "slora_b200.h"

namespace slora {

// Kernels launched so far by this process, per family: 0 simple, 1 pipelined, 2 tensor core, 3 plan / tables / cache.
extern std::atomic<long long> g_launches[4];

// Keeps the message for slora_last_error() and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Turns a launch error into a status; counts `kernels` launches of `family` otherwise.
int check_launch(const char* what, int kernels, int family = 3);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace slora
