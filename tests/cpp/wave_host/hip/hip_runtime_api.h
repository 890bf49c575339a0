// The few names of the HIP runtime that a kernel source needs to compile as plain
// C++ (see hip_runtime.h beside it).
#pragma once

#include <cstddef>
#include <cstdint>

typedef int   hipError_t;
typedef void *hipStream_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t    hipGetLastError() { return hipSuccess; }
inline const char   *hipGetErrorString(hipError_t) { return ""; }
