// Launch interface of rotary_kernel (kernels/rotary.hip).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace tiny_llm {
namespace detail {

constexpr int kRotaryPairs = 128;

struct RotaryCall {
    const __half  *q = nullptr, *k = nullptr;
    __half        *q_out = nullptr, *k_out = nullptr;
    const __half  *q_weight = nullptr, *k_weight = nullptr;
    const int32_t *positions = nullptr;
    int64_t        q_stride = 0, k_stride = 0;
    int            T = 0, Hq = 0, Hkv = 0, rd = 0, interleaved = 0;
    float          eps = 0.0f;
    uint8_t        axis[kRotaryPairs] = {};
    double         turns[kRotaryPairs] = {};
};
// False: more tokens than one launch takes.
bool launch_rotary(const RotaryCall &c, int D, hipStream_t stream);

} // namespace detail
} // namespace tiny_llm
