// Launch interface of attn_cross_kernel (kernels/attention_cross.hip).
#pragma once

#include "../stream_plan.h"
#include "kv_kernels.h"

#include <cstddef>
#include <cstdint>
#include <utility>
#include <vector>

namespace tiny_llm {
namespace detail {

struct CrossCall {
    const __half *q = nullptr; // [tokens][Hq][D]
    __half       *out = nullptr;
    float         scale = 1.0f;
    int           Hq = 0, Hkv = 0, D = 0;
};

// Workspace (floats) of launch_attn_cross.
size_t cross_workspace_floats(const CrossPlan &plan, int Hkv, int D);

void launch_attn_cross(const CrossCall &c, const KvView &kv, const CrossPlan &plan, float *workspace,
                       hipStream_t stream);

// Rows of zeros for queries over no states: tokens first .. first + second - 1 of `out`
// ([token][row] halves, row a multiple of 8) for every range.
void launch_cross_zeros(__half *out, int row, const std::vector<std::pair<int32_t, int32_t>> &ranges, hipStream_t stream);

} // namespace detail
} // namespace tiny_llm
