// Launch interface of the prompt's account (kernels/attention_account.hip).
#pragma once

#include "../stream_plan.h"
#include "kv_kernels.h"

#include <cstddef>
#include <cstdint>

namespace tiny_llm {
namespace detail {

struct AccountCall {
    const __half *q = nullptr;    // [tokens][Hq][D]
    const float  *w_in = nullptr; // [row][Hkv][room], null: zeros
    float        *w_out = nullptr;
    int64_t       room = 0;
    float         scale = 1.0f;
    int           Hq = 0, Hkv = 0, D = 0;
};

// Workspace (floats) of launch_account.
size_t account_workspace_floats(const AccountPlan &plan, int Hkv);

// w_out[t] = (t < p0 ? w_in[t] : 0) + the weights of token t over the entry's
// last w queries and the kv head's query heads, for every t < p0 + n.
void launch_account(const AccountCall &c, const KvView &kv, const AccountPlan &plan, float *workspace,
                    hipStream_t stream);

} // namespace detail
} // namespace tiny_llm
