// Launch interface of attn_stream_kernel (kernels/attention_stream.hip).
#pragma once

#include "../stream_plan.h"
#include "kv_kernels.h"

#include <cstddef>
#include <cstdint>

namespace tiny_llm {
namespace detail {

struct StreamCall {
    const __half *q = nullptr; // [tokens][Hq][D]
    __half       *out = nullptr;
    // The last attended token of every entry comes from here ([entry][Hkv][D], entry
    // i of the plan; one query token per entry) and is appended; or null.
    const __half *new_k = nullptr, *new_v = nullptr;
    // Accounts [row][Hkv][room], or null: w_out = (t < S - fresh ? w_in : 0) + the
    // weights of token t, over the entry's queries and the kv head's query heads.
    const float *w_in = nullptr; // null: zeros
    float       *w_out = nullptr;
    int64_t      room = 0;
    int          fresh = 0;
    float        scale = 1.0f;
    int          Hq = 0, Hkv = 0, D = 0;
};

// Workspace (floats) of launch_attn_stream.
size_t stream_workspace_floats(const StreamPlan &plan, int Hq, int Hkv, int D, bool account);

// Attention of the plan's entries, at most kStreamRows rows each.  An entry
// with S = 0 gets zero rows.
void launch_attn_stream(const StreamCall &c, const KvView &kv, const StreamPlan &plan, float *workspace,
                        hipStream_t stream);

} // namespace detail
} // namespace tiny_llm
