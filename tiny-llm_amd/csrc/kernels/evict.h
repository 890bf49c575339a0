// Launch interface of the eviction kernels (kernels/evict.hip).
#pragma once

#include "kv_kernels.h"

#include <cstddef>
#include <cstdint>
#include <vector>

namespace tiny_llm {
namespace detail {

// One sequence of an eviction: of the `len` tokens of cache row `row`, `keep`
// stay.  Token t < base has its position in the caller's positions, token t >=
// base the position t + gone.  list: the entry's first pair in the workspace (in
// pairs per kv head), room for min(len - keep, keep) of them.
struct EvictEntry {
    int32_t row, len, keep, base, gone, list;
};

// Entries per launch: they travel in the kernel arguments, so that a launch
// depends on no memory that a later step rewrites.
constexpr int kEvictBatch = 144;

// The accounts and positions of one layer, [row][Hkv][room].
struct EvictState {
    const float   *w_in = nullptr;
    float         *w_out = nullptr;
    const int32_t *pos_in = nullptr;
    int32_t       *pos_out = nullptr;
    int64_t        room = 0;
};

// Workspace (int32 words) of launch_evict: the entries' pair lists, for every kv
// head, and their lengths.  Sets the entries' `list`.
size_t evict_workspace_words(std::vector<EvictEntry> &entries, int Hkv);

// Selects and moves for one layer, on `stream`: two launches for every
// kEvictBatch entries.
void launch_evict(const KvView &kv, const std::vector<EvictEntry> &entries, const EvictState &st, int recent, int Hkv,
                  int D, int32_t *workspace, hipStream_t stream);

} // namespace detail
} // namespace tiny_llm
