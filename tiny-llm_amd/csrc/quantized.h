// Prepared steps of batches over a cache in 8 bits (KVCacheManager::createQuantized).
#pragma once

#include "kernels/kv_kernels.h"
#include "kernels/quant.h"
#include "runtime.h"
#include "tiny_llm/kv_cache.h"

#include <initializer_list>
#include <string>
#include <vector>

namespace tiny_llm {
namespace detail {

// "" when a call may run on the manager's device with these (possibly null) buffers.
std::string check_quant_call(const char *who, const KVCacheManager &mgr, std::initializer_list<const void *> buffers);

// Tokens that a sequence's cache holds, appended ones that it did not advance over included.
int held_tokens(const KVCacheManager &mgr, int seq_id, int slot);

// Ahead of an append to these layers: what a sequence advanced over in its open group though nobody brought it,
// behind the last append to the layer, becomes zeros there.
void zero_unbrought(const KVCacheManager &mgr, const std::vector<QuantAppend> &appends, int layer_begin, int num_layers,
                    hipStream_t stream);

struct QuantStep {
    std::vector<QuantEntry>  entries; // in the batch's order
    std::vector<QuantAppend> appends;
    QuantPlan                stream;  // entries of up to kQuantRows query rows,
    QuantPrefillPlan         prefill; // and those of more
    Workspace                work;

    void clear();
    int  items() const;
    void prepareDecode(const KVCacheManager &mgr, const std::vector<int32_t> &ids, const std::vector<int32_t> &slots,
                       const std::vector<int32_t> &lens, bool appendable, int num_q_heads);
    // False: too many query rows for one step.
    bool preparePrefill(const KVCacheManager &mgr, const std::vector<int32_t> &ids, const std::vector<int32_t> &slots,
                        const std::vector<int32_t> &counts, int num_q_heads);

    Result<void> appendOne(KVCacheManager &mgr, int layer_begin, int num_layers, const half *new_k, const half *new_v,
                           hipStream_t stream);
    Result<void> append(const char *who, KVCacheManager &mgr, int layer_idx, const half *new_k, const half *new_v,
                        hipStream_t stream);
    // new_k, new_v (null: nothing new) are appended in front: by a launch of their own (apart), or as
    // the entries' one token by the attention itself.
    Result<void> attention(const char *who, KVCacheManager &mgr, int layer_idx, const half *q, const half *new_k,
                           const half *new_v, half *out, float scale, int num_q_heads, bool apart, hipStream_t stream);
    Result<void> gather(KVCacheManager &mgr, int layer_idx, half *k_out, half *v_out, int s_max, hipStream_t stream);

  private:
    // The sequences as prepare found them: their lengths; where a step reads appended tokens that they
    // have not advanced over, what they held (else -1); and where the last append to a layer has to end (or
    // nothing be behind len) for the entry's open tile to have its tokens (-1: it is the one that
    // has those before len too).
    struct Seen {
        int32_t id, slot, len, held, end;
    };
    std::vector<Seen> seen_;
    std::string       check(const char *who, const KVCacheManager &mgr, std::initializer_list<const void *> buffers) const;
    std::string       checkRead(const char *who, const KVCacheManager &mgr, int layer_idx) const;
    void              noteAppends(KVCacheManager &mgr, int layer_begin, int num_layers) const;
};

} // namespace detail
} // namespace tiny_llm
