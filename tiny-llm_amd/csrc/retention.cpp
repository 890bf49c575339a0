// Accounts of the cached tokens' attention weights and EvictBatch: what a bounded
// cache keeps (tiny_llm/kv_cache.h).
#include "kernels/account.h"
#include "kernels/evict.h"
#include "kernels/stream.h"
#include "runtime.h"
#include "tiny_llm/kv_cache.h"

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>
#include <vector>

namespace tiny_llm {

namespace {

bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Two arrays of `bytes` that overlap without being the same.
bool overlap(const void *x, const void *y, uintptr_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    return a != b && a < b + bytes && b < a + bytes;
}

uintptr_t account_bytes(const KVCacheConfig &cfg) {
    return static_cast<uintptr_t>(cfg.max_batch_size) * cfg.num_heads * cfg.max_seq_len * 4;
}

// "" when the accounts can be used, else the reason.
std::string check_accounts(const char *who, const KVCacheConfig &cfg, const float *in, const float *out) {
    if (!out) return std::string(who) + ": weights_out is null";
    if (!aligned(in, 4) || !aligned(out, 4)) return std::string(who) + ": weights must be 4-byte aligned";
    if (in && overlap(in, out, account_bytes(cfg)))
        return std::string(who) + ": weights_out overlaps weights_in without being it";
    return "";
}

std::string check_device(const char *who, int device) {
    const int now = detail::current_device();
    return now == device ? std::string()
                         : std::string(who) + ": the cache is on device " + std::to_string(device) +
                               ", the current one is " + std::to_string(now);
}

} // namespace

// ======================================================================
// DecodeBatch::decodeWeights
// ======================================================================

Result<void> DecodeBatch::decodeWeights(int layer_idx, const half *q, const half *new_k, const half *new_v, half *out,
                                        float scale, const float *weights_in, float *weights_out,
                                        hipStream_t stream) {
    const KVCacheConfig &cfg = mgr_.getConfig();
    if (mgr_.isQuantized()) return Result<void>::err("DecodeBatch: accounts are kept over fp16 caches only");
    if (q == nullptr || out == nullptr) return Result<void>::err("DecodeBatch: q/out is null");
    if ((new_k == nullptr) != (new_v == nullptr))
        return Result<void>::err(new_k ? "new_v is null" : "new_k is null");
    if (new_k && !appendable_) return Result<void>::err("DecodeBatch: append needs a batch made by prepare()");
    if (layer_idx < 0 || layer_idx >= cfg.num_layers)
        return Result<void>::err("DecodeBatch: Invalid layer_idx: " + std::to_string(layer_idx));
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(new_k, 16) || !aligned(new_v, 16))
        return Result<void>::err("DecodeBatch: q, out, new_k and new_v must be 16-byte aligned");
    if (std::string err = check_accounts("DecodeBatch", cfg, weights_in, weights_out); !err.empty())
        return Result<void>::err(err);
    if (n_ == 0) return Result<void>::ok();
    if (std::string err = check_device("DecodeBatch", mgr_.device()); !err.empty()) return Result<void>::err(err);
    detail::StreamPlan &plan = *account_plan_;
    if (plan.entries.empty()) {
        for (int i = 0; i < n_; ++i)
            plan.entries.push_back({slot_[static_cast<size_t>(i)], lens_[static_cast<size_t>(i)], i, 1, 0, 0});
        detail::plan_stream(plan, cfg.num_heads, cfg.head_dim, num_q_heads_ / cfg.num_heads, detail::device_cus());
    }
    const size_t floats = detail::stream_workspace_floats(plan, num_q_heads_, cfg.num_heads, cfg.head_dim, true);
    if (!account_work_->holds(floats) && detail::stream_capturing(stream))
        return Result<void>::err("DecodeBatch: the workspace cannot grow while the stream is captured: make one "
                                 "call of this size before");
    detail::StreamCall c;
    c.q = q;
    c.out = out;
    c.new_k = new_k;
    c.new_v = new_v;
    c.w_in = weights_in;
    c.w_out = weights_out;
    c.room = cfg.max_seq_len;
    c.fresh = appendable_ ? 1 : 0;
    c.scale = scale;
    c.Hq = num_q_heads_;
    c.Hkv = cfg.num_heads;
    c.D = cfg.head_dim;
    detail::launch_attn_stream(c, mgr_.layerView(layer_idx, nullptr), plan, account_work_->get(floats), stream);
    return Result<void>::ok();
}

// ======================================================================
// PrefillBatch::weights
// ======================================================================

Result<void> PrefillBatch::weights(int layer_idx, const half *q, float scale, int window, const float *weights_in,
                                   float *weights_out, hipStream_t stream) {
    const KVCacheConfig &cfg = mgr_.getConfig();
    if (mgr_.isQuantized()) return Result<void>::err("PrefillBatch: accounts are kept over fp16 caches only");
    if (layer_idx < 0 || layer_idx >= cfg.num_layers)
        return Result<void>::err("PrefillBatch: Invalid layer_idx: " + std::to_string(layer_idx));
    if (q == nullptr) return Result<void>::err("PrefillBatch: q is null");
    if (!aligned(q, 16)) return Result<void>::err("PrefillBatch: q must be 16-byte aligned");
    if (window < 0) return Result<void>::err("PrefillBatch: window must be >= 0 (got " + std::to_string(window) + ")");
    if (std::string err = check_accounts("PrefillBatch", cfg, weights_in, weights_out); !err.empty())
        return Result<void>::err(err);
    if (n_ == 0) return Result<void>::ok();
    if (std::string err = check_device("PrefillBatch", mgr_.device()); !err.empty()) return Result<void>::err(err);
    detail::AccountPlan &plan = *account_plan_;
    if (plan.window != window) {
        plan.clear();
        int32_t tok = 0;
        for (int i = 0; i < n_; ++i) {
            const size_t k = static_cast<size_t>(i);
            const int    w = window ? std::min(window, counts_[k]) : counts_[k];
            plan.entries.push_back({slots_[k], pos0_[k], counts_[k], w, tok, 1, 0, 0, 1, 0});
            tok += counts_[k];
        }
        if (!detail::plan_account(plan, num_q_heads_ / cfg.num_heads, cfg.num_heads, detail::device_cus())) {
            plan.clear();
            return Result<void>::err("PrefillBatch: too many query rows in one step");
        }
        plan.window = window;
    }
    const size_t floats = detail::account_workspace_floats(plan, cfg.num_heads);
    if (!account_work_->holds(floats) && detail::stream_capturing(stream))
        return Result<void>::err("PrefillBatch: the workspace cannot grow while the stream is captured: make one "
                                 "call of this size before");
    detail::AccountCall c;
    c.q = q;
    c.w_in = weights_in;
    c.w_out = weights_out;
    c.room = cfg.max_seq_len;
    c.scale = scale;
    c.Hq = num_q_heads_;
    c.Hkv = cfg.num_heads;
    c.D = cfg.head_dim;
    detail::launch_account(c, mgr_.layerView(layer_idx, nullptr), plan, account_work_->get(floats), stream);
    return Result<void>::ok();
}

// ======================================================================
// EvictBatch
// ======================================================================

EvictBatch::EvictBatch(KVCacheManager &mgr, int max_seqs)
    : mgr_(mgr), max_seqs_(max_seqs), work_(new detail::Workspace()) {}

EvictBatch::~EvictBatch() = default;

Result<std::unique_ptr<EvictBatch>> EvictBatch::create(KVCacheManager &mgr, int max_seqs) {
    using R = Result<std::unique_ptr<EvictBatch>>;
    const int d = mgr.getConfig().head_dim;
    if (mgr.isQuantized()) return R::err("EvictBatch: tokens are evicted from fp16 caches only");
    if (max_seqs <= 0) return R::err("EvictBatch: max_seqs must be positive");
    if (d != 32 && d != 64 && d != 128 && d != 256)
        return R::err("EvictBatch: unsupported head_dim " + std::to_string(d) + " (32, 64, 128 or 256)");
    return R::ok(std::unique_ptr<EvictBatch>(new EvictBatch(mgr, max_seqs)));
}

Result<void> EvictBatch::prepare(const int *seq_ids, const int *budgets, int n, int recent, hipStream_t stream) {
    for (size_t i = 0; i < ids_.size(); ++i)
        if (mgr_.sequence(ids_[i]) && mgr_.evictions_[static_cast<size_t>(entries_[i].row)].by == this)
            return Result<void>::err("EvictBatch: " + detail::eviction_begun(ids_[i]));
    // A failing prepare leaves an empty batch.
    ids_.clear();
    entries_.clear();
    ran_.assign(static_cast<size_t>(mgr_.getConfig().num_layers), 0);
    evicted_ = 0;
    if (n < 0 || n > max_seqs_)
        return Result<void>::err("EvictBatch: n=" + std::to_string(n) + " outside [0, " + std::to_string(max_seqs_) +
                                 "]");
    if (n > 0 && (seq_ids == nullptr || budgets == nullptr))
        return Result<void>::err("EvictBatch: seq_ids / budgets is null");
    if (recent < 0) return Result<void>::err("EvictBatch: recent must be >= 0 (got " + std::to_string(recent) + ")");
    if (std::string err = check_device("EvictBatch", mgr_.device()); !err.empty()) return Result<void>::err(err);
    const KVCacheConfig            &cfg = mgr_.getConfig();
    std::vector<char>               taken(static_cast<size_t>(cfg.max_batch_size), 0);
    std::vector<detail::EvictEntry> entries(static_cast<size_t>(n));
    int64_t                         evicted = 0, pairs = 0;
    for (int i = 0; i < n; ++i) {
        const SequenceCache *sc = mgr_.sequence(seq_ids[i]);
        if (!sc) return Result<void>::err("EvictBatch: sequence not found: " + std::to_string(seq_ids[i]));
        const int slot = mgr_.slotOf(seq_ids[i]);
        if (taken[static_cast<size_t>(slot)])
            return Result<void>::err("EvictBatch: duplicate sequence in batch: " + std::to_string(seq_ids[i]));
        taken[static_cast<size_t>(slot)] = 1;
        if (budgets[i] < 1 || budgets[i] < recent)
            return Result<void>::err("EvictBatch: budget " + std::to_string(budgets[i]) + " of sequence " +
                                     std::to_string(seq_ids[i]) + " must be positive and hold the " +
                                     std::to_string(recent) + " newest tokens");
        const KVCacheManager::Eviction &ev = mgr_.evictions_[static_cast<size_t>(slot)];
        if (ev.by) return Result<void>::err("EvictBatch: " + detail::eviction_begun(seq_ids[i]));
        if (ev.gone > INT32_MAX - cfg.max_seq_len)
            return Result<void>::err("EvictBatch: positions of sequence " + std::to_string(seq_ids[i]) +
                                     " exceed 31 bits");
        const int keep = std::min(sc->current_len, budgets[i]);
        entries[static_cast<size_t>(i)] = {slot, sc->current_len, keep, ev.base, ev.gone, 0};
        evicted += sc->current_len - keep;
        pairs += std::min(sc->current_len - keep, keep);
    }
    if (pairs > INT32_MAX) return Result<void>::err("EvictBatch: too many tokens in one step");
    const size_t words = detail::evict_workspace_words(entries, cfg.num_heads);
    if (!work_->holds(words) && detail::stream_capturing(stream))
        return Result<void>::err("EvictBatch: the workspace cannot grow while the stream is captured: prepare before "
                                 "the capture");
    lists_ = reinterpret_cast<int32_t *>(work_->get(std::max<size_t>(words, 1)));
    mgr_.syncTable(stream);
    entries_ = std::move(entries);
    ids_.assign(seq_ids, seq_ids + n);
    recent_ = recent;
    evicted_ = evicted;
    return Result<void>::ok();
}

// Sequences that were released since prepare() leave the step, and those that nothing is
// taken from when another eviction changed them.  The id of a released one, or -1.
int EvictBatch::leaveOut() {
    int    released = -1;
    size_t n = 0;
    for (size_t i = 0; i < ids_.size(); ++i) {
        const detail::EvictEntry e = entries_[i];
        if (!mgr_.sequence(ids_[i])) {
            released = ids_[i];
            evicted_ -= e.len - e.keep;
        } else if (e.keep < e.len || mgr_.evictions_[static_cast<size_t>(e.row)].gone == e.gone) {
            ids_[n] = ids_[i];
            entries_[n++] = e;
        }
    }
    if (n < ids_.size()) {
        ids_.resize(n);
        entries_.resize(n);
        detail::evict_workspace_words(entries_, mgr_.getConfig().num_heads); // (their lists, fewer than before)
    }
    return released;
}

std::string EvictBatch::changed() const {
    for (size_t i = 0; i < ids_.size(); ++i) {
        const detail::EvictEntry &e = entries_[i];
        if (e.keep == e.len) continue; // stays as it is, also where it has grown
        if (mgr_.sequence(ids_[i])->current_len != e.len || mgr_.evictions_[static_cast<size_t>(e.row)].gone != e.gone)
            return "EvictBatch: sequence " + std::to_string(ids_[i]) + " changed since prepare";
    }
    return "";
}

Result<void> EvictBatch::run(int layer_idx, const float *weights_in, float *weights_out, const int32_t *positions_in,
                             int32_t *positions_out, hipStream_t stream) {
    const KVCacheConfig &cfg = mgr_.getConfig();
    if (layer_idx < 0 || layer_idx >= cfg.num_layers)
        return Result<void>::err("EvictBatch: Invalid layer_idx: " + std::to_string(layer_idx));
    if (!weights_in || !weights_out || !positions_in || !positions_out)
        return Result<void>::err("EvictBatch: weights / positions is null");
    if (!aligned(weights_in, 4) || !aligned(weights_out, 4) || !aligned(positions_in, 4) || !aligned(positions_out, 4))
        return Result<void>::err("EvictBatch: weights and positions must be 4-byte aligned");
    const uintptr_t bytes = account_bytes(cfg);
    const void     *wi = weights_in, *wo = weights_out, *pi = positions_in, *po = positions_out;
    if (overlap(wi, wo, bytes) || overlap(pi, po, bytes) || wo == po || wi == po || wo == pi || overlap(wo, po, bytes) ||
        overlap(wi, po, bytes) || overlap(wo, pi, bytes))
        return Result<void>::err("EvictBatch: an output overlaps an array that it is not");
    if (ids_.empty()) return Result<void>::ok();
    if (const int id = leaveOut(); ids_.empty() && id >= 0)
        return Result<void>::err("EvictBatch: sequence not found: " + std::to_string(id));
    if (const std::string err = changed(); !err.empty()) return Result<void>::err(err);
    char &ran = ran_[static_cast<size_t>(layer_idx)];
    if (ran == 2)
        return Result<void>::err("EvictBatch: layer " + std::to_string(layer_idx) +
                                 " ran in place: commit before it runs again");
    if (std::string err = check_device("EvictBatch", mgr_.device()); !err.empty()) return Result<void>::err(err);
    for (size_t i = 0; i < ids_.size(); ++i) {
        const EvictBatch *by = mgr_.evictions_[static_cast<size_t>(entries_[i].row)].by;
        if (by && by != this) return Result<void>::err("EvictBatch: " + detail::eviction_begun(ids_[i]));
    }
    for (const auto &e : entries_)
        if (e.keep < e.len) mgr_.evictions_[static_cast<size_t>(e.row)].by = this;
    detail::EvictState st;
    st.w_in = weights_in;
    st.w_out = weights_out;
    st.pos_in = positions_in;
    st.pos_out = positions_out;
    st.room = cfg.max_seq_len;
    detail::launch_evict(mgr_.layerView(layer_idx, nullptr), entries_, st, recent_, cfg.num_heads, cfg.head_dim, lists_,
                         stream);
    ran = wi == wo || pi == po ? 2 : 1;
    return Result<void>::ok();
}

Result<void> EvictBatch::commit() {
    if (const int id = leaveOut(); evicted_ == 0 && id >= 0) // nothing is left to take
        return Result<void>::err("EvictBatch: sequence not found: " + std::to_string(id));
    if (const std::string err = changed(); !err.empty()) return Result<void>::err(err);
    if (evicted_ > 0) {
        for (size_t l = 0; l < ran_.size(); ++l)
            if (!ran_[l]) return Result<void>::err("EvictBatch: layer " + std::to_string(l) + " has not run");
    }
    for (const auto &e : entries_)
        if (e.keep < e.len) mgr_.truncate(e.row, e.keep);
    ids_.clear();
    entries_.clear();
    evicted_ = 0;
    return Result<void>::ok();
}

} // namespace tiny_llm
