// CrossBatch: attention to cached states of another length (tiny_llm/kv_cache.h).
#include "kernels/cross.h"
#include "kernels/stream.h"
#include "runtime.h"
#include "tiny_llm/kv_cache.h"

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>
#include <vector>

namespace tiny_llm {

CrossBatch::CrossBatch(KVCacheManager &mgr, int max_entries, int num_q_heads)
    : mgr_(mgr), max_entries_(max_entries), num_q_heads_(num_q_heads), stream_plan_(new detail::StreamPlan()),
      cross_plan_(new detail::CrossPlan()), work_(new detail::Workspace()) {}

CrossBatch::~CrossBatch() = default;

Result<std::unique_ptr<CrossBatch>> CrossBatch::create(KVCacheManager &mgr, int max_entries, int num_q_heads) {
    using R = Result<std::unique_ptr<CrossBatch>>;
    const KVCacheConfig &cfg = mgr.getConfig();
    if (mgr.isQuantized()) return R::err("CrossBatch: attends to fp16 caches only");
    if (max_entries <= 0) return R::err("CrossBatch: max_entries must be positive");
    if (num_q_heads <= 0 || num_q_heads % cfg.num_heads != 0)
        return R::err("CrossBatch: num_q_heads (" + std::to_string(num_q_heads) +
                      ") must be a positive multiple of num_heads (" + std::to_string(cfg.num_heads) + ")");
    if (!detail::attn_shape_supported(cfg.head_dim, num_q_heads / cfg.num_heads))
        return R::err("CrossBatch: unsupported head_dim/group (head_dim in {32,64,128,256}, "
                      "num_q_heads/num_heads in {1,2,4,8})");
    return R::ok(std::unique_ptr<CrossBatch>(new CrossBatch(mgr, max_entries, num_q_heads)));
}

Result<void> CrossBatch::prepare(const int *seq_ids, const int *num_queries, const int *attended, int n,
                                 hipStream_t stream) {
    // A failing prepare leaves an empty batch.
    n_ = 0;
    tokens_ = 0;
    ids_.clear();
    lens_.clear();
    empty_.clear();
    stream_plan_->clear();
    cross_plan_->clear();
    if (n < 0 || n > max_entries_)
        return Result<void>::err("CrossBatch: n=" + std::to_string(n) + " outside [0, " +
                                 std::to_string(max_entries_) + "]");
    if (n > 0 && (seq_ids == nullptr || num_queries == nullptr))
        return Result<void>::err("CrossBatch: seq_ids / num_queries is null");
    if (const int now = detail::current_device(); now != mgr_.device())
        return Result<void>::err("CrossBatch: the cache is on device " + std::to_string(mgr_.device()) +
                                 ", the current one is " + std::to_string(now));
    const KVCacheConfig &cfg = mgr_.getConfig();
    const int            group = num_q_heads_ / cfg.num_heads;
    std::vector<int32_t> lens(static_cast<size_t>(n));
    int64_t              total = 0;
    for (int i = 0; i < n; ++i) {
        const SequenceCache *sc = mgr_.sequence(seq_ids[i]);
        if (!sc) return Result<void>::err("CrossBatch: sequence not found: " + std::to_string(seq_ids[i]));
        if (mgr_.evictionBegun(mgr_.slotOf(seq_ids[i])))
            return Result<void>::err("CrossBatch: " + detail::eviction_begun(seq_ids[i]));
        if (num_queries[i] <= 0)
            return Result<void>::err("CrossBatch: num_queries must be positive: " + std::to_string(num_queries[i]));
        const int a = attended ? attended[i] : sc->current_len;
        if (a < 0 || a > sc->current_len)
            return Result<void>::err("CrossBatch: attended length " + std::to_string(a) + " of sequence " +
                                     std::to_string(seq_ids[i]) + " outside [0, " + std::to_string(sc->current_len) +
                                     "]");
        lens[static_cast<size_t>(i)] = a;
        total += num_queries[i];
    }
    if (total * group > INT32_MAX / 2) return Result<void>::err("CrossBatch: too many query rows in one step");
    mgr_.syncTable(stream);
    // Neighbours over the same states are one entry of the plans: their rows share
    // every key.  Up to 16 rows take attn_stream_kernel, which reads the states once at
    // the memory's rate; more take attn_cross_kernel; queries over nothing get zeros.
    int64_t tok = 0;
    for (int i = 0; i < n;) {
        const int slot = mgr_.slotOf(seq_ids[i]);
        const int len = lens[static_cast<size_t>(i)];
        const int first = static_cast<int>(tok);
        int       nq = 0;
        for (const int id = seq_ids[i]; i < n && seq_ids[i] == id && lens[static_cast<size_t>(i)] == len; ++i)
            nq += num_queries[i];
        tok += nq;
        if (len > 0) {
            if (nq * static_cast<int64_t>(group) > detail::kStreamRows) cross_plan_->entries.push_back({slot, len, first, nq, 1, 0});
            else stream_plan_->entries.push_back({slot, len, first, nq, 0, 0});
        } else if (!empty_.empty() && empty_.back().first + empty_.back().second == first) {
            empty_.back().second += nq;
        } else {
            empty_.push_back({first, nq});
        }
    }
    detail::plan_stream(*stream_plan_, cfg.num_heads, cfg.head_dim, 0, detail::device_cus());
    if (!detail::plan_cross(*cross_plan_, cfg.head_dim, group, cfg.num_heads, detail::device_cus())) {
        empty_.clear();
        stream_plan_->clear();
        cross_plan_->clear();
        return Result<void>::err("CrossBatch: too many query rows in one step");
    }
    ids_.assign(seq_ids, seq_ids + n);
    lens_ = std::move(lens);
    n_ = n;
    tokens_ = static_cast<int>(total);
    return Result<void>::ok();
}

Result<void> CrossBatch::attention(int layer_idx, const half *q, half *out, float scale, hipStream_t stream) {
    const KVCacheConfig &cfg = mgr_.getConfig();
    if (layer_idx < 0 || layer_idx >= cfg.num_layers)
        return Result<void>::err("CrossBatch: Invalid layer_idx: " + std::to_string(layer_idx));
    if (q == nullptr || out == nullptr) return Result<void>::err("CrossBatch: q/out is null");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15u)
        return Result<void>::err("CrossBatch: q and out must be 16-byte aligned");
    if (n_ == 0) return Result<void>::ok();
    if (const int now = detail::current_device(); now != mgr_.device())
        return Result<void>::err("CrossBatch: the cache is on device " + std::to_string(mgr_.device()) +
                                 ", the current one is " + std::to_string(now));
    for (size_t i = 0; i < ids_.size(); ++i) {
        const SequenceCache *sc = mgr_.sequence(ids_[i]);
        if (!sc) return Result<void>::err("CrossBatch: sequence not found: " + std::to_string(ids_[i]));
        if (sc->current_len < lens_[i])
            return Result<void>::err("CrossBatch: sequence " + std::to_string(ids_[i]) + " is shorter than prepare found it");
    }
    const size_t floats = std::max(
        detail::stream_workspace_floats(*stream_plan_, num_q_heads_, cfg.num_heads, cfg.head_dim, false),
        detail::cross_workspace_floats(*cross_plan_, cfg.num_heads, cfg.head_dim));
    if (!work_->holds(floats) && detail::stream_capturing(stream))
        return Result<void>::err("CrossBatch: the workspace cannot grow while the stream is captured: make one call "
                                 "of this size before");
    float               *ws = work_->get(floats);
    const detail::KvView view = mgr_.layerView(layer_idx, nullptr);
    detail::launch_cross_zeros(out, num_q_heads_ * cfg.head_dim, empty_, stream);
    if (!stream_plan_->entries.empty()) {
        detail::StreamCall c;
        c.q = q;
        c.out = out;
        c.scale = scale;
        c.Hq = num_q_heads_;
        c.Hkv = cfg.num_heads;
        c.D = cfg.head_dim;
        detail::launch_attn_stream(c, view, *stream_plan_, ws, stream);
    }
    if (!cross_plan_->entries.empty()) {
        detail::CrossCall c;
        c.q = q;
        c.out = out;
        c.scale = scale;
        c.Hq = num_q_heads_;
        c.Hkv = cfg.num_heads;
        c.D = cfg.head_dim;
        detail::launch_attn_cross(c, view, *cross_plan_, ws, stream);
    }
    return Result<void>::ok();
}

} // namespace tiny_llm
