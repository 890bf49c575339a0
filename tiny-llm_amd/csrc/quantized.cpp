// The cache in 8 bits: KVCacheManager::createQuantized and the steps of batches over it.
#include "quantized.h"

#include "block_allocator.h"
#include "tl_log.h"

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>
#include <vector>

namespace tiny_llm {

using detail::kGroup;

Result<std::unique_ptr<KVCacheManager>> KVCacheManager::createQuantized(const KVCacheConfig &config, int block_tokens,
                                                                        int num_blocks) {
    using R = Result<std::unique_ptr<KVCacheManager>>;
    if (block_tokens < kGroup || (block_tokens & (block_tokens - 1)) != 0)
        return R::err("KVCacheManager: block_tokens of an 8-bit cache must be a power of two >= 32 (got " +
                      std::to_string(block_tokens) + ")");
    if (num_blocks <= 0 || num_blocks == INT32_MAX)
        return R::err("KVCacheManager: num_blocks must be in [1, 2^31 - 2] (got " + std::to_string(num_blocks) + ")");
    const int d = config.head_dim;
    if (d > 0 && d != 32 && d != 64 && d != 128 && d != 256)
        return R::err("KVCacheManager: unsupported head_dim " + std::to_string(d) + " of an 8-bit cache (32, 64, 128 or 256)");
    return build(config, block_tokens, num_blocks, true);
}

detail::QuantView KVCacheManager::quantView(int layer_idx) const {
    const int64_t     heads = config_.num_heads, tile = 2 * kGroup * static_cast<int64_t>(config_.head_dim);
    const int64_t     layer = (static_cast<int64_t>(blocks_->numBlocks()) + 1) * heads * (block_tokens_ / kGroup); // groups
    detail::QuantView v;
    v.tiles = reinterpret_cast<uint8_t *>(memory_pool_) + layer_idx * layer * tile;
    v.scales = scales_ + layer_idx * layer;
    v.open = open_tiles_ + layer_idx * (static_cast<int64_t>(config_.max_batch_size) * 2 * heads * tile);
    v.table = block_map_dev_;
    v.bt_stride = blocks_->blocksPerRow();
    while ((kGroup << v.lg) < block_tokens_) ++v.lg;
    return v;
}

const detail::OpenGroup &KVCacheManager::openGroup(int slot) const noexcept { return open_[static_cast<size_t>(slot)]; }

int KVCacheManager::appendedEnd(int slot, int layer) const noexcept {
    return appended_end_[static_cast<size_t>(slot) * static_cast<size_t>(config_.num_layers) + static_cast<size_t>(layer)];
}

void KVCacheManager::noteAppend(int slot, int layer_begin, int num_layers, int n) noexcept {
    const int len = slots_[static_cast<size_t>(slot)].current_len;
    open_[static_cast<size_t>(slot)].append(len, n);
    std::fill_n(appended_end_.begin() + static_cast<std::ptrdiff_t>(slot) * config_.num_layers + layer_begin, num_layers, len + n);
}

std::string KVCacheManager::cannotAdvance(int slot, int seq_id, int to) const {
    detail::OpenGroup open = open_[static_cast<size_t>(slot)];
    const int         len = slots_[static_cast<size_t>(slot)].current_len, end = open.end;
    const int        *ends = &appended_end_[static_cast<size_t>(slot) * static_cast<size_t>(config_.num_layers)];
    const bool        alike = open.alike(ends, config_.num_layers, len, to);
    if (alike && open.advance(len, to)) return std::string();
    const std::string length = "advanceSeqLen: length " + std::to_string(to) + " of sequence " + std::to_string(seq_id);
    const std::string beyond = length + " is beyond the tokens up to " + std::to_string(end);
    if (!alike)
        return length + ": its layers differ in what was appended last, and one of them would lose tokens of its open group";
    if (open.replaced(to)) return beyond + " of the last append, which replaced one that brought more: append those again";
    if (open.leaves_rows(to))
        return beyond + " that were appended, and in an 8-bit cache the last of them wait in their group of " +
               std::to_string(kGroup) + " for those that complete it";
    return length + " lies inside the tokens up to " + std::to_string(end) +
           " that were appended at once: an 8-bit cache can be cut there at a multiple of " + std::to_string(kGroup) +
           ", in the group in which they begin or in the one in which they end";
}

namespace detail {

std::string check_quant_call(const char *who, const KVCacheManager &mgr, std::initializer_list<const void *> buffers) {
    if (const int now = current_device(); now != mgr.device())
        return std::string(who) + ": the cache is on device " + std::to_string(mgr.device()) + ", the current one is " +
               std::to_string(now);
    for (const void *p : buffers)
        if (reinterpret_cast<uintptr_t>(p) & 15u) return std::string(who) + ": buffers must be 16-byte aligned";
    return std::string();
}

int held_tokens(const KVCacheManager &mgr, int seq_id, int slot) {
    return mgr.openGroup(slot).held(mgr.sequence(seq_id)->current_len).first;
}

void zero_unbrought(const KVCacheManager &mgr, const std::vector<QuantAppend> &appends, int layer_begin, int num_layers,
                    hipStream_t stream) {
    const KVCacheConfig &cfg = mgr.getConfig();
    for (int layer = layer_begin; layer < layer_begin + num_layers; ++layer) {
        std::vector<QuantRows> rows;
        for (const QuantAppend &a : appends) {
            const int group = a.p0 / kGroup * kGroup, lo = std::max(mgr.appendedEnd(a.row, layer), group);
            if (lo < a.p0) rows.push_back({a.row, a.first_last & 1, lo - group, a.p0 - group});
        }
        if (!rows.empty()) launch_quant_zero_rows(mgr.quantView(layer), rows, cfg.num_heads, cfg.head_dim, stream);
    }
}

void QuantStep::clear() {
    entries.clear();
    appends.clear();
    stream.clear();
    prefill.clear();
    seen_.clear();
}

int QuantStep::items() const {
    int n = 0;
    for (const auto &l : stream.launches) n += l.items;
    for (const auto &l : prefill.launches) n += l.items;
    return n;
}

std::string QuantStep::check(const char *who, const KVCacheManager &mgr, std::initializer_list<const void *> buffers) const {
    for (const Seen &s : seen_) {
        const SequenceCache *sc = mgr.sequence(s.id);
        if (!sc || mgr.slotOf(s.id) != s.slot || sc->current_len != s.len || (s.held >= 0 && held_tokens(mgr, s.id, s.slot) != s.held))
            return std::string(who) + ": sequence " + std::to_string(s.id) + " has changed since prepare";
    }
    return check_quant_call(who, mgr, buffers);
}

std::string QuantStep::checkRead(const char *who, const KVCacheManager &mgr, int layer_idx) const {
    for (const Seen &s : seen_)
        if (const int end = mgr.appendedEnd(s.slot, layer_idx); s.end >= 0 && end > s.len && end != s.end)
            return std::string(who) + ": another append to sequence " + std::to_string(s.id) + ", up to " + std::to_string(end) +
                   ", has replaced tokens up to " + std::to_string(s.end) + " of layer " + std::to_string(layer_idx);
    return std::string();
}

void QuantStep::noteAppends(KVCacheManager &mgr, int layer_begin, int num_layers) const {
    for (const QuantAppend &a : appends) mgr.noteAppend(a.row, layer_begin, num_layers, a.n);
}

void QuantStep::prepareDecode(const KVCacheManager &mgr, const std::vector<int32_t> &ids, const std::vector<int32_t> &slots,
                              const std::vector<int32_t> &lens, bool appendable, int num_q_heads) {
    const KVCacheConfig &cfg = mgr.getConfig();
    for (size_t i = 0; i < ids.size(); ++i) {
        const int S = lens[i], tok = static_cast<int>(i), len = mgr.sequence(ids[i])->current_len;
        if (appendable) {
            const int tile = mgr.openGroup(slots[i]).cur;
            seen_.push_back({ids[i], slots[i], len, -1, -1});
            appends.push_back({slots[i], S - 1, 1, tok, tile | tile << 1, 0});
            entries.push_back({slots[i], S, tok, 1, tile, 0});
        } else {
            // A last group that is complete in the cache is read there; what a sequence has
            // advanced over stands as it did then, whatever was appended behind it.
            auto [held, tile] = mgr.openGroup(slots[i]).held(len);
            seen_.push_back({ids[i], slots[i], len, S > len ? held : -1, S > len ? held : -1});
            if (S <= len) {
                held = len;
                tile = mgr.openGroup(slots[i]).cur;
            }
            entries.push_back({slots[i], S, tok, 1, S > held / kGroup * kGroup ? tile : -1, 0});
        }
    }
    stream.entries = entries;
    plan_quant(stream, num_q_heads / cfg.num_heads, cfg.num_heads, cfg.head_dim, device_cus());
}

bool QuantStep::preparePrefill(const KVCacheManager &mgr, const std::vector<int32_t> &ids, const std::vector<int32_t> &slots,
                               const std::vector<int32_t> &counts, int num_q_heads) {
    const KVCacheConfig &cfg = mgr.getConfig();
    const int            group = num_q_heads / cfg.num_heads;
    int                  tok = 0;
    for (size_t i = 0; i < ids.size(); ++i) {
        const int n = counts[i], p0 = mgr.sequence(ids[i])->current_len, S = p0 + n;
        const auto [first, last] = mgr.openGroup(slots[i]).tiles(p0, n);
        const int open = S % kGroup != 0 ? last : -1;
        seen_.push_back({ids[i], slots[i], p0, -1, open >= 0 && last != first ? S : -1});
        appends.push_back({slots[i], p0, n, tok, first | last << 1, 0});
        entries.push_back({slots[i], S, tok, n, open, 0});
        if (static_cast<int64_t>(n) * group <= kQuantRows) stream.entries.push_back(entries.back());
        else if (static_cast<int64_t>(n) * group > INT32_MAX / 2) return false;
        else prefill.entries.push_back({slots[i], S, tok, n, open, 1, 0});
        tok += n;
    }
    plan_quant(stream, group, cfg.num_heads, cfg.head_dim, device_cus());
    return plan_quant_prefill(prefill, cfg.head_dim, group, cfg.num_heads, device_cus());
}

Result<void> QuantStep::appendOne(KVCacheManager &mgr, int layer_begin, int num_layers, const half *new_k,
                                  const half *new_v, hipStream_t stream) {
    if (std::string err = check("DecodeBatch", mgr, {new_k, new_v}); !err.empty()) return Result<void>::err(err);
    const KVCacheConfig &cfg = mgr.getConfig();
    const QuantView      v = mgr.quantView(layer_begin);
    QuantLayerSteps      steps;
    if (num_layers > 1) {
        const QuantView w = mgr.quantView(layer_begin + 1);
        steps = {w.tiles - v.tiles, w.scales - v.scales, w.open - v.open};
    }
    zero_unbrought(mgr, appends, layer_begin, num_layers, stream);
    launch_quant_append_one(v, steps, appends, num_layers, cfg.num_heads, cfg.head_dim, new_k, new_v, stream);
    noteAppends(mgr, layer_begin, num_layers);
    return Result<void>::ok();
}

Result<void> QuantStep::append(const char *who, KVCacheManager &mgr, int layer_idx, const half *new_k, const half *new_v,
                               hipStream_t stream) {
    if (std::string err = check(who, mgr, {new_k, new_v}); !err.empty()) return Result<void>::err(err);
    const KVCacheConfig &cfg = mgr.getConfig();
    zero_unbrought(mgr, appends, layer_idx, 1, stream);
    launch_quant_append(mgr.quantView(layer_idx), appends, cfg.num_heads, cfg.head_dim, new_k, new_v, stream);
    noteAppends(mgr, layer_idx, 1);
    return Result<void>::ok();
}

Result<void> QuantStep::attention(const char *who, KVCacheManager &mgr, int layer_idx, const half *q, const half *new_k,
                                  const half *new_v, half *out, float scale, int num_q_heads, bool apart, hipStream_t stream) {
    if (std::string err = check(who, mgr, {q, new_k, new_v, out}); !err.empty()) return Result<void>::err(err);
    if (std::string err = new_k ? std::string() : checkRead(who, mgr, layer_idx); !err.empty()) return Result<void>::err(err);
    const KVCacheConfig &cfg = mgr.getConfig();
    const size_t floats = std::max(quant_workspace_floats(this->stream, cfg.num_heads, cfg.head_dim),
                                   quant_prefill_workspace_floats(prefill, cfg.num_heads, cfg.head_dim));
    if (!work.holds(floats) && stream_capturing(stream))
        return Result<void>::err(std::string(who) + ": the workspace cannot grow while the stream is captured: make one "
                                                    "call of this size before");
    float            *ws = work.get(floats);
    const QuantView   v = mgr.quantView(layer_idx);
    // (behind the checks: a refused call has appended nothing)
    if (new_k) zero_unbrought(mgr, appends, layer_idx, 1, stream);
    if (new_k && apart) launch_quant_append(v, appends, cfg.num_heads, cfg.head_dim, new_k, new_v, stream);
    QuantCall c;
    c.q = q;
    c.out = out;
    c.new_k = apart ? nullptr : new_k;
    c.new_v = apart ? nullptr : new_v;
    c.scale = scale;
    c.Hq = num_q_heads;
    c.Hkv = cfg.num_heads;
    c.D = cfg.head_dim;
    if (!this->stream.entries.empty()) launch_attn_quant(c, v, this->stream, ws, stream);
    if (!prefill.entries.empty()) launch_quant_prefill(c, v, prefill, ws, stream);
    if (new_k) noteAppends(mgr, layer_idx, 1);
    return Result<void>::ok();
}

Result<void> QuantStep::gather(KVCacheManager &mgr, int layer_idx, half *k_out, half *v_out, int s_max,
                               hipStream_t stream) {
    if (std::string err = check("DecodeBatch", mgr, {k_out, v_out}); !err.empty()) return Result<void>::err(err);
    if (std::string err = checkRead("DecodeBatch", mgr, layer_idx); !err.empty()) return Result<void>::err(err);
    const KVCacheConfig &cfg = mgr.getConfig();
    launch_quant_gather(mgr.quantView(layer_idx), entries, cfg.num_heads, cfg.head_dim, s_max, k_out, v_out, stream);
    return Result<void>::ok();
}

} // namespace detail
} // namespace tiny_llm
