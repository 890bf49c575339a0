// kernels::Rotary (tiny_llm/kernels/rotary.h).
#include "tiny_llm/kernels/rotary.h"

#include "kernels/rotary.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <iterator>
#include <string>

namespace tiny_llm {
namespace kernels {

Result<std::unique_ptr<Rotary>> Rotary::create(const RotaryConfig &config) {
    using R = Result<std::unique_ptr<Rotary>>;
    const int d = config.head_dim, rd = config.rotary_dim, n = rd / 2;
    if (d != 32 && d != 64 && d != 128 && d != 256)
        return R::err("Rotary: unsupported head_dim " + std::to_string(d) + " (32, 64, 128 or 256)");
    if (rd <= 0 || rd > d || rd % 16 != 0)
        return R::err("Rotary: rotary_dim must be a multiple of 16 in [16, head_dim] (got " + std::to_string(rd) + ")");
    if (!config.inv_freq.empty() && static_cast<int>(config.inv_freq.size()) != n)
        return R::err("Rotary: expected " + std::to_string(n) + " inverse frequencies, got " +
                      std::to_string(config.inv_freq.size()));
    if (config.inv_freq.empty() && !(config.theta > 0.0 && std::isfinite(config.theta)))
        return R::err("Rotary: theta must be positive and finite");
    if (!config.axis_of.empty() && static_cast<int>(config.axis_of.size()) != n)
        return R::err("Rotary: expected " + std::to_string(n) + " axes, got " + std::to_string(config.axis_of.size()));
    std::unique_ptr<Rotary> r(new Rotary(config));
    for (const int a : config.axis_of) {
        if (a < 0 || a > 7) return R::err("Rotary: axis " + std::to_string(a) + " outside [0, 7]");
        r->axes_ = std::max(r->axes_, a + 1);
    }
    for (int i = 0; i < n; ++i) {
        const double f = config.inv_freq.empty() ? std::pow(config.theta, -static_cast<double>(i) / n)
                                                 : config.inv_freq[static_cast<size_t>(i)];
        if (!std::isfinite(f)) return R::err("Rotary: inverse frequency " + std::to_string(i) + " is not finite");
        r->turns_.push_back(f / (2.0 * M_PI));
    }
    return R::ok(std::move(r));
}

namespace {

struct Range {
    uintptr_t lo, hi;
    bool      meets(const Range &o) const { return lo < o.hi && o.lo < hi; }
};
constexpr int64_t kMostStride = int64_t(1) << 30; // (2^31 tokens of it are still an offset in 64 bits)
Range             range(const half *p, int64_t tokens, int64_t stride, int64_t row) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return {a, a + static_cast<uintptr_t>(((tokens - 1) * stride + row) * static_cast<int64_t>(sizeof(half)))};
}

} // namespace

Result<void> Rotary::apply(const half *q, int64_t q_stride, const half *k, int64_t k_stride, half *q_out, half *k_out,
                           const int32_t *positions, int num_tokens, int num_q_heads, int num_kv_heads,
                           const half *q_weight, const half *k_weight, float eps, hipStream_t stream) const {
    auto err = [](const std::string &m) { return Result<void>::err("Rotary: " + m); };
    if (num_tokens < 0) return err("num_tokens must be >= 0 (got " + std::to_string(num_tokens) + ")");
    if (!q || !q_out) return err("q/q_out is null");
    if ((k == nullptr) != (k_out == nullptr)) return err("k and k_out must be both set or both null");
    if (!positions) return err("positions is null");
    if (num_q_heads <= 0 || (k && num_kv_heads <= 0)) return err("heads must be positive");
    if (num_q_heads > 65536 || (k && num_kv_heads > 65536)) return err("more than 65536 heads");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return err("eps must be finite and >= 0");
    const int64_t q_row = static_cast<int64_t>(num_q_heads) * config_.head_dim;
    const int64_t k_row = k ? static_cast<int64_t>(num_kv_heads) * config_.head_dim : 0;
    if (q_stride < q_row || q_stride % 8 != 0 || (k && (k_stride < k_row || k_stride % 8 != 0)))
        return err("strides must be multiples of 8, at least heads * head_dim");
    if (q_stride > kMostStride || (k && k_stride > kMostStride)) return err("strides must be at most 2^30");
    for (const void *p : {static_cast<const void *>(q), static_cast<const void *>(k), static_cast<const void *>(q_out),
                          static_cast<const void *>(k_out), static_cast<const void *>(q_weight),
                          static_cast<const void *>(k_weight)})
        if (reinterpret_cast<uintptr_t>(p) & 15u) return err("q, k, their outputs and weights must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(positions) & 3u) return err("positions must be 4-byte aligned");
    if (num_tokens == 0) return Result<void>::ok();
    const Range qi = range(q, num_tokens, q_stride, q_row), qo = range(q_out, num_tokens, q_row, q_row);
    const uintptr_t pos = reinterpret_cast<uintptr_t>(positions);
    const Range     given[] = {{pos, pos + static_cast<uintptr_t>(num_tokens) * axes_ * sizeof(int32_t)},
                               range(q_weight, 1, 0, q_weight ? config_.head_dim : 0),
                               range(k_weight, 1, 0, k_weight ? config_.head_dim : 0)};
    auto            meets_given = [&](const Range &out) {
        return std::any_of(std::begin(given), std::end(given), [&](const Range &x) { return out.meets(x); });
    };
    const bool  q_in_place = q_out == q && (q_stride == q_row || num_tokens == 1);
    if (qo.meets(qi) && !q_in_place) return err("q_out overlaps q");
    if (meets_given(qo)) return err("q_out overlaps positions or weights");
    if (k) {
        const Range ki = range(k, num_tokens, k_stride, k_row), ko = range(k_out, num_tokens, k_row, k_row);
        const bool  k_in_place = k_out == k && (k_stride == k_row || num_tokens == 1);
        if (ko.meets(ki) && !k_in_place) return err("k_out overlaps k");
        if (meets_given(ko)) return err("k_out overlaps positions or weights");
        if (qo.meets(ki) || ko.meets(qi) || qo.meets(ko)) return err("q, k and their outputs overlap");
    }
    detail::RotaryCall c;
    c.q = q;
    c.k = k;
    c.q_out = q_out;
    c.k_out = k_out;
    c.q_weight = q_weight;
    c.k_weight = k ? k_weight : nullptr;
    c.positions = positions;
    c.q_stride = q_stride;
    c.k_stride = k_stride;
    c.T = num_tokens;
    c.Hq = num_q_heads;
    c.Hkv = k ? num_kv_heads : 0;
    c.rd = config_.rotary_dim;
    c.interleaved = config_.interleaved ? 1 : 0;
    c.eps = eps;
    for (size_t i = 0; i < turns_.size(); ++i) {
        c.turns[i] = turns_[i];
        c.axis[i] = config_.axis_of.empty() ? 0 : static_cast<uint8_t>(config_.axis_of[i]);
    }
    if (!detail::launch_rotary(c, config_.head_dim, stream)) return err("too many tokens and heads for one call");
    return Result<void>::ok();
}

} // namespace kernels
} // namespace tiny_llm
