// Norms of query and key heads and their rotation by position, in one pass.
#pragma once

#include "tiny_llm/result.h"

#include <hip/hip_fp16.h>
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <memory>
#include <vector>

namespace tiny_llm {
namespace kernels {

// What a model's rotation is: made once, used by every layer and step, from any thread,
// on any stream and device.
struct RotaryConfig {
    int    head_dim = 128;      // 32, 64, 128 or 256
    int    rotary_dim = 128;    // the first dims of a head that are rotated: a multiple of 16, at most head_dim
    double theta = 10000.0;     // inverse frequency of pair i: theta^(-2 i / rotary_dim)
    bool   interleaved = false; // pair i is dims (2 i, 2 i + 1); else (i, i + rotary_dim / 2)
    // Axis (0 .. 7) of each of the rotary_dim / 2 pairs, whose positions turn it; empty: all 0.
    std::vector<int> axis_of;
    // The pairs' inverse frequencies themselves, for scaled ones; empty: by theta.
    std::vector<double> inv_freq;
};

class Rotary {
  public:
    static Result<std::unique_ptr<Rotary>> create(const RotaryConfig &config);

    // For every token t and head h of q, and of k:
    //   y = x * rsqrt(mean(x^2) + eps) * weight      over head_dim; weight null: y = x
    //   (a, b) -> (a cos - b sin, a sin + b cos)     for pair i, angle positions[axis_of[i]][t] * inv_freq[i]
    // in fp32, rounded to fp16 once; angles are reduced in 64 bits, so positions of any size keep
    // theirs.  q: rows of num_q_heads * head_dim, q_stride elements from token to token (a
    // multiple of 8 up to 2^30), k likewise; q_out, k_out: [num_tokens][heads][head_dim]; positions: int32
    // [axes][num_tokens]; weights [head_dim].  k, k_out null: queries alone.  An output may be its own
    // input where that is dense, and must not overlap inputs, positions or weights otherwise.
    // Everything 16-byte aligned but positions.
    Result<void> apply(const half *q, int64_t q_stride, const half *k, int64_t k_stride, half *q_out, half *k_out,
                       const int32_t *positions, int num_tokens, int num_q_heads, int num_kv_heads, const half *q_weight,
                       const half *k_weight, float eps, hipStream_t stream) const;

    int axes() const noexcept { return axes_; }

  private:
    explicit Rotary(const RotaryConfig &config) : config_(config) {}
    RotaryConfig        config_;
    int                 axes_ = 1;
    std::vector<double> turns_; // of pair i per unit of position
};

} // namespace kernels
} // namespace tiny_llm
