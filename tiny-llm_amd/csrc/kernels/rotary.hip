// RMS norm of every query and key head and its rotation by position, in one pass, for gfx950.
//
//   y = x rsqrt(mean x^2 + eps) w;   (a, b) -> (a cos - b sin, a sin + b cos) per pair of dims
// Bound by HBM (a value is read and written once, 4 bytes) and, for a decode step, by the launch.
//
// D / 16 threads have a head's row, 8 + 8 values each: those of 8 pairs (dims that are not
// rotated: 16 neighbours), so that a rotation needs no other thread.  A workgroup computes the angles
// of its tokens once, into LDS, and a thread keeps its 8 over several heads of its token: an angle
// costs about as much as 8 values' loads and stores (the turns, position * inv_freq / 2 pi, are
// reduced to half a turn in 64 bits, where a far position times a high frequency still has its
// fraction; sine and cosine are then fp32).  Each thread its own angles took 45 us where this takes 30
// (8000 tokens, 40 heads of 128, 164 MB: 5.5 TB/s); a step of 64 tokens 4 us, the launch and one
// dependent read of positions.
#include "rotary.h"

#include "kv_kernels.h"
#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

namespace tiny_llm {
namespace detail {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kHeads = 2; // heads of a thread on their way at once

// hs: threads' rows per token (a power of two); blockIdx.y: heads y * per * hs ..
template <int D, bool NORM>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryCall a, int lg_hs, int per) {
    constexpr int LPR = D / 16;
    const int     p = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const int     hs = 1 << lg_hs, h_first = (int)blockIdx.y * per * hs + (slot & (hs - 1));
    const int     H = a.Hq + a.Hkv, tokens = kThreads / LPR >> lg_hs, pairs = a.rd / 2;
    const int64_t t0 = (int64_t)blockIdx.x * tokens, t = t0 + (slot >> lg_hs);
    __shared__ float2 s_angle[kThreads / LPR * D / 2]; // (cosine, sine) of the block's tokens
    const bool turned = 16 * p < a.rd;
    const int  d0 = turned && !a.interleaved ? 8 * p : 16 * p, d1 = turned && !a.interleaved ? a.rd / 2 + 8 * p : 16 * p + 8;

    f16x8 wq[2], wk[2];
    if constexpr (NORM) {
        const f16x8 one = {1.0f16, 1.0f16, 1.0f16, 1.0f16, 1.0f16, 1.0f16, 1.0f16, 1.0f16};
        wq[0] = wq[1] = wk[0] = wk[1] = one;
        if (a.q_weight) {
            wq[0] = *reinterpret_cast<const f16x8 *>(a.q_weight + d0);
            wq[1] = *reinterpret_cast<const f16x8 *>(a.q_weight + d1);
        }
        if (a.k_weight) {
            wk[0] = *reinterpret_cast<const f16x8 *>(a.k_weight + d0);
            wk[1] = *reinterpret_cast<const f16x8 *>(a.k_weight + d1);
        }
    }
    f16x8 x[kHeads][2];
    auto  fetch = [&](int n) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const int h = h_first + (n + u) * hs;
            if (n + u < per && h < H && t < a.T) {
                const __half *src = h < a.Hq ? a.q + t * a.q_stride + (int64_t)h * D : a.k + t * a.k_stride + (int64_t)(h - a.Hq) * D;
                x[u][0] = *reinterpret_cast<const f16x8 *>(src + d0);
                x[u][1] = *reinterpret_cast<const f16x8 *>(src + d1);
            }
        }
    };
    fetch(0);
    // The block's angles, one a thread at a time, while its first rows are on their way.
    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int     pair = i % pairs;
        const int64_t at = t0 + i / pairs;
        if (at < a.T) {
            const double turn = (double)a.positions[(int64_t)a.axis[pair] * a.T + at] * a.turns[pair];
            float        sn, cs;
            sincospif(2.0f * (float)(turn - __builtin_rint(turn)), &sn, &cs);
            s_angle[i] = make_float2(cs, sn);
        }
    }
    __syncthreads();
    if (t >= a.T) return; // (whole rows: the sums below stay among a row's threads)
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 v = turned ? s_angle[(slot >> lg_hs) * pairs + 8 * p + i] : make_float2(1.0f, 0.0f);
        cs[i] = v.x;
        sn[i] = v.y;
    }
    for (int n = 0; n < per; n += kHeads) {
        if (n) fetch(n);
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const int h = h_first + (n + u) * hs;
            if (n + u >= per || h >= H) continue;
            const bool is_q = h < a.Hq;
            float      y[2][8];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) y[s][i] = (float)x[u][s][i];
            if constexpr (NORM) {
                float sum = 0.0f;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = fmaf(y[s][i], y[s][i], sum);
#pragma unroll
                for (int o = 1; o < LPR; o <<= 1) sum += __shfl_xor(sum, o);
                if (is_q ? a.q_weight != nullptr : a.k_weight != nullptr) {
                    const float r = 1.0f / sqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[s][i] = y[s][i] * r * (float)(is_q ? wq[s][i] : wk[s][i]);
                }
            }
            f16x8 z[2];
            if (turned && a.interleaved) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float c = cs[4 * s + i / 2], w = sn[4 * s + i / 2];
                        z[s][i] = (_Float16)(y[s][i] * c - y[s][i + 1] * w);
                        z[s][i + 1] = (_Float16)(y[s][i] * w + y[s][i + 1] * c);
                    }
            } else { // (not turned: by the angle 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    z[0][i] = (_Float16)(turned ? y[0][i] * cs[i] - y[1][i] * sn[i] : y[0][i]);
                    z[1][i] = (_Float16)(turned ? y[0][i] * sn[i] + y[1][i] * cs[i] : y[1][i]);
                }
            }
            __half *dst = is_q ? a.q_out + (t * a.Hq + h) * D : a.k_out + (t * a.Hkv + h - a.Hq) * D;
            *reinterpret_cast<f16x8 *>(dst + d0) = z[0];
            *reinterpret_cast<f16x8 *>(dst + d1) = z[1];
        }
    }
}

template <int D> void launch_d(const RotaryCall &c, dim3 grid, int lg_hs, int per, hipStream_t stream) {
    if (c.q_weight || c.k_weight) hipLaunchKernelGGL((rotary_kernel<D, true>), grid, dim3(kThreads), 0, stream, c, lg_hs, per);
    else hipLaunchKernelGGL((rotary_kernel<D, false>), grid, dim3(kThreads), 0, stream, c, lg_hs, per);
}

} // namespace

bool launch_rotary(const RotaryCall &c, int D, hipStream_t stream) {
    const int     slots = kThreads / (D / 16), H = c.Hq + c.Hkv, cus = device_cus();
    const int64_t rows = (int64_t)c.T * H;
    // A thread takes one head while there are few rows, up to eight of its token where they fill the chip.
    int64_t per = std::max<int64_t>(1, std::min<int64_t>(8, rows / ((int64_t)slots * 8 * cus)));
    int     lg_hs = 0;
    while ((1 << lg_hs) < slots && ((int64_t)per << lg_hs) < H) ++lg_hs;
    const int64_t heads = per << lg_hs, tokens = slots >> lg_hs;
    const int64_t x = (c.T + tokens - 1) / tokens, y = (H + heads - 1) / heads;
    if (x * y > (int64_t(1) << 32) / kThreads - 1 || y > 65535) return false;
    const dim3 grid((unsigned)x, (unsigned)y);
    profile_begin(KernelId::Rotary, stream);
    switch (D) {
    case 32: launch_d<32>(c, grid, lg_hs, (int)per, stream); break;
    case 64: launch_d<64>(c, grid, lg_hs, (int)per, stream); break;
    case 128: launch_d<128>(c, grid, lg_hs, (int)per, stream); break;
    case 256: launch_d<256>(c, grid, lg_hs, (int)per, stream); break;
    default: throw std::invalid_argument("rotary: unsupported head_dim");
    }
    HIP_CHECK(hipGetLastError());
    profile_end(KernelId::Rotary, stream);
    return true;
}

} // namespace detail
} // namespace tiny_llm
