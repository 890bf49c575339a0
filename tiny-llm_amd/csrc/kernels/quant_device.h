// Device functions of the kernels of a cache in 8 bits (layout: quant.h).
#pragma once

#include "quant.h"

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <type_traits>

namespace tiny_llm {
namespace detail {
namespace quant {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Pieces are numbered so that lane l of a wave has pieces 2 (64 s + l) and 2 (64 s + l) + 1 of
// K: dims 32 s + 8 (l / 16) .. + 7 of the tokens l % 16 and 16 + l % 16; of V: dims 32 s + l % 16 and
// 32 s + 16 + l % 16 of the tokens 4 (l / 16) .. + 3 and 16 more.
__device__ __forceinline__ int k_piece(int r, int o) { return ((o >> 2) * 64 + (o & 3) * 16 + (r & 15)) * 2 + (r >> 4); }
__device__ __forceinline__ int v_piece(int q, int d) { return ((d >> 5) * 64 + q * 16 + (d & 15)) * 2 + ((d >> 4) & 1); }
// Half of token r and dim d in V's pieces.
__device__ __forceinline__ int v_half(int r, int d) { return v_piece((r & 15) >> 2, d) * 8 + 4 * (r >> 4) + (r & 3); }

// Four stored bytes as whole numbers in fp16: 0x6400 | x is 1024 + x, and 1152 = 1024 + 128.
__device__ __forceinline__ u32x2 whole4(uint32_t w) {
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
    return u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}
__device__ __forceinline__ f16x8 whole8(uint32_t a, uint32_t b) {
    const u32x2 lo = whole4(a), hi = whole4(b);
    return __builtin_bit_cast(f16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
}

// The scale of a group from the bits of its largest magnitude in fp16: / 127, cut down to
// 11 significant bits, NaN where the group holds a value that is not finite.  Cut down, so
// that 127 steps never exceed the largest value (nor 65504), while that value is at most 127.13
// steps; and with 11 bits a quotient x / s that is not itself a half-integer is at least 2^-19
// of one away from it, so that fp32 rounds every quotient to the right whole number.
__device__ __forceinline__ float group_scale(uint32_t most) {
    if (most >= 0x7C00u) return __builtin_nanf("");
    const float a = __half2float(__builtin_bit_cast(__half, (uint16_t)most));
    return __uint_as_float(__float_as_uint(a / 127.0f) & 0xFFFFE000u);
}

// The last entry whose first item is at most `item`.
#define QUANT_ENTRY_OF(a, item, out)                                                                                   \
    do {                                                                                                               \
        int seen_ = 0;                                                                                                 \
        for (int k_ = 0; k_ < (a).n; k_ += 64) {                                                                       \
            const int i_ = k_ + (int)(threadIdx.x & 63);                                                               \
            seen_ += __popcll(__ballot(i_ < (a).n && (a).e[min(i_, (a).n - 1)].item0 <= (item)));                      \
        }                                                                                                              \
        out = __builtin_amdgcn_readfirstlane(seen_ - 1);                                                               \
    } while (0)

// Workgroup b of a grid of quant_grid(items, Hkv): the heads of an item on one XCD (workgroups
// go to the eight in turn), eight items at a time, so that an XCD's address translation serves
// an eighth of the sequences' pages.
__host__ __device__ inline int64_t quant_grid(int64_t items, int Hkv) { return (items + 7) / 8 * 8 * Hkv; }
__device__ __forceinline__ void quant_place(int b, int Hkv, int &item, int &g) {
    const int eights = b / (8 * Hkv), rest = b - eights * 8 * Hkv;
    g = rest >> 3;
    item = eights * 8 + (rest & 7);
}

// Index of a group's tile and scales.
__device__ __forceinline__ int64_t tile_of(const QuantView &v, int Hkv, int row, int g, int group) {
    const int64_t block = v.table[(int64_t)row * v.bt_stride + (group >> v.lg)];
    return ((block * Hkv + g) << v.lg) + (group & ((1 << v.lg) - 1));
}
template <int D> __device__ __forceinline__ uint16_t *open_of(const QuantView &v, int Hkv, int row, int which, int g) {
    return reinterpret_cast<uint16_t *>(v.open) + (((int64_t)row * 2 + which) * Hkv + g) * (64 * D);
}

// Largest magnitude (bits) of two packed halves.
__device__ __forceinline__ uint32_t most_of(uint32_t most, uint32_t two) {
    const uint32_t lo = two & 0x7FFFu, hi = (two >> 16) & 0x7FFFu;
    return max(most, max(lo, hi));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
    return x;
}

// Round-half-even of x / s, + 128, in the low byte.  x * (1 / s) is two roundings off the
// quotient; one step of Newton's method with the exact remainder takes it to the nearest fp32
// value (a half-integer quotient exactly); adding 1.5 * 2^23 + 128 rounds to a whole number.
__device__ __forceinline__ uint32_t stored_byte(float x, float s, float inv) {
    float q = x * inv;
    q = fmaf(fmaf(-q, s, x), inv, q);
    return __float_as_uint(q + 12583040.0f);
}
__device__ __forceinline__ uint32_t stored4(uint32_t a, uint32_t b, float s, float inv) {
    const f16x2    x = __builtin_bit_cast(f16x2, a), y = __builtin_bit_cast(f16x2, b);
    const uint32_t lo = __builtin_amdgcn_perm(stored_byte((float)x[1], s, inv), stored_byte((float)x[0], s, inv), 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(stored_byte((float)y[1], s, inv), stored_byte((float)y[0], s, inv), 0x0C0C0400u);
    return lo | hi << 16;
}
// 16 halves (two pieces) as stored bytes.
__device__ __forceinline__ u32x4 stored16(u32x4 a, u32x4 b, float s) {
    if (!(s > 0.0f)) return u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u}; // zeros; NaN: by the scale alone
    const float inv = 1.0f / s;
    return u32x4{stored4(a[0], a[1], s, inv), stored4(a[2], a[3], s, inv), stored4(b[0], b[1], s, inv), stored4(b[2], b[3], s, inv)};
}

// Closes a group: the pieces of `open` (64 D halves, in memory or LDS) as a tile and its
// scales.  By the NT threads of a workgroup; red: 2 NT / 64 words of LDS.
template <int D, int NT>
__device__ __forceinline__ void close_group(const uint16_t *open, uint8_t *tile, float2 *scale, uint32_t *red) {
    constexpr int PAIRS = 2 * D; // pairs of pieces of K, and of V
    constexpr int N = (2 * PAIRS + NT - 1) / NT;
    static_assert(PAIRS % 64 == 0, "a wave has pairs of K or of V");
    u32x4    a[N], b[N];
    uint32_t most[2] = {0u, 0u};
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int p = u * NT + (int)threadIdx.x;
        if (p < 2 * PAIRS) {
            const u32x4 *src = reinterpret_cast<const u32x4 *>(open) + 2 * p;
            a[u] = src[0];
            b[u] = src[1];
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = most_of(most_of(m, a[u][i]), b[u][i]);
            if (p < PAIRS) most[0] = max(most[0], m);
            else most[1] = max(most[1], m);
        }
    }
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const uint32_t m = wave_max(most[w]);
        if ((threadIdx.x & 63) == 0) red[w * (NT / 64) + wave] = m;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < NT / 64; ++k) m = max(m, red[w * (NT / 64) + k]);
        most[w] = m;
    }
    const float sk = group_scale(most[0]), sv = group_scale(most[1]);
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int p = u * NT + (int)threadIdx.x;
        if (p < 2 * PAIRS) reinterpret_cast<u32x4 *>(tile)[p] = stored16(a[u], b[u], p < PAIRS ? sk : sv);
    }
    if (threadIdx.x == 0) *scale = make_float2(sk, sv);
    __syncthreads(); // (red is free again)
}

// A wave's registers hold a group as the operands of the products: kf[tt][s] the token 16 tt +
// l % 16 (dims 32 s + 8 (l / 16) ..), vf[dt] the dim 16 dt + l % 16 (tokens 4 (l / 16) .. and 16 more).
template <int D> struct GroupRegs {
    static constexpr int KS = D / 32, DT = D / 16;
    f16x8                kf[2][KS], vf[DT];
    float                ks = 1.0f, vs = 1.0f;

    __device__ __forceinline__ void load(const uint16_t *open) {
        const f16x8 *k = reinterpret_cast<const f16x8 *>(open) + 2 * (threadIdx.x & 63), *v = k + 4 * D;
#pragma unroll
        for (int i = 0; i < KS; ++i) kf[0][i] = k[128 * i], kf[1][i] = k[128 * i + 1];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[dt] = v[128 * (dt / 2) + (dt & 1)];
    }
    // Token r of the group comes from rows of D halves: on their way to the lanes that take it ...
    f16x8    xk[KS];
    uint16_t xv[DT];
    __device__ __forceinline__ void fetch(int r, const uint16_t *new_k, const uint16_t *new_v) {
        const int c = threadIdx.x & 15, q = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int i = 0; i < KS; ++i) xk[i] = *reinterpret_cast<const f16x8 *>(new_k + 32 * i + 8 * q);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) xv[dt] = new_v[16 * dt + c];
    }
    // ... and into them and the open tile.
    __device__ __forceinline__ void append(uint16_t *open, int r) {
        const int  c = threadIdx.x & 15, q = (threadIdx.x & 63) >> 4, tr = r >> 4, slot = 4 * tr + (r & 3);
        const bool mine_k = c == (r & 15), mine_v = q == (r & 15) >> 2;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            if (mine_k) *reinterpret_cast<f16x8 *>(open + 8 * k_piece(r, 4 * i + q)) = xk[i];
            kf[0][i] = mine_k && !tr ? xk[i] : kf[0][i];
            kf[1][i] = mine_k && tr ? xk[i] : kf[1][i];
        }
        uint32_t mask[4]; // of the half that is replaced
#pragma unroll
        for (int w = 0; w < 4; ++w) mask[w] = mine_v && w == slot >> 1 ? (slot & 1 ? 0xFFFF0000u : 0x0000FFFFu) : 0u;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            if (mine_v) open[32 * D + v_half(r, 16 * dt + c)] = xv[dt];
            u32x4          v = __builtin_bit_cast(u32x4, vf[dt]);
            const uint32_t x = xv[dt] | (uint32_t)xv[dt] << 16;
#pragma unroll
            for (int w = 0; w < 4; ++w) v[w] = (v[w] & ~mask[w]) | (x & mask[w]);
            vf[dt] = __builtin_bit_cast(f16x8, v);
        }
    }
    // The group's whole numbers and scales, in the registers and in the cache.
    __device__ __forceinline__ void close(uint8_t *tile, float2 *scale) {
        uint32_t mk = 0, mv = 0;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                mk = most_of(most_of(mk, __builtin_bit_cast(u32x4, kf[0][i])[x]), __builtin_bit_cast(u32x4, kf[1][i])[x]);
                mv = most_of(most_of(mv, __builtin_bit_cast(u32x4, vf[2 * i])[x]), __builtin_bit_cast(u32x4, vf[2 * i + 1])[x]);
            }
        ks = group_scale(wave_max(mk));
        vs = group_scale(wave_max(mv));
        u32x4 *to = reinterpret_cast<u32x4 *>(tile) + (threadIdx.x & 63);
        auto   put = [&](u32x4 *at, f16x8 &a, f16x8 &b, float s) __attribute__((always_inline)) {
            const u32x4 w = stored16(__builtin_bit_cast(u32x4, a), __builtin_bit_cast(u32x4, b), s);
            *at = w;
            a = whole8(w[0], w[1]);
            b = whole8(w[2], w[3]);
        };
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            put(to + 64 * i, kf[0][i], kf[1][i], ks);
            put(to + 2 * D + 64 * i, vf[2 * i], vf[2 * i + 1], vs);
        }
        if ((threadIdx.x & 63) == 0) *scale = make_float2(ks, vs);
    }
};

template <typename F> void for_head_dim(int D, F &&f) {
    switch (D) {
    case 32: f(std::integral_constant<int, 32>()); break;
    case 64: f(std::integral_constant<int, 64>()); break;
    case 128: f(std::integral_constant<int, 128>()); break;
    case 256: f(std::integral_constant<int, 256>()); break;
    default: throw std::invalid_argument("8-bit cache: unsupported head_dim");
    }
}

} // namespace quant
} // namespace detail
} // namespace tiny_llm
