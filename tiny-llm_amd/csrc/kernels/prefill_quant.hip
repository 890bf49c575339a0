// Causal attention of many query rows over a cache in 8 bits (layout: quant.h), for gfx950.
//
// Query token j of an entry (nq of them, the last at position S - 1) attends to the tokens
// 0 .. S - nq + j; the formulas are those of attention_quant.hip.  Bound by the matrix units:
// 4 D operations a query row and token, and K and V pass through the CUs once per tile of
// rows.
//
// quant_prefill_kernel: a workgroup of four waves at head_dim 128 and of eight elsewhere, two a CU up to
// head_dim 128 (figures: quant_prefill_waves), per (row tile, chunk of key tiles, kv head);
// a wave has 32 rows (16 at head_dim 256: tokens x heads of the kv head).  A tile of 64 tokens (32 at
// head_dim 256) is loaded as stored while the one before is computed, made fp16 once per workgroup and put
// into one of two LDS buffers as operands, 16 bytes a lane in lane order, so that every LDS access is
// a whole row of the banks:
//   K   whole numbers, exact in fp16; a group's scale meets the scores, in the softmax's fma
//   V   times the scale's first 4 bits, exact in fp16 too (7 + 4 bits); what the scale is
//       more than that, below 1.125 times, meets the weights in the softmax's exponent, and
//       the row sums are freed of it.  Scaling the products instead would cost as
//       much as the softmax.  (V times the whole scale, rounded: 564 us below in place of 570, and the
//       error of outputs 3.6e-4 in place of 2.9e-4, of which the outputs' own rounding is 2.1e-4)
//   P   rounded to fp16, 2^-11 with errors of either sign, and summed as rounded: with V's rounding below
//       scales of 2^-14 (scale_values) all that there is between the stored numbers and the output's
//       rounding.  The lower halves as a second product, as in attention_quant.hip, would take the
//       error from 2.9e-4 to 2.1e-4, and 8192 tokens from 594 us to 782, 4 x 400 .. 512 over 2500 .. 6000 from 181
//       to 236; at head_dim 64 they do not fit the 128 registers.
//   S^T = K Q^T, O^T += V^T P^T by v_mfma_f32_16x16x32_f16 as in attention_quant.hip; the row
//   sums of P by a product with ones
// 8192 tokens, 32 heads over 8 of 128: 566-618 us by card and clock, 0.89-0.97 PFLOP/s (a large fp16 product takes
// 1.10-1.17).  Of a SIMD's cycles MFMA takes 38-41%, VALU 37-40%; the LDS is read
// 40% of the time, without bank conflicts.  What is left are the two waves of a SIMD waiting for each
// other at barriers and for operands: a third needs 168 registers, and a wave has 219.
// Tried and slower: eight waves of which four multiply while four do their softmax (636),
// one group a step, priorities around the products.
// quant_prefill_merge_kernel: joins the chunks of entries whose keys were split.
#include "quant_device.h"

#include "../runtime.h"
#include "kv_kernels.h"
#include "tiny_llm/hip_utils.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace tiny_llm {
namespace detail {

namespace {

using namespace quant;

constexpr float kBelow = 7.0f, kLazyMax = 15.0f; // (see attention_quant.hip)
constexpr float kNone = -3e38f;

struct PrefillArgs {
    const uint16_t   *q;
    uint16_t         *out;
    float            *part_o;  // [item][Hkv][ROWS][D]
    float            *part_ml; // [item][Hkv][ROWS][2]
    QuantView         v;
    float             scale_log2; // positive
    int               negate;
    int               Hq, Hkv, lgG, n;
    QuantPrefillEntry e[kQuantPrefillBatch];
};
static_assert(sizeof(PrefillArgs) <= 4096, "kernel arguments");

template <int S> __device__ __forceinline__ float xor_lane_max(float x) {
    const unsigned u = __float_as_uint(x);
    if constexpr (S == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
}

// The first 4 significant bits of a scale.
__device__ __forceinline__ float coarse(float s) { return __uint_as_float(__float_as_uint(s) & 0xFFF00000u); }

// A group's values in fp16 from its whole numbers and a scale of 4 bits: exact where the scale
// is a normal fp16 number; a smaller one by way of its 2^17-fold.  The result is then rounded
// where it is subnormal, by at most 2^-25, and the weights' part of 1 (1.125 with the scale's rest) of
// that in an output is no more than half the last place of the smallest fp16 numbers.
constexpr uint32_t kLeastHalf = 0x38800000u, kInfinite = 0x7F800000u; // bits of 2^-14, and of infinity
template <bool SMALL> __device__ __forceinline__ void scale_values(u32x4 &x, uint32_t scale_bits) {
    const bool     twice = SMALL && scale_bits < kLeastHalf;
    const float    s = coarse(__uint_as_float(scale_bits));
    const _Float16 one = (_Float16)(SMALL && scale_bits > kInfinite ? 0.0f : twice ? s * 131072.0f : s); // (NaN: its rows have it from their scores)
    f16x2          y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __builtin_bit_cast(f16x2, (uint32_t)x[j]) * f16x2{one, one};
    if (SMALL && twice) {
        const _Float16 then = (_Float16)(1.0f / 131072.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] *= f16x2{then, then};
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __builtin_bit_cast(uint32_t, y[j]);
}

template <int D>
__global__ __launch_bounds__(quant_prefill_waves(D) * 64) __attribute__((amdgpu_waves_per_eu(quant_prefill_waves(D) * quant_prefill_per_cu(D) / 4))) void
quant_prefill_kernel(PrefillArgs a) {
    constexpr int NW = quant_prefill_waves(D), ROWS = quant_prefill_rows(D);
    constexpr int R = ROWS / NW, NQG = R / 16;                      // rows of a wave, in parts of 16
    constexpr int TILE = quant_prefill_tile(D), NG = TILE / kGroup; // tokens and groups of a tile
    constexpr int KS = D / 32, DT = D / 16;
    constexpr int UNITS = 2 * NG * KS;                  // of a tile: 64 pairs of pieces, K's first, then V's
    constexpr int NU = (UNITS + NW - 1) / NW;           // of a wave: units wave, NW + wave, ...
    __shared__ __align__(16) uint16_t s_k[2][TILE * D], s_v[2][TILE * D];
    __shared__ float4                 s_scale[2][NG]; // the tiles' groups': x K's scale, 1 of an open one, NaN where
                                                      // V's is; y log2 of V's over its first 4 bits, z 1 over it
    __shared__ int                    s_odd;          // the open group has values that are not finite

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    QUANT_ENTRY_OF(a, item, ei);
    const int row = a.e[ei].row, S = a.e[ei].S, tok0 = a.e[ei].tok0, nq = a.e[ei].nq, open = a.e[ei].open, nch = a.e[ei].nch;
    const int rows = nq << a.lgG;
    const int rel = item - a.e[ei].item0, ch = rel % nch, rt = (rows + ROWS - 1) / ROWS - 1 - rel / nch;
    const int seen = S - nq + 1 + ((min(rows, (rt + 1) * ROWS) - 1) >> a.lgG); // tokens that the row tile sees
    const int tiles = (seen + TILE - 1) / TILE;
    const int t_lo = (int)((int64_t)ch * tiles / nch), t_n = (int)((int64_t)(ch + 1) * tiles / nch) - t_lo;
    const int closed = open < 0 ? S : S / kGroup * kGroup;
    const int groups = (closed + kGroup - 1) / kGroup;
    const int c = lane & 15, qg = lane >> 4;
    if (tid == 0) s_odd = 0;

    auto row_of = [&](int r) -> int64_t { // element offset of query row r in q and out
        return ((int64_t)(tok0 + (r >> a.lgG)) * a.Hq + (g << a.lgG) + (r & ((1 << a.lgG) - 1))) * D;
    };
    const int r_w = rt * ROWS + wave * R; // the wave's first row
    f16x8     qb[NQG][KS];
    auto      seen_by = [&](int j) { return S - nq + 1 + (min(r_w + j * 16 + c, rows - 1) >> a.lgG); }; // tokens that row c of part j sees
#pragma unroll
    for (int j = 0; j < NQG; ++j) {
        const int       r = min(r_w + j * 16 + c, rows - 1);
        const uint16_t *qp = a.q + row_of(r);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            // (a negative scale's sign goes into q: the maximum over s is then that over s * scale)
            const f16x8 v = *reinterpret_cast<const f16x8 *>(qp + 32 * s + 8 * qg);
            qb[j][s] = a.negate ? -v : v;
        }
    }
    const int all = S - nq + 1 + (min(r_w, rows - 1) >> a.lgG); // tokens that every row of the wave sees,
    const int some = r_w < rows ? S - nq + 1 + (min(r_w + R - 1, rows - 1) >> a.lgG) : 0; // and that some row does

    // Tile i of the chunk.  at: where the next one to load has its groups, lane k group k; made of
    // blocks that were asked for a tile earlier.
    const int32_t *bt = a.v.table + (int64_t)row * a.v.bt_stride;
    const int      lane_g = min(lane, NG - 1);
    u32x4          raw[NU];
    float2         sc = {}; // scales of the loaded tile's groups, lane k those of group k.  (Loaded per lane: a
                            // scalar load would be waited for with the LDS accesses, at every barrier.)
    int            id = 0;
    auto           group_of = [&](int i) { return max(0, min(NG * (t_lo + i) + lane_g, groups - 1)); };
    auto           blocks = [&](int i) { id = bt[group_of(i) >> a.v.lg]; };
    auto           load = [&](int i) __attribute__((always_inline)) {
        if (groups == 0) return;
        const int64_t  at = (((int64_t)id * a.Hkv + g) << a.v.lg) + (group_of(i) & ((1 << a.v.lg) - 1));
        const uint8_t *tile = a.v.tiles + at * (64 * D);
        sc = a.v.scales[at];
        const __attribute__((address_space(1))) uint8_t *base[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const uint64_t x = reinterpret_cast<uint64_t>(tile);
            base[k] = reinterpret_cast<const __attribute__((address_space(1))) uint8_t *>((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, k) |
                                                        (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), k) << 32);
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int q = u * NW + wave;
            if (UNITS % NW != 0 && q >= UNITS) break;
            const int x = q % (NG * KS);
            raw[u] = *reinterpret_cast<const __attribute__((address_space(1))) u32x4 *>((NG == 2 && x >= KS ? base[NG - 1] : base[0]) +
                                                      ((q >= NG * KS ? 2 * D : 0) + x % KS * 64 + lane) * 16);
        }
        blocks(i + 1);
    };
    auto stage = [&](int i) __attribute__((always_inline)) {
        u32x4     *k16 = reinterpret_cast<u32x4 *>(s_k[i % 2]) + lane, *v16 = reinterpret_cast<u32x4 *>(s_v[i % 2]) + lane;
        const int  group0 = NG * (t_lo + i);
        if (wave == 0 && lane < NG) {
            const bool  closed_one = group0 + lane < groups;
            const float y = closed_one ? fmaxf(sc.y, 1e-37f) : 1.0f; // (not 0, not NaN)
            const float less = coarse(y);
            s_scale[i % 2][lane] = make_float4(closed_one ? (sc.y == sc.y ? sc.x : sc.y) : 1.0f,
                                               __builtin_amdgcn_logf(y * __builtin_amdgcn_rcpf(less)),
                                               less * __builtin_amdgcn_rcpf(y), 0.0f);
        }
        auto unit = [&](int u, auto place) __attribute__((always_inline)) {
            const int  q = u * NW + wave, k = q % (NG * KS) / KS, st = q % KS;
            const bool is_v = q >= NG * KS;
            u32x4      x[2];
            place(x, is_v, k, st, u);
            u32x4 *to = is_v ? v16 + (k * DT + 2 * st) * 64 : k16 + (2 * k * KS + st) * 64;
            to[0] = x[0];
            to[(is_v ? 1 : KS) * 64] = x[1];
        };
        const uint32_t vs0 = __builtin_amdgcn_readlane(__float_as_uint(sc.y), 0); // the groups' value scales' bits
        const uint32_t vs1 = __builtin_amdgcn_readlane(__float_as_uint(sc.y), NG - 1);
        const bool     plain = group0 + NG <= groups && vs0 - kLeastHalf < kInfinite - kLeastHalf && vs1 - kLeastHalf < kInfinite - kLeastHalf;
        auto stored = [&](u32x4 *x, bool is_v, int k, int u, auto small) __attribute__((always_inline)) {
            const u32x4 w = raw[u];
#pragma unroll
            for (int h = 0; h < 2; ++h) x[h] = __builtin_bit_cast(u32x4, whole8(w[2 * h], w[2 * h + 1]));
            if (is_v)
#pragma unroll
                for (int h = 0; h < 2; ++h) scale_values<decltype(small)::value>(x[h], k == 0 ? vs0 : vs1);
        };
        auto normal = [&](u32x4 *x, bool is_v, int k, int, int u) __attribute__((always_inline)) {
            stored(x, is_v, k, u, std::false_type{});
        };
        auto any = [&](u32x4 *x, bool is_v, int k, int st, int u) __attribute__((always_inline)) {
            const int group = group0 + k;
            if (group < groups) return stored(x, is_v, k, u, std::true_type{});
            x[0] = x[1] = u32x4{0u, 0u, 0u, 0u};
            if (open < 0 || group != groups) return;
            const u32x4 *src = reinterpret_cast<const u32x4 *>(open_of<D>(a.v, a.Hkv, row, open, g)) +
                               2 * ((is_v ? 2 * D : 0) + st * 64 + lane);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[h] = src[h];
                if (is_v) { // 0 times what is behind the last token, or not finite, could be NaN
                    f16x8 v = __builtin_bit_cast(f16x8, x[h]);
                    bool  odd = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool there = group * kGroup + 16 * (j >> 2) + 4 * qg + (j & 3) < S;
                        const bool finite = __builtin_fabsf16(v[j]) <= (_Float16)65504.0f;
                        odd |= there && !finite;
                        if (!there || !finite) v[j] = (_Float16)0.0f;
                    }
                    if (odd) s_odd = 1;
                    x[h] = __builtin_bit_cast(u32x4, v);
                }
            }
        };
        if (__builtin_expect(plain, 1)) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
                if (UNITS % NW == 0 || u * NW + wave < UNITS) unit(u, normal);
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u)
                if (UNITS % NW == 0 || u * NW + wave < UNITS) unit(u, any);
        }
    };

    f32x4 acc[NQG][DT], s[NQG][2 * NG];
    f16x8 pf[NQG][NG];
    float m_run[NQG], l_run[NQG];
    float4 of[NG]; // s_scale of the tile
#pragma unroll
    for (int j = 0; j < NQG; ++j) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[j][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        l_run[j] = 0.0f;
        m_run[j] = kNone;
    }

    const f16x8 ones = __builtin_bit_cast(f16x8, u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});

    // Operands come from LDS in batches, the next one on its way while one is multiplied.  (Left to itself the
    // compiler reads two and waits for them: 607 us where this took 598.)
    // (Two at head_dim 64, and those of the values behind the softmax: 128 registers.)
    constexpr int BATCH = D == 64 ? 2 : 4, NB = 2 * NG * KS / BATCH; // batches of scores, and of values
    f16x8         kf[BATCH], vf[BATCH];
    auto scores_batch = [&](int i, int b, f16x8 *f) __attribute__((always_inline)) { // keys 16 tt .., dims 32 st ..
        const f16x8 *k16 = reinterpret_cast<const f16x8 *>(s_k[i % 2]) + lane;
#pragma unroll
        for (int u = 0; u < BATCH; ++u) f[u] = k16[(BATCH * b + u) * 64];
    };
    auto values_batch = [&](int i, int b, f16x8 *f) __attribute__((always_inline)) {
        const f16x8 *v16 = reinterpret_cast<const f16x8 *>(s_v[i % 2]) + lane;
#pragma unroll
        for (int u = 0; u < BATCH; ++u) f[u] = v16[(BATCH * b + u) * 64];
    };
    // (the first batch is in kf, vf)
    auto scores = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < 2 * NG; ++tt)
#pragma unroll
            for (int j = 0; j < NQG; ++j) s[j][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f16x8 next[BATCH];
            if (b + 1 < NB) scores_batch(i, b + 1, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
#pragma unroll
                for (int j = 0; j < NQG; ++j) {
                    const int tt = (BATCH * b + u) / KS, st = (BATCH * b + u) % KS;
                    s[j][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[u], qb[j][st], s[j][tt], 0, 0, 0);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (b + 1 < NB)
#pragma unroll
                for (int u = 0; u < BATCH; ++u) kf[u] = next[u];
        }
    };
    auto softmax = [&](int i) __attribute__((always_inline)) {
        const int t0 = (t_lo + i) * TILE;
        float     f[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) f[k] = a.scale_log2 * of[k].x;
        if (__builtin_expect(t0 + TILE > all, 0)) { // some score does not count
#pragma unroll
            for (int j = 0; j < NQG; ++j) {
                const int end = seen_by(j) - t0 - 4 * qg;
#pragma unroll
                for (int tt = 0; tt < 2 * NG; ++tt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[j][tt][x] = 16 * tt + x < end ? s[j][tt][x] * f[tt >> 1] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < NG; ++k) f[k] = 1.0f;
        }
#pragma unroll
        for (int j = 0; j < NQG; ++j) {
            float mloc = -INFINITY;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                float mk = -INFINITY;
#pragma unroll
                for (int x = 0; x < 8; ++x) mk = __builtin_elementwise_maximum(mk, s[j][2 * k + (x >> 2)][x & 3]);
                mloc = __builtin_elementwise_maximum(mloc, mk * f[k]); // (NaN: of a group that all rows see, or in scores)
            }
            if (__builtin_expect(__any(mloc > m_run[j] + kLazyMax), 0)) {
                const float m_tile = xor_lane_max<32>(xor_lane_max<16>(mloc));
                const float m_new = fmaxf(m_run[j], m_tile - kBelow);
                const float alpha = m_run[j] == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run[j] - m_new);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[j][dt] *= alpha;
                l_run[j] *= alpha;
                m_run[j] = m_new;
            }
            float less[NG];
#pragma unroll
            for (int k = 0; k < NG; ++k) less[k] = of[k].y - m_run[j];
#pragma unroll
            for (int tt = 0; tt < 2 * NG; ++tt)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    pf[j][tt >> 1][4 * (tt & 1) + x] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[j][tt][x], f[tt >> 1], less[tt >> 1]));
        }
    };
    auto values = [&](int i) __attribute__((always_inline)) {
        f32x4 sums[NQG][NG];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f16x8 next[BATCH];
            if (b + 1 < NB) values_batch(i, b + 1, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
#pragma unroll
                for (int j = 0; j < NQG; ++j) {
                    const int k = (BATCH * b + u) / DT, dt = (BATCH * b + u) % DT;
                    if (dt == 0) sums[j][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[j][k], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                    acc[j][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[u], pf[j][k], acc[j][dt], 0, 0, 0);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (b + 1 < NB)
#pragma unroll
                for (int u = 0; u < BATCH; ++u) vf[u] = next[u];
        }
#pragma unroll
        for (int j = 0; j < NQG; ++j)
#pragma unroll
            for (int k = 0; k < NG; ++k) l_run[j] = __builtin_fmaf(of[k].z, sums[j][k][0], l_run[j]);
    };
    if (t_n > 0) {
        blocks(0);
        load(0);
        __syncthreads(); // s_odd
        stage(0);
        if (t_n > 1) load(1);
        __syncthreads();
        for (int i = 0; i < t_n; ++i) {
            if ((t_lo + i) * TILE < some) { // some row of the wave sees the tile
                scores_batch(i, 0, kf);
#pragma unroll
                for (int k = 0; k < NG; ++k) of[k] = s_scale[i % 2][k];
                scores(i);
                if (D != 64) values_batch(i, 0, vf);
                softmax(i);
                if (D == 64) values_batch(i, 0, vf);
                values(i);
            }
            if (i + 1 < t_n) stage(i + 1);
            if (i + 2 < t_n) load(i + 2);
            __syncthreads();
        }
    }
    // (behind every product: a value that is infinite decides)
    if (open >= 0 && t_n > 0 && (t_lo + t_n) * NG > groups && s_odd) { // the open group's values that are not finite, token by token
        const int       first = groups * kGroup;
        const uint16_t *tile = open_of<D>(a.v, a.Hkv, row, open, g) + 32 * D;
        for (int r = 0; r < S - first; ++r)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float y = (float)__builtin_bit_cast(_Float16, tile[v_half(r, 16 * dt + 4 * qg + x)]);
#pragma unroll
                    for (int j = 0; j < NQG; ++j)
                        if (!(__builtin_fabsf(y) <= 65504.0f) && first + r < seen_by(j)) acc[j][dt][x] += y;
                }
    }

    const int64_t p0 = ((int64_t)item * a.Hkv + g) * ROWS;
#pragma unroll
    for (int j = 0; j < NQG; ++j) {
        const int r = wave * R + j * 16 + c;
        if (rt * ROWS + r >= rows) continue;
        if (nch > 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                *reinterpret_cast<f32x4 *>(a.part_o + (p0 + r) * D + 16 * dt + 4 * qg) = acc[j][dt];
            if (qg == 0) *reinterpret_cast<float2 *>(a.part_ml + (p0 + r) * 2) = make_float2(m_run[j], l_run[j]);
            continue;
        }
        const float inv = 1.0f / (l_run[j] + 1e-6f);
        uint16_t   *op = a.out + row_of(rt * ROWS + r);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const __half2 lo = __floats2half2_rn(acc[j][dt][0] * inv, acc[j][dt][1] * inv);
            const __half2 hi = __floats2half2_rn(acc[j][dt][2] * inv, acc[j][dt][3] * inv);
            *reinterpret_cast<u32x2 *>(op + 16 * dt + 4 * qg) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
        }
    }
}

constexpr int kMergeThreads = 256, kMergeChunks = 4; // chunks on their way at once

// Workgroup (row tile of a cut entry, kv head; a few rows): `split` times D / 4 threads a row, which meet in
// LDS.  (A workgroup for every item,
// all but a row tile's first leaving at once: 14 us where this takes 8.6, 512 items of 80 row tiles.)
__global__ __launch_bounds__(kMergeThreads) void quant_prefill_merge_kernel(PrefillArgs a, int D, int ROWS, int split) {
    __shared__ f32x4  s_o[kMergeThreads];
    __shared__ float2 s_ml[kMergeThreads];
    const int b = blockIdx.x / a.Hkv, g = blockIdx.x - b * a.Hkv;
    // Row tile b of those of cut entries, in the entries' order.
    int ei = 0, before = 0;
    for (int k = 0; k < a.n; k += 64) {
        const int i = k + (int)(threadIdx.x & 63);
        int       own = i < a.n && a.e[i].nch > 1 ? ((a.e[i].nq << a.lgG) + ROWS - 1) / ROWS : 0;
        const int mine = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int other = __shfl_up(own, o);
            if ((int)(threadIdx.x & 63) >= o) own += other;
        }
        const uint64_t in = __ballot(before + own > b);
        if (in) {
            const int l = __builtin_ctzll(in);
            ei = k + l;
            before += __shfl(own - mine, l);
            break;
        }
        before += __shfl(own, 63);
    }
    const int nch = a.e[ei].nch, rel = (b - before) * nch, item = a.e[ei].item0 + rel;
    const int per = D / 4, grp = threadIdx.x / per, part = grp % split, d = 4 * (threadIdx.x % per);
    const int r = blockIdx.y * (kMergeThreads / per / split) + grp / split;
    const int rows = a.e[ei].nq << a.lgG, rt = (rows + ROWS - 1) / ROWS - 1 - rel / nch, qr = rt * ROWS + r;
    const bool there = r < ROWS && qr < rows;
    const int64_t p0 = ((int64_t)item * a.Hkv + g) * ROWS + r, pc = (int64_t)a.Hkv * ROWS;
    float         m = kNone, l = 0.0f;
    f32x4         o = {0.0f, 0.0f, 0.0f, 0.0f};
    auto          raise = [&](float most) {
        const float by = __builtin_amdgcn_exp2f(m - most);
        l *= by;
        o *= by;
        m = most;
    };
    auto join = [&](float2 ml, f32x4 x) { // (ml.x at most m)
        const float wgt = __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(wgt, ml.y, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(wgt, x[i], o[i]);
    };
    for (int c0 = there ? part : nch; c0 < nch; c0 += kMergeChunks * split) {
        float2 ml[kMergeChunks];
        f32x4  x[kMergeChunks];
#pragma unroll
        for (int u = 0; u < kMergeChunks; ++u) {
            const int64_t pr = p0 + min(c0 + u * split, nch - 1) * pc;
            ml[u] = *reinterpret_cast<const float2 *>(a.part_ml + pr * 2);
            x[u] = *reinterpret_cast<const f32x4 *>(a.part_o + pr * D + d);
        }
        float most = m;
#pragma unroll
        for (int u = 0; u < kMergeChunks; ++u) most = fmaxf(most, ml[u].x);
        raise(most);
#pragma unroll
        for (int u = 0; u < kMergeChunks; ++u)
            if (c0 + u * split < nch) join(ml[u], x[u]);
    }
    if (split > 1) {
        s_o[threadIdx.x] = o;
        s_ml[threadIdx.x] = make_float2(m, l);
        __syncthreads();
        for (int k = 1; k < split && part == 0; ++k) {
            const float2 ml = s_ml[threadIdx.x + k * per];
            raise(fmaxf(m, ml.x));
            join(ml, s_o[threadIdx.x + k * per]);
        }
    }
    if (part != 0 || !there) return;
    const float   inv = 1.0f / (l + 1e-6f);
    const __half2 lo = __floats2half2_rn(o[0] * inv, o[1] * inv), hi = __floats2half2_rn(o[2] * inv, o[3] * inv);
    uint16_t     *op = a.out + ((int64_t)(a.e[ei].tok0 + (qr >> a.lgG)) * a.Hq + (g << a.lgG) + (qr & ((1 << a.lgG) - 1))) * D + d;
    *reinterpret_cast<u32x2 *>(op) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

size_t part_ml_floats(size_t rows) { return (2 * rows + 3) / 4 * 4; }

} // namespace

size_t quant_prefill_workspace_floats(const QuantPrefillPlan &plan, int Hkv, int D) {
    size_t most = 0;
    for (const auto &l : plan.launches) {
        const size_t rows = (size_t)l.parts * (size_t)quant_prefill_rows(D) * (size_t)Hkv;
        if (l.parts) most = std::max(most, part_ml_floats(rows) + rows * (size_t)D);
    }
    return most;
}

void launch_quant_prefill(const QuantCall &c, const QuantView &v, const QuantPrefillPlan &plan, float *workspace,
                          hipStream_t stream) {
    PrefillArgs a{};
    a.q = reinterpret_cast<const uint16_t *>(c.q);
    a.out = reinterpret_cast<uint16_t *>(c.out);
    a.v = v;
    a.scale_log2 = std::fabs(c.scale) * 1.4426950408889634f;
    a.negate = std::signbit(c.scale) ? 1 : 0;
    a.Hq = c.Hq;
    a.Hkv = c.Hkv;
    while ((c.Hkv << a.lgG) < c.Hq) ++a.lgG;
    const int ROWS = quant_prefill_rows(c.D);
    for (const auto &l : plan.launches) {
        if (l.n == 0 || l.items == 0) continue;
        if ((int64_t)l.items * c.Hkv > kQuantMostItems) throw std::invalid_argument("attention: too many work items");
        a.n = l.n;
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(QuantPrefillEntry) * (size_t)l.n);
        a.part_ml = workspace;
        a.part_o = l.parts ? workspace + part_ml_floats((size_t)l.parts * (size_t)ROWS * (size_t)c.Hkv) : nullptr;
        profile_begin(KernelId::PrefillQuant, stream);
        for_head_dim(c.D, [&](auto d) {
            constexpr int D = decltype(d)::value;
            hipLaunchKernelGGL(quant_prefill_kernel<D>, dim3((unsigned)l.items * (unsigned)a.Hkv),
                               dim3(quant_prefill_waves(D) * 64), 0, stream, a);
        });
        HIP_CHECK(hipGetLastError());
        if (l.parts) {
            int row_tiles = 0, most = 1, split = 1, rows = kMergeThreads / (c.D / 4);
            for (int i = 0; i < l.n; ++i)
                if (a.e[i].nch > 1) {
                    row_tiles += ((a.e[i].nq << a.lgG) + ROWS - 1) / ROWS;
                    most = std::max(most, a.e[i].nch);
                }
            // (while there are few: 3 x 291 tokens of one kv head, to 39 chunks of 15 row tiles, 31 us a call, 37 with one
            // thread; 100 of 8 heads of 64 over 30000 in 157 chunks 31, 47)
            while (rows > 1 && split * kMergeChunks < most && (int64_t)row_tiles * c.Hkv * (ROWS / rows) * 2 <= 8 * device_cus()) {
                split *= 2;
                rows /= 2;
            }
            hipLaunchKernelGGL(quant_prefill_merge_kernel, dim3((unsigned)(row_tiles * c.Hkv), (unsigned)((ROWS + rows - 1) / rows)),
                               dim3(kMergeThreads), 0, stream, a, c.D, ROWS, split);
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::PrefillQuant, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
