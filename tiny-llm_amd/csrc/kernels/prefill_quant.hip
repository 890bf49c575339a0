// Causal attention of many query rows over a cache in 8 bits (layout: quant.h), for gfx950.
//
// Query token j of an entry (nq of them, the last at position S - 1) attends to the tokens
// 0 .. S - nq + j; the formulas are those of attention_quant.hip.  Bound by the matrix units:
// 4 D operations a query row and token, and K and V pass through the CUs once per tile of
// rows.
//
// quant_prefill_kernel: a workgroup of NW waves per (row tile, chunk of key tiles, kv head);
// a wave has 32 rows (16 at head_dim 256: tokens x heads of the kv head).  A tile of 64 tokens is
// loaded as stored while the one before is computed, made fp16 once per workgroup and put
// into one of two LDS buffers as operands, 16 bytes a lane in lane order, so that every LDS access is
// a whole row of the banks:
//   K   whole numbers, exact in fp16; a group's scale meets the scores, in the softmax's fma
//   V   times the group's scale, rounded to fp16 (a rounding 2^-11 beside the 2^-8 of the
//       stored numbers): scaling the products instead would cost as much as the softmax
//   S^T = K Q^T, O^T += V^T P^T by v_mfma_f32_16x16x32_f16 as in attention_quant.hip; the row
//   sums of P by a product with ones
// quant_prefill_merge_kernel: joins the chunks of entries whose keys were split.
#include "quant_device.h"

#include "../runtime.h"
#include "kv_kernels.h"
#include "tiny_llm/hip_utils.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

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

// A group's values in fp16 from its whole numbers: one rounding where the scale is a normal
// fp16 number, which holds its 11 bits; a smaller scale by way of its 2^17-fold (the result
// is then rounded again where it is subnormal).
struct ValueScale {
    f16x2 by, then;
    bool  twice;
    __device__ explicit ValueScale(float s) {
        twice = s < 6.103515625e-05f;
        const _Float16 a = (_Float16)(twice ? s * 131072.0f : s), b = (_Float16)(1.0f / 131072.0f);
        by = f16x2{a, a};
        then = f16x2{b, b};
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
        f16x2 y = __builtin_bit_cast(f16x2, x) * by;
        if (twice) y = y * then;
        return __builtin_bit_cast(uint32_t, y);
    }
};

template <int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void
quant_prefill_kernel(PrefillArgs a) {
    constexpr int NQG = D <= 128 ? 2 : 1; // 16-row parts of a wave
    constexpr int NT = NW * 64;
    constexpr int R = 16 * NQG;
    constexpr int ROWS = NW * R;
    static_assert(ROWS == quant_prefill_rows(D, NW), "the planner's row tile");
    constexpr int KS = D / 32, DT = D / 16;
    constexpr int PAIRS = 4 * D;                      // pairs of pieces of a group, K and V
    constexpr int NU = (2 * PAIRS + NT - 1) / NT;     // of a tile, per thread
    __shared__ __align__(16) uint16_t ks0[kQuantTile * D], ks1[kQuantTile * D];
    __shared__ __align__(16) uint16_t vs0[kQuantTile * D], vs1[kQuantTile * D];
    __shared__ int                    s_odd; // the open group has values that are not finite

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    QUANT_ENTRY_OF(a, item, ei);
    const int row = a.e[ei].row, S = a.e[ei].S, tok0 = a.e[ei].tok0, nq = a.e[ei].nq, open = a.e[ei].open, nch = a.e[ei].nch;
    const int rows = nq << a.lgG;
    const int rel = item - a.e[ei].item0, ch = rel % nch, rt = (rows + ROWS - 1) / ROWS - 1 - rel / nch;
    const int seen = S - nq + 1 + ((min(rows, (rt + 1) * ROWS) - 1) >> a.lgG); // tokens that the tile sees
    const int tiles = (seen + kQuantTile - 1) / kQuantTile;
    const int t_lo = (int)((int64_t)ch * tiles / nch), t_hi = (int)((int64_t)(ch + 1) * tiles / nch);
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
    const int all = S - nq + 1 + (min(r_w, rows - 1) >> a.lgG);         // tokens that every row of the wave sees,
    const int some = S - nq + 1 + (min(r_w + R - 1, rows - 1) >> a.lgG); // and that some row does

    // A wave's 64 pairs of a load lie in one group, K or V.
    const int32_t *bt = a.v.table + (int64_t)row * a.v.bt_stride;
    auto blocks = [&](int kt) -> int { return lane < 2 ? bt[max(0, min(2 * kt + lane, groups - 1)) >> a.v.lg] : 0; };
    auto tile_at = [&](int kt, int k, int ids) __attribute__((always_inline)) -> int64_t {
        const int i = min(2 * kt + k, groups - 1) & ((1 << a.v.lg) - 1);
        return (((int64_t)__builtin_amdgcn_readlane(ids, k) * a.Hkv + g) << a.v.lg) + i;
    };
    u32x4  raw[NU];
    float2 sc[2]; // scales of the loaded tile's groups
    auto   load = [&](int kt, int ids) __attribute__((always_inline)) {
        if (groups > 0) {
            int64_t at[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                at[k] = tile_at(kt, k, ids);
                sc[k] = a.v.scales[at[k]];
            }
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int p0 = u * NT + wave * 64; // wave-uniform
                if (2 * PAIRS % NT != 0 && p0 >= 2 * PAIRS) break;
                const int k = p0 / PAIRS;
                raw[u] = reinterpret_cast<const u32x4 *>(a.v.tiles + (k ? at[1] : at[0]) * (64 * D))[p0 % PAIRS + lane];
            }
        }
    };
    auto stage = [&](int kt, uint16_t *kd, uint16_t *vd) __attribute__((always_inline)) {
        u32x4 *k16 = reinterpret_cast<u32x4 *>(kd), *v16 = reinterpret_cast<u32x4 *>(vd);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int p0 = u * NT + wave * 64;
            if (2 * PAIRS % NT != 0 && p0 >= 2 * PAIRS) break;
            const int  k = p0 / PAIRS, s = p0 % (PAIRS / 2) / 64, group = 2 * kt + k;
            const bool is_v = p0 % PAIRS >= PAIRS / 2;
            u32x4      x[2];
            if (group < groups) {
                const u32x4 w = raw[u];
#pragma unroll
                for (int h = 0; h < 2; ++h) x[h] = __builtin_bit_cast(u32x4, whole8(w[2 * h], w[2 * h + 1]));
                if (is_v) {
                    const float vs = k ? sc[1].y : sc[0].y;
                    const ValueScale by(vs == vs ? vs : 0.0f); // (NaN: its rows get it below)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[h][i] = by(x[h][i]);
                }
            } else if (open >= 0 && group == groups) {
                const u32x4 *src = reinterpret_cast<const u32x4 *>(open_of<D>(a.v, a.Hkv, row, open, g)) + 2 * (p0 % PAIRS + lane);
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
            } else {
                x[0] = x[1] = u32x4{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!is_v) k16[((2 * k + h) * KS + s) * 64 + lane] = x[h];
                else v16[(k * DT + 2 * s + h) * 64 + lane] = x[h];
            }
        }
    };

    f32x4 acc[NQG][DT], l_run[NQG];
    float m_run[NQG];
#pragma unroll
    for (int j = 0; j < NQG; ++j) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[j][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        l_run[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m_run[j] = kNone;
    }
    const f16x8 ones = __builtin_bit_cast(f16x8, u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u});

    auto compute = [&](int kt, float2 now0, float2 now1, const uint16_t *kd, const uint16_t *vd) __attribute__((always_inline)) {
        const int t0 = kt * kQuantTile;
        if (t0 >= some) return; // no row of the wave sees the tile
        const f16x8 *k16 = reinterpret_cast<const f16x8 *>(kd) + lane, *v16 = reinterpret_cast<const f16x8 *>(vd) + lane;
        float        f[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) f[k] = a.scale_log2 * (2 * kt + k < groups ? (k ? now1 : now0).x : 1.0f);
        f32x4 s[NQG][4];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int j = 0; j < NQG; ++j) s[j][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int th = 0; th < 4; th += 2)
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                f16x8 kf[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) kf[u] = k16[((th + u) * KS + st) * 64];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < NQG; ++j)
                        s[j][th + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[u], qb[j][st], s[j][th + u], 0, 0, 0);
            }
        if (t0 + kQuantTile > all) { // some score does not count
#pragma unroll
            for (int j = 0; j < NQG; ++j)
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[j][tt][i] = t0 + 16 * tt + 4 * qg + i < seen_by(j) ? s[j][tt][i] * f[tt >> 1] : -INFINITY;
            f[0] = f[1] = 1.0f;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) // a group whose scale is NaN: the rows that see some of it
            if (const float vs = (k ? now1 : now0).y; 2 * kt + k < groups && !(vs == vs))
#pragma unroll
                for (int j = 0; j < NQG; ++j)
                    if (t0 + kGroup * k < seen_by(j)) l_run[j] += vs;
        f16x8 pf[NQG][2];
#pragma unroll
        for (int j = 0; j < NQG; ++j) {
            float mk[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mk[tt >> 1] = fmaxf(mk[tt >> 1], s[j][tt][i]);
            const float mloc = fmaxf(mk[0] * f[0], mk[1] * f[1]);
            if (__any(mloc > m_run[j] + kLazyMax)) {
                const float m_tile = xor_lane_max<32>(xor_lane_max<16>(mloc));
                const float m_new = fmaxf(m_run[j], m_tile - kBelow);
                const float alpha = m_run[j] == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run[j] - m_new);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[j][dt] *= alpha;
                l_run[j] *= alpha;
                m_run[j] = m_new;
            }
            const float m_new = m_run[j];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    pf[j][tt >> 1][4 * (tt & 1) + i] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[j][tt][i], f[tt >> 1], -m_new));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int j = 0; j < NQG; ++j) l_run[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[j][k], l_run[j], 0, 0, 0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const f16x8 vf = v16[(k * DT + dt) * 64];
#pragma unroll
                for (int j = 0; j < NQG; ++j) acc[j][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[j][k], acc[j][dt], 0, 0, 0);
            }
        }
        if (open >= 0 && 2 * kt + 1 >= groups && s_odd) { // the open group's values that are not finite, token by token
            const uint16_t *tile = open_of<D>(a.v, a.Hkv, row, open, g) + 32 * D;
            const int first = groups * kGroup;
            for (int r = 0; r < S - first; ++r)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = (float)__builtin_bit_cast(_Float16, tile[v_half(r, 16 * dt + 4 * qg + i)]);
#pragma unroll
                        for (int j = 0; j < NQG; ++j)
                            if (!(__builtin_fabsf(x) <= 65504.0f) && first + r < seen_by(j)) acc[j][dt][i] += x;
                    }
        }
    };

    if (t_lo < t_hi) {
        int    ids = blocks(t_lo), next = t_lo + 1 < t_hi ? blocks(t_lo + 1) : 0;
        __syncthreads(); // s_odd
        load(t_lo, ids);
        stage(t_lo, ks0, vs0);
        __syncthreads();
        auto step = [&](int kt, uint16_t *kd, uint16_t *vd, uint16_t *kn, uint16_t *vn) __attribute__((always_inline)) {
            const float2 now0 = sc[0], now1 = sc[1];
            const bool   more = kt + 1 < t_hi;
            if (more) {
                ids = next;
                if (kt + 2 < t_hi) next = blocks(kt + 2);
                load(kt + 1, ids);
            }
            compute(kt, now0, now1, kd, vd);
            if (more) stage(kt + 1, kn, vn);
            __syncthreads();
        };
        for (int kt = t_lo; kt < t_hi; kt += 2) {
            step(kt, ks0, vs0, ks1, vs1);
            if (kt + 1 < t_hi) step(kt + 1, ks1, vs1, ks0, vs0);
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
            if (qg == 0) *reinterpret_cast<float2 *>(a.part_ml + (p0 + r) * 2) = make_float2(m_run[j], l_run[j][0]);
            continue;
        }
        const float inv = 1.0f / (l_run[j][0] + 1e-6f);
        uint16_t   *op = a.out + row_of(rt * ROWS + r);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const __half2 lo = __floats2half2_rn(acc[j][dt][0] * inv, acc[j][dt][1] * inv);
            const __half2 hi = __floats2half2_rn(acc[j][dt][2] * inv, acc[j][dt][3] * inv);
            *reinterpret_cast<u32x2 *>(op + 16 * dt + 4 * qg) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
        }
    }
}

constexpr int kMergeThreads = 256;

// Workgroup (item that is a row tile's first, kv head; a few rows): D / 4 threads a row.
__global__ __launch_bounds__(kMergeThreads) void quant_prefill_merge_kernel(PrefillArgs a, int D, int ROWS) {
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    QUANT_ENTRY_OF(a, item, ei);
    const int nch = a.e[ei].nch, rel = item - a.e[ei].item0;
    if (nch == 1 || rel % nch != 0) return;
    const int per = D / 4, r = blockIdx.y * (kMergeThreads / per) + threadIdx.x / per, d = 4 * (threadIdx.x % per);
    const int rows = a.e[ei].nq << a.lgG, rt = (rows + ROWS - 1) / ROWS - 1 - rel / nch, qr = rt * ROWS + r;
    if (r >= ROWS || qr >= rows) return;
    const int64_t p0 = ((int64_t)item * a.Hkv + g) * ROWS + r, pc = (int64_t)a.Hkv * ROWS;
    float         m = kNone, l = 0.0f;
    for (int ch = 0; ch < nch; ++ch) m = fmaxf(m, a.part_ml[(p0 + ch * pc) * 2]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int ch = 0; ch < nch; ++ch) {
        const int64_t pr = p0 + ch * pc;
        const float2  ml = *reinterpret_cast<const float2 *>(a.part_ml + pr * 2);
        const float   wgt = __builtin_amdgcn_exp2f(ml.x - m);
        const f32x4   x = *reinterpret_cast<const f32x4 *>(a.part_o + pr * D + d);
        l = fmaf(wgt, ml.y, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(wgt, x[i], o[i]);
    }
    const float   inv = 1.0f / (l + 1e-6f);
    const __half2 lo = __floats2half2_rn(o[0] * inv, o[1] * inv), hi = __floats2half2_rn(o[2] * inv, o[3] * inv);
    uint16_t     *op = a.out + ((int64_t)(a.e[ei].tok0 + (qr >> a.lgG)) * a.Hq + (g << a.lgG) + (qr & ((1 << a.lgG) - 1))) * D + d;
    *reinterpret_cast<u32x2 *>(op) = u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

size_t part_ml_floats(size_t rows) { return (2 * rows + 3) / 4 * 4; }

template <int D, int NW> void launch_one(const PrefillArgs &a, int items, hipStream_t stream) {
    hipLaunchKernelGGL((quant_prefill_kernel<D, NW>), dim3((unsigned)items * (unsigned)a.Hkv), dim3(NW * 64), 0, stream, a);
}

} // namespace

size_t quant_prefill_workspace_floats(const QuantPrefillPlan &plan, int Hkv, int D) {
    size_t most = 0;
    for (const auto &l : plan.launches) {
        const size_t rows = (size_t)l.items * (size_t)quant_prefill_rows(D, plan.waves) * (size_t)Hkv;
        if (l.split) most = std::max(most, part_ml_floats(rows) + rows * (size_t)D);
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
    const int ROWS = quant_prefill_rows(c.D, plan.waves);
    for (const auto &l : plan.launches) {
        if (l.n == 0 || l.items == 0) continue;
        if ((int64_t)l.items * c.Hkv > kQuantMostItems) throw std::invalid_argument("attention: too many work items");
        a.n = l.n;
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(QuantPrefillEntry) * (size_t)l.n);
        a.part_ml = workspace;
        a.part_o = l.split ? workspace + part_ml_floats((size_t)l.items * (size_t)ROWS * (size_t)c.Hkv) : nullptr;
        profile_begin(KernelId::PrefillQuant, stream);
        for_head_dim(c.D, [&](auto d) {
            constexpr int D = decltype(d)::value;
            if constexpr (D <= 128) {
                if (plan.waves == 8) return launch_one<D, 8>(a, l.items, stream);
            }
            launch_one<D, 4>(a, l.items, stream);
        });
        HIP_CHECK(hipGetLastError());
        if (l.split) {
            const int rows = kMergeThreads / (c.D / 4);
            hipLaunchKernelGGL(quant_prefill_merge_kernel, dim3((unsigned)(l.items * c.Hkv), (unsigned)((ROWS + rows - 1) / rows)),
                               dim3(kMergeThreads), 0, stream, a, c.D, ROWS);
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::PrefillQuant, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
