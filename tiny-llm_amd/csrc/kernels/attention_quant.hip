// Attention of a few query rows over a cache in 8 bits (layout: quant.h), read once, for
// gfx950: decode steps, and up to 16 rows (tokens x query heads of a kv head) of a prompt.
//
//   s_rt = (q_r . K_t) scale ks,   P_rt = exp(s_rt - max_t s_rt) / sum_t exp(...)
//   o_r  = sum_groups vs sum_t P_rt V_t       (sum + 1e-6 in the denominator, as in decode)
// K_t, V_t: the stored whole numbers, ks, vs: the scales of t's group.  Bound by HBM: 2 D
// bytes a token and kv head.
//
// A workgroup of NW waves (8, 4 at head_dim 256, 2 for many short entries) per (entry, chunk of tiles of 64
// tokens, kv head); wave w takes every NW-th tile (half a tile at a time at head_dim 256) and keeps its own running
// maximum, sum and output; the next tile is on its way while one is computed.  Tiles lie in
// memory as the operands that the matrix instructions take, so nothing passes through LDS:
//   S^T = K Q^T      v_mfma_f32_16x16x32_f16: A = K (token l%16, dims 8(l/16)..+7),
//                    B = Q (row l%16), D = S^T (tokens 4(l/16)+i, row l%16)
//   O^T += vs V^T P^T  A = V^T (dim l%16, the group's tokens that the lane has weights of),
//                    B = the weights as they came out, their upper and then their lower half in
//                    fp16 (22 bits); a group's product is scaled in fp32
// Whole numbers up to 127 are exact in fp16, so the scales are all that rounds them.  The weights' lower halves
// are a second product of the matrix units, which wait for HBM as it is: 64 x 8192 169.4 us with them, 166.8
// without, 131072 alone 51.3 and 50.6, and without them outputs are 2.9e-4 off, of which their own rounding is 2.1e-4.
// The open group (fp16, at most 31 tokens), and the one that the call's token closes, is a step of its
// own of one wave, the one with the fewest others.
// Measured, 8 kv heads of 128: 64 x 8192 tokens, groups of 4, 163-182 us by clock, a call 169, 6.4 TB/s (counters: 1.08 GB
// read, the cache's own size); 96 ragged ones of 8, 11 million tokens times heads in all 110-119 us and 5 us for the join;
// 1 x 131072 42-45 and 5; four sequences of 8 x 64 6.6 us, of which the launch is most.  What did not
// help: loads that stay in the caches (187 us for 175), one group a step, tiles in another order per workgroup,
// more workgroups a CU.
#include "quant_device.h"

#include "../runtime.h"
#include "kv_kernels.h"
#include "tiny_llm/hip_utils.h"

#include <algorithm>
#include <climits>
#include <cstring>
#include <mutex>

namespace tiny_llm {
namespace detail {

namespace {

using namespace quant;

// Weights are 2^(s - ref): the reference is 2^7 below the maximum when it moves, and moves on
// scores 2^15 above it only (below 2^15 in fp16, and 2^-31 of the largest still counts).
constexpr float kBelow = 7.0f, kLazyMax = 15.0f;
// The reference over no score, or over -infinite ones only: finite, and below every finite score.
constexpr float kNone = -3e38f;

struct QuantArgs {
    const uint16_t *q;
    uint16_t       *out;
    const uint16_t *new_k, *new_v;
    float          *part_o;  // [item][Hkv][rows][D]
    float          *part_ml; // [item][Hkv][rows][2]
    QuantView       v;
    float           scale_log2;
    int             Hq, Hkv, G, n, items, chunk, rows;
    int             each; // work items of every entry, 0: they differ
    QuantEntry      e[kQuantBatch];
};
static_assert(sizeof(QuantArgs) <= 4096, "kernel arguments");

template <int D, int NW>
__global__ __launch_bounds__(NW * 64, D <= 128 ? 2 : 1) void attn_quant_kernel(QuantArgs a) {
    constexpr int NG = D <= 128 ? 2 : 1;  // groups of a step
    constexpr int SUB = 2 / NG;           // steps per tile
    constexpr int KS = D / 32, DT = D / 16;
    constexpr int NT = NW * 64;
    extern __shared__ __align__(16) float so[]; // the waves' outputs [NW][rows][D]
    __shared__ float    sm[NW][16], sl[NW][16], s_l[16];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int       item, g;
    quant_place(blockIdx.x, a.Hkv, item, g);
    if (item >= a.items) return;
    int ei = a.each ? item / a.each : 0;
    if (!a.each) QUANT_ENTRY_OF(a, item, ei);
    const int row = a.e[ei].row, S = a.e[ei].S, tok0 = a.e[ei].tok0, nq = a.e[ei].nq, rows = nq * a.G;
    const int tiles = (S + kQuantTile - 1) / kQuantTile;
    const int nch = (tiles + a.chunk - 1) / a.chunk, ch = item - a.e[ei].item0;
    const int tile_lo = (int)((int64_t)ch * tiles / nch), tile_hi = (int)((int64_t)(ch + 1) * tiles / nch);
    const int open = S % kGroup == 0 ? -1 : a.e[ei].open; // (-1: the last token closes its group)
    const int last = (S - 1) / kGroup * kGroup;           // first token of the last group
    // The last group is a step of its own where it is open, and where this launch appends to it, by
    // the wave that has the fewest others.
    const bool apart = a.new_k || open >= 0;
    const int  closed = apart ? last : S;               // tokens of the other steps,
    const int  groups = (closed + kGroup - 1) / kGroup; // all in 8 bits
    const int  end = min(tile_hi, (groups + 1) / 2);
    const bool ends = apart && ch == nch - 1 && wave == max(0, end - tile_lo) % NW;

    const int c = lane & 15, qg = lane >> 4;
    f16x8     qb[KS]; // B operand: row c, dims 32s + 8qg .. +7
    {
        const int       r = min(c, rows - 1);
        const uint16_t *qp = a.q + ((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const f16x8 *>(qp + 32 * s + 8 * qg);
    }
    const int all = S - nq + 1;                         // tokens that every row sees
    const int lim = min(S, all + min(c, rows - 1) / a.G); // that row c sees
    f32x4     acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kNone, l_run = 0.0f;
    auto  raise = [&](float mloc) __attribute__((always_inline)) { // the reference, where a score is far above it
        if (__any(mloc > m_run + kLazyMax)) {
            mloc = fmaxf(mloc, __shfl_xor(mloc, 16));
            mloc = fmaxf(mloc, __shfl_xor(mloc, 32));
            const float m_new = fmaxf(m_run, mloc - kBelow);
            const float alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
            l_run *= alpha;
            m_run = m_new;
        }
    };
    auto weigh = [&](float score, f16x8 &hi, f16x8 &lo, int at) __attribute__((always_inline)) { // the weight's 22 bits
        const float p = __builtin_amdgcn_exp2f(score - m_run);
        l_run += p;
        hi[at] = (_Float16)p;
        lo[at] = (_Float16)(p - (float)hi[at]);
    };
    auto times_weights = [](f16x8 v, f16x8 hi, f16x8 lo) __attribute__((always_inline)) {
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi, __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo, zero, 0, 0, 0), 0, 0, 0);
    };

    // The wave's steps: step x is half (all) of tile tile_lo + x / SUB * NW + wave.
    const int steps = max(0, (end - tile_lo - wave + NW - 1) / NW) * SUB;
    auto      first_group = [&](int x) { return (tile_lo + x / SUB * NW + wave) * 2 + x % SUB * NG; };
    const int32_t *bt = a.v.table + (int64_t)row * a.v.bt_stride;
    // Blocks of a step's groups, lane k that of group k; asked for a step before the tiles.  (Neither
    // these loads nor the tiles' are conditional: the compiler waits by counting the
    // loads on their way, and behind a branch it waits for all of them.)
    auto blocks = [&](int x) -> int { return bt[min(first_group(min(x, steps - 1)) + min(lane, NG - 1), groups - 1) >> a.v.lg]; };
    auto tile_at = [&](int x, int k, int ids) __attribute__((always_inline)) -> int64_t {
        const int i = min(first_group(x) + k, groups - 1) & ((1 << a.v.lg) - 1);
        return (((int64_t)__builtin_amdgcn_readlane(ids, k) * a.Hkv + g) << a.v.lg) + i;
    };
    u32x4  kr[NG][KS], vr[NG][DT / 2];
    float2 sc[NG];
    auto   load_k = [&](int x, int ids) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const int64_t at = tile_at(x, k, ids);
            const u32x4  *p = reinterpret_cast<const u32x4 *>(a.v.tiles + at * (64 * D)) + lane;
#pragma unroll
            for (int s = 0; s < KS; ++s) kr[k][s] = __builtin_nontemporal_load(p + 64 * s);
            sc[k] = a.v.scales[at];
        }
    };
    auto load_v = [&](int x, int ids) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const u32x4 *p = reinterpret_cast<const u32x4 *>(a.v.tiles + tile_at(x, k, ids) * (64 * D) + 32 * D) + lane;
#pragma unroll
            for (int s = 0; s < DT / 2; ++s) vr[k][s] = __builtin_nontemporal_load(p + 64 * s);
        }
    };

    int  ids = 0, next = 0;
    auto step = [&](int x, auto more) __attribute__((always_inline)) {
        const int g0 = first_group(x), t0 = g0 * kGroup;
        if constexpr (more) {
            ids = next;
            next = blocks(x + 2);
        }
        // The scales in scalar registers, before the next ones' loads.
        float ks[NG], vs[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            ks[k] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(sc[k].x)));
            vs[k] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(sc[k].y)));
        }
        f32x4 s[NG][2];
#pragma unroll
        for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                s[k][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    s[k][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(whole8(kr[k][i][2 * tt], kr[k][i][2 * tt + 1]), qb[i], s[k][tt], 0, 0, 0);
            }
        if constexpr (more) load_k(x + 1, ids);
        float mloc = -INFINITY;
        const bool masked = t0 + NG * kGroup > min(all, closed); // some score does not count
        const int  bound = min(lim, closed);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            const float f = ks[k] * a.scale_log2;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = s[k][tt][i] * f;
                    s[k][tt][i] = !masked || t0 + 32 * k + 16 * tt + 4 * qg + i < bound ? y : -INFINITY;
                    mloc = fmaxf(mloc, s[k][tt][i]);
                }
        }
        raise(mloc);
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            f16x8 hi, lo;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) weigh(s[k][tt][i], hi, lo, 4 * tt + i);
            // (a group whose scale is NaN is none of the rows' business that see none of it)
            const float by = t0 + 32 * k < bound ? vs[k] : 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const u32x4 w = vr[k][dt / 2];
                const f32x4 o = times_weights(whole8(w[2 * (dt & 1)], w[2 * (dt & 1) + 1]), hi, lo);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[dt][i] = fmaf(by, o[i], acc[dt][i]);
            }
        }
        if constexpr (more) load_v(x + 1, ids);
    };
    GroupRegs<D> group;
    if (ends) {
        const int64_t src = ((int64_t)tok0 * a.Hkv + g) * D;
        if (a.new_k) group.fetch(S - 1 - last, a.new_k + src, a.new_v + src);
        group.load(open_of<D>(a.v, a.Hkv, row, a.e[ei].open, g));
    }
    if (steps > 0) {
        ids = blocks(0);
        next = blocks(1);
        load_k(0, ids);
        load_v(0, ids);
    }
    if (ends) { // (while the first tile is on its way)
        const int cnt = S - last;
        if (a.new_k) {
            group.append(open_of<D>(a.v, a.Hkv, row, a.e[ei].open, g), cnt - 1);
            if (open < 0) {
                const int64_t at = tile_of(a.v, a.Hkv, row, g, last / kGroup);
                group.close(a.v.tiles + at * (64 * D), a.v.scales + at);
            }
        }
        f32x4 s[2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KS; ++i) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(group.kf[tt][i], qb[i], s[tt], 0, 0, 0);
        }
        float       mloc = -INFINITY;
        const float f = group.ks * a.scale_log2;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y = s[tt][i] * f;
                s[tt][i] = last + 16 * tt + 4 * qg + i < lim ? y : -INFINITY;
                mloc = fmaxf(mloc, s[tt][i]);
            }
        raise(mloc);
        f16x8 hi, lo;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) weigh(s[tt][i], hi, lo, 4 * tt + i);
        // Values of tokens behind the last are whatever the tile held: 0 times them could be
        // NaN.  The same goes for infinite values that only some of the rows see.
        bool odd = false;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f16x8 v = group.vf[dt];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool there = 16 * (j >> 2) + 4 * qg + (j & 3) < cnt;
                const bool finite = __builtin_fabsf16(v[j]) <= (_Float16)65504.0f;
                odd |= there && !finite;
                if (!there || !finite) v[j] = (_Float16)0.0f;
            }
            const f32x4 o = times_weights(v, hi, lo);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[dt][i] = fmaf(group.vs, o[i], acc[dt][i]);
        }
        if (__any(odd)) { // (of an open group: stored numbers are finite)
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const uint16_t *tile = open_of<D>(a.v, a.Hkv, row, a.e[ei].open, g) + 32 * D;
            for (int r = 0; r < cnt; ++r)
                if (last + r < lim)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = (float)__builtin_bit_cast(_Float16, tile[v_half(r, 16 * dt + 4 * qg + i)]);
                            if (!(__builtin_fabsf(x) <= 65504.0f)) acc[dt][i] += x;
                        }
        }
    }
    if (steps > 0) {
        for (int x = 0; x < steps - 1; ++x) step(x, std::true_type());
        step(steps - 1, std::false_type());
    }

    // The waves' (m, l, o) through LDS.
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    if (c < rows)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4 *>(so + ((wave * a.rows + c) * D + 16 * dt + 4 * qg)) = acc[dt];
    if (qg == 0) {
        sm[wave][c] = m_run;
        sl[wave][c] = l_run;
    }
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        const int r = threadIdx.x;
        float     m = sm[0][r], l = 0.0f;
#pragma unroll
        for (int w = 1; w < NW; ++w) m = fmaxf(m, sm[w][r]);
#pragma unroll
        for (int w = 0; w < NW; ++w) { // sm: the waves' weights
            const float wgt = __builtin_amdgcn_exp2f(sm[w][r] - m);
            l = fmaf(wgt, sl[w][r], l);
            sm[w][r] = wgt;
        }
        s_l[r] = l;
        if (nch > 1)
            *reinterpret_cast<float2 *>(a.part_ml + (((int64_t)item * a.Hkv + g) * a.rows + r) * 2) = make_float2(m, l);
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < rows * (D / 4); idx += NT) {
        const int r = idx / (D / 4), d = 4 * (idx - r * (D / 4));
        f32x4     o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(so + (w * a.rows + r) * D + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(sm[w][r], x[i], o[i]);
        }
        if (nch == 1) {
            const float   inv = 1.0f / (s_l[r] + 1e-6f);
            const __half2 lo = __floats2half2_rn(o[0] * inv, o[1] * inv), hi = __floats2half2_rn(o[2] * inv, o[3] * inv);
            *reinterpret_cast<u32x2 *>(a.out + ((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D + d) =
                u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
        } else {
            *reinterpret_cast<f32x4 *>(a.part_o + (((int64_t)item * a.Hkv + g) * a.rows + r) * D + d) = o;
        }
    }
}

constexpr int kFinishThreads = 256;

// Entries of several chunks, or of no tokens (zeros).  Workgroup (entry, kv head; a few rows):
// every thread joins a few chunks' maxima, sums and outputs of four dims of a row, all on their
// way at once, then the row's `split` threads of equal dims meet in LDS.
constexpr int kFinishChunks = 4; // on their way at once
__global__ __launch_bounds__(kFinishThreads) void quant_finish_kernel(QuantArgs a, int D, int split) {
    __shared__ f32x4  s_o[kFinishThreads];
    __shared__ float2 s_ml[kFinishThreads];
    const int ei = blockIdx.x / a.Hkv, g = blockIdx.x - ei * a.Hkv;
    const int per = D / 4, grp = threadIdx.x / per, d = 4 * (threadIdx.x % per), part = grp % split;
    const int r = blockIdx.y * (kFinishThreads / per / split) + grp / split;
    const int S = a.e[ei].S, tok0 = a.e[ei].tok0, rows = a.e[ei].nq * a.G;
    const int tiles = (S + kQuantTile - 1) / kQuantTile, nch = (tiles + a.chunk - 1) / a.chunk;
    if (nch == 1) return;
    const int64_t p0 = ((int64_t)a.e[ei].item0 * a.Hkv + g) * a.rows + r; // of chunk 0
    const int64_t pc = (int64_t)a.Hkv * a.rows;                          // from chunk to chunk
    constexpr int U = kFinishChunks;
    float         m = kNone, l = 0.0f;
    f32x4         o = {0.0f, 0.0f, 0.0f, 0.0f};
    auto          join = [&](float m2, float l2, f32x4 o2) {
        const float mn = fmaxf(m, m2), x = __builtin_amdgcn_exp2f(m - mn), y = __builtin_amdgcn_exp2f(m2 - mn);
        l = l * x + l2 * y;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * x + o2[i] * y;
        m = mn;
    };
    for (int c0 = r < rows ? part : nch; c0 < nch; c0 += split * U) {
        float2 ml[U];
        f32x4  po[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t pr = p0 + min(c0 + u * split, nch - 1) * pc;
            ml[u] = *reinterpret_cast<const float2 *>(a.part_ml + pr * 2);
            po[u] = *reinterpret_cast<const f32x4 *>(a.part_o + pr * D + d);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c0 + u * split < nch) join(ml[u].x, ml[u].y, po[u]);
    }
    s_o[threadIdx.x] = o;
    s_ml[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (part == 0 && r < rows) {
        for (int k = 1; k < split; ++k) {
            const float2 ml = s_ml[threadIdx.x + k * per];
            join(ml.x, ml.y, s_o[threadIdx.x + k * per]);
        }
        const float   inv = nch ? 1.0f / (l + 1e-6f) : 0.0f;
        const __half2 lo = __floats2half2_rn(o[0] * inv, o[1] * inv), hi = __floats2half2_rn(o[2] * inv, o[3] * inv);
        *reinterpret_cast<u32x2 *>(a.out + ((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D + d) =
            u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
    }
}

// Floats of the partial maxima and sums, then the outputs at a multiple of 16 bytes.
size_t part_ml_floats(size_t rows) { return (2 * rows + 3) / 4 * 4; }

template <int D, int NW> void launch_one(const QuantArgs &a, int items, hipStream_t stream) {
    auto                 *fn = attn_quant_kernel<D, NW>;
    static std::once_flag once[64]; // per device
    std::call_once(once[current_device() & 63], [&] {
        HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      NW * kQuantRows * D * 4));
    });
    hipLaunchKernelGGL(fn, dim3((unsigned)quant_grid(items, a.Hkv)), dim3(NW * 64), (size_t)(NW * a.rows * D * 4), stream, a);
}

} // namespace

size_t quant_workspace_floats(const QuantPlan &plan, int Hkv, int D) {
    size_t most = 0;
    for (const auto &l : plan.launches) {
        const size_t rows = (size_t)l.items * (size_t)l.rows * (size_t)Hkv;
        if (l.finish) most = std::max(most, part_ml_floats(rows) + rows * (size_t)D);
    }
    return most;
}

void launch_attn_quant(const QuantCall &c, const QuantView &v, const QuantPlan &plan, float *workspace, hipStream_t stream) {
    QuantArgs a{};
    a.q = reinterpret_cast<const uint16_t *>(c.q);
    a.out = reinterpret_cast<uint16_t *>(c.out);
    a.new_k = reinterpret_cast<const uint16_t *>(c.new_k);
    a.new_v = reinterpret_cast<const uint16_t *>(c.new_v);
    a.v = v;
    a.scale_log2 = c.scale * 1.4426950408889634f;
    a.Hq = c.Hq;
    a.Hkv = c.Hkv;
    a.G = c.Hq / c.Hkv;
    a.chunk = plan.chunk;
    for (const auto &l : plan.launches) {
        if (l.n == 0) continue;
        a.n = l.n;
        a.items = l.items;
        a.rows = l.rows;
        if (a.rows > kQuantRows) throw std::invalid_argument("attention: too many query rows per entry");
        if (quant_grid(l.items, c.Hkv) > kQuantMostItems) throw std::invalid_argument("attention: too many work items");
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(QuantEntry) * (size_t)l.n);
        a.each = quant_items(a.e[0].S, plan.chunk);
        for (int i = 1; i < l.n; ++i)
            if (quant_items(a.e[i].S, plan.chunk) != a.each) a.each = 0;
        a.part_ml = workspace;
        a.part_o = l.finish ? workspace + part_ml_floats((size_t)l.items * c.Hkv * a.rows) : nullptr;
        profile_begin(KernelId::AttnQuant, stream);
        if (l.items > 0) {
            for_head_dim(c.D, [&](auto d) {
                constexpr int D = decltype(d)::value;
                if (plan.small) launch_one<D, kQuantSmallWaves>(a, l.items, stream);
                else launch_one<D, quant_waves(D)>(a, l.items, stream);
            });
            HIP_CHECK(hipGetLastError());
        }
        if (l.finish) {
            int       most = 1, split = 1;
            const int groups = kFinishThreads / (c.D / 4);
            for (int i = 0; i < l.n; ++i) most = std::max(most, quant_items(a.e[i].S, plan.chunk));
            while (split < groups && split * kFinishChunks < most) split *= 2;
            const int rows = groups / split;
            hipLaunchKernelGGL(quant_finish_kernel, dim3((unsigned)(l.n * c.Hkv), (unsigned)((a.rows + rows - 1) / rows)),
                               dim3(kFinishThreads), 0, stream, a, c.D, split);
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::AttnQuant, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
