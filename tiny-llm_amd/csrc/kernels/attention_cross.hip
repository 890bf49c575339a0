// Attention of many query rows to cached states of another length, for gfx950.
//
// Every query row (token x head of kv head g) of an entry attends to all S states:
//   o_r = (sum_t p_rt v_t) / (sum_t p_rt + 1e-6),  p_rt = 2^(s_rt - m_r),
//   s_rt = (q_r . k_t) * scale * log2(e)
// Bound by the matrix rate (4 S D operations a row).  The pieces are those of
// attn_prefill_kernel without its causal mask: a workgroup of 8 or 4 waves with 32
// (head_dim 256: 16) query rows each in registers; key tiles of 64 tokens through
// double-buffered LDS by the LDS DMA load, in XOR-swizzled 16-byte slots;
//   S^T = K Q^T      v_mfma_f32_16x16x32_f16: A = K rows, B = Q
//   online softmax   per query column, over a reference point 2^7 below the maximum,
//                    which moves on jumps above 2^15 only; p rounded to fp16 for the
//                    product, the normaliser sums the rounded ones (on the matrix
//                    unit, a row of ones)
//   O^T += V^T P^T   V^T by the transposing ds_read_b64_tr_b16, P^T as the S^T
//                    fragments stand
// The rounding of p, 2^-11 of a weight, is of the size of the output's own (2.9e-4 from
// 64 bits in the 2-norm, 2.1e-4 for fp32 weights).  As two fp16 numbers, as in
// attn_stream_kernel, p costs a second product where the matrix unit is the bound: 2 x 2048
// queries over 8192 670 us against 480, ragged prompts 39 against 30, so it has one.
// Row tiles that do not fill the chip have their keys split into chunks, whose
// (m, l, o) go through a workspace in fp32 to cross_merge_kernel.  Grid: kv head
// fastest, so that with 8 kv heads an XCD's workgroups share one head's keys in
// its L2.
//
// Measured: 2 x 2048 queries over 8192 states, 8 heads of 128, group 4: 492 us = 1.12
// PFLOP/s (an 8192^3 fp16 matrix product 1.2-1.34), matrix unit busy 47% of the
// cycles, VALU 21%; 16 x 64..448 over 300..1500, 16 heads of 64: 28 us; 8 over 32768, a
// quarter of a tile's rows in use: 30 us for the 134 MB of states, + 7 for the merge.
#include "cross.h"

#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <stdexcept>

namespace tiny_llm {
namespace detail {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef short    s16x4 __attribute__((ext_vector_type(4)));

constexpr float kBelow = 7.0f, kLazyMax = 15.0f; // of the softmax reference, as in attn_stream_kernel
constexpr float kNone = -3e38f; // ... over no score, or over -infinite ones only
constexpr int   kVmcnt0 = 0x0F70; // s_waitcnt vmcnt(0)
constexpr int   kTile = kStreamTile;

struct CrossArgs {
    const __half *q;
    __half       *out;
    float        *part_o;  // [item][Hkv][rows of a workgroup][D]
    float        *part_ml; // [item][Hkv][rows][2]
    KvView        kv;
    float         scale_log2; // positive
    int           negate;
    int           Hq, Hkv, lg, n; // lg: log2 of the query heads per kv head
    CrossEntry    e[kCrossBatch];
};
static_assert(sizeof(CrossArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ __attribute__((address_space(3))) s16x4 *lds_ptr(const uint16_t *p) {
    return (__attribute__((address_space(3))) s16x4 *)(p);
}

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

// The last entry whose first item is at most `item`.
#define CROSS_ENTRY_OF(a, item, out)                                                                                   \
    do {                                                                                                               \
        int seen_ = 0;                                                                                                 \
        for (int k_ = 0; k_ < (a).n; k_ += 64) {                                                                       \
            const int i_ = k_ + (int)(threadIdx.x & 63);                                                               \
            seen_ += __popcll(__ballot(i_ < (a).n && (a).e[min(i_, (a).n - 1)].item0 <= (item)));                      \
        }                                                                                                              \
        out = __builtin_amdgcn_readfirstlane(seen_ - 1);                                                               \
    } while (0)

template <int D, bool PAGED, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1))) void
attn_cross_kernel(CrossArgs a) {
    static_assert(NW == 4 || (NW == 8 && cross_wide(D)), "waves");
    constexpr int NQG = D <= 128 ? 2 : 1; // 16-row groups per wave
    constexpr int NT = NW * 64;
    constexpr int R = 16 * NQG;           // rows of a wave
    constexpr int ROWS = NW * R;
    static_assert(ROWS == cross_rows(D, NW), "the planner's row tile");
    constexpr int KS = D / 32, DT = D / 16, KP = D / 8;
    constexpr int PIECES = kTile * KP;
    constexpr int NKI = (PIECES + NT - 1) / NT;
    // Distinct arrays: the DMA into one does not alias the reads of another.
    __shared__ __align__(16) uint16_t ks0[kTile * D], ks1[kTile * D];
    __shared__ __align__(16) uint16_t vt0[kTile * D], vt1[kTile * D];
    auto swz = [](int r) {
        if constexpr (KP <= 4) return r & (KP - 1);
        const int f = ((r & 3) << 1) ^ (((r >> 2) & 1) * 9) ^ (((r >> 3) & 1) << 3);
        return f & (KP - 1);
    };
    auto slot = [&](int r, int x) { return r * KP + (x ^ swz(r)); };

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    CROSS_ENTRY_OF(a, item, ei);
    const int row = a.e[ei].row, S = a.e[ei].S, tok0 = a.e[ei].tok0, nch = a.e[ei].nch;
    const int rows = a.e[ei].nq << a.lg;
    const int rel = item - a.e[ei].item0, rt = rel / nch, ch = rel - rt * nch;
    const int tiles = (S + kTile - 1) / kTile;
    const int t_lo = (int)((int64_t)ch * tiles / nch), t_hi = (int)((int64_t)(ch + 1) * tiles / nch);
    const int c = lane & 15, qg = lane >> 4;
    const int vrow = 4 * qg + (c >> 2);
    const int vxor = ((c & 3) >> 1) ^ swz(vrow);
    const int vlane = vrow * KP * 8 + 4 * (c & 1);
    auto vt_read = [&](const uint16_t *vd, int r0, int dt) __attribute__((always_inline)) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr(&vd[vlane + ((2 * dt) ^ vxor) * 8 + r0 * KP * 8]));
    };
    auto row_of = [&](int r) -> int64_t { // element offset of query row r in q and out
        return ((int64_t)(tok0 + (r >> a.lg)) * a.Hq + (g << a.lg) + (r & ((1 << a.lg) - 1))) * D;
    };
    f16x8 qb[NQG][KS];
#pragma unroll
    for (int j = 0; j < NQG; ++j) {
        const __half *qp = a.q + row_of(min(rt * ROWS + wave * R + j * 16 + c, rows - 1));
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            // (a negative scale's sign goes into q: the maximum over s is then that over s * scale)
            const f16x8 v = *reinterpret_cast<const f16x8 *>(qp + 32 * s + 8 * qg);
            qb[j][s] = a.negate ? -v : v;
        }
    }

    const int64_t  head = (int64_t)g * a.kv.head_stride * 2;
    const char    *kb = reinterpret_cast<const char *>(a.kv.k_base) + head;
    const char    *vb = reinterpret_cast<const char *>(a.kv.v_base) + head;
    const int64_t  blk_bytes = a.kv.blk_stride * 2, tokb = a.kv.tok_stride * 2;
    const int32_t *bt = PAGED ? a.kv.block_table + (int64_t)row * a.kv.bt_stride : nullptr;
    // A wave's 64 pieces of a load lie in one quarter of 16 tokens, whose offset is
    // uniform: ids has the quarters' blocks in its first lanes (paged views), asked
    // for a tile ahead.
    auto blocks = [&](int kt) -> int {
        if constexpr (PAGED) return lane < 4 ? bt[min(kt * kTile + 16 * lane, S - 1) >> a.kv.log2_blk] : 0;
        else return 0;
    };
    int  ids = 0;
    auto issue_tile = [&](int kt, int now, uint16_t *kdst, uint16_t *vdst) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NKI; ++u) {
            const int sl = u * NT + tid;
            if (NKI * NT > PIECES && sl >= PIECES) break; // whole waves (PIECES % 64 == 0)
            const int r = sl / KP, x = (sl % KP) ^ swz(r);
            const int q = __builtin_amdgcn_readfirstlane((u * NT + wave * 64) / KP / 16); // the quarter
            const int tq = min(kt * kTile + 16 * q, S - 1), more = S - 1 - tq;
            int64_t   off;
            if constexpr (PAGED)
                off = (int64_t)__builtin_amdgcn_readlane(now, q) * blk_bytes + (int64_t)(tq & ((1 << a.kv.log2_blk) - 1)) * tokb;
            else off = (int64_t)row * blk_bytes + (int64_t)tq * tokb;
            const uint32_t lane_off = (uint32_t)min(r % 16, more) * (uint32_t)tokb + 16u * x;
            const int      lbase = (u * NT + wave * 64) * 8; // halves, wave-uniform
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(kb + off + lane_off),
                                             (__attribute__((address_space(3))) void *)(&kdst[lbase]), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(vb + off + lane_off),
                                             (__attribute__((address_space(3))) void *)(&vdst[lbase]), 16, 0, 0);
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
    const f16x8 ones = __builtin_bit_cast(f16x8, make_uint4(0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u));

    auto tile_step = [&](int kt, const uint16_t *kd, uint16_t *vd, uint16_t *kn, uint16_t *vn)
                         __attribute__((always_inline)) {
        if (kt + 1 < t_hi) {
            const int now = ids;
            if (PAGED && kt + 2 < t_hi) ids = blocks(kt + 2);
            issue_tile(kt + 1, now, kn, vn);
        }
        if ((kt + 1) * kTile > S) { // rows past the end, read as the last one: 0 times its value would be NaN where that is infinite
            for (int x = (S - kt * kTile) * KP + tid; x < kTile * KP; x += NT)
                *reinterpret_cast<uint4 *>(&vd[8 * x]) = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
        }
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
                for (int u = 0; u < 2; ++u)
                    kf[u] = *reinterpret_cast<const f16x8 *>(&kd[slot(16 * (th + u) + c, 4 * st + qg) * 8]);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < NQG; ++j)
                        s[j][th + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[u], qb[j][st], s[j][th + u], 0, 0, 0);
            }
        f16x8 pf[NQG][2];
        if ((kt + 1) * kTile > S) { // the last tile: keys past the end
            const int tb = kt * kTile + 4 * qg;
#pragma unroll
            for (int j = 0; j < NQG; ++j)
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (tb + 16 * tt + i >= S) s[j][tt][i] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < NQG; ++j) {
            float mloc = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mloc = fmaxf(mloc, s[j][tt][i]);
            if (__any(mloc * a.scale_log2 > m_run[j] + kLazyMax)) {
                const float m_tile = xor_lane_max<32>(xor_lane_max<16>(mloc)) * a.scale_log2;
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
                    pf[j][tt >> 1][4 * (tt & 1) + i] =
                        (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[j][tt][i], a.scale_log2, -m_new));
        }
#pragma unroll
        for (int tp = 0; tp < 2; ++tp) {
#pragma unroll
            for (int j = 0; j < NQG; ++j) l_run[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[j][tp], l_run[j], 0, 0, 0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint2 v0 = __builtin_bit_cast(uint2, vt_read(vd, 32 * tp, dt));
                const uint2 v1 = __builtin_bit_cast(uint2, vt_read(vd, 32 * tp + 16, dt));
                const f16x8 vf = __builtin_bit_cast(f16x8, make_uint4(v0.x, v0.y, v1.x, v1.y));
#pragma unroll
                for (int j = 0; j < NQG; ++j) acc[j][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[j][tp], acc[j][dt], 0, 0, 0);
            }
        }
        __builtin_amdgcn_s_waitcnt(kVmcnt0); // this wave's part of the next tile has landed
        __syncthreads();                      // ... every wave's, and this tile's buffer is free
    };
    issue_tile(t_lo, blocks(t_lo), ks0, vt0);
    if (PAGED && t_lo + 1 < t_hi) ids = blocks(t_lo + 1);
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    for (int kt = t_lo; kt < t_hi; kt += 2) {
        tile_step(kt, ks0, vt0, ks1, vt1);
        if (kt + 1 < t_hi) tile_step(kt + 1, ks1, vt1, ks0, vt0);
    }

    if (nch > 1) {
        const int64_t p0 = ((int64_t)item * a.Hkv + g) * ROWS;
#pragma unroll
        for (int j = 0; j < NQG; ++j) {
            const int r = wave * R + j * 16 + c;
            if (rt * ROWS + r >= rows) continue;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                *reinterpret_cast<f32x4 *>(a.part_o + (p0 + r) * D + 16 * dt + 4 * qg) = acc[j][dt];
            if (qg == 0) *reinterpret_cast<float2 *>(a.part_ml + (p0 + r) * 2) = make_float2(m_run[j], l_run[j][0]);
        }
        return;
    }
    // The wave's rows through LDS, so that every store is of whole rows: 8-wave
    // workgroups have a region for it, 4-wave ones (two per CU) a K/V buffer per wave.
    constexpr int  OP = D + 8;
    constexpr int  PPR = D / 8, NCH = R * PPR / 64;
    constexpr bool OWN = D <= 128 && NW == 8;
    __shared__ __align__(16) uint16_t own_stg[OWN ? NW * R * OP : 8];
    static_assert(OWN || R * OP <= kTile * D, "staging fits a K/V buffer");
    uint16_t *stg = OWN ? own_stg + wave * R * OP : (wave == 0 ? ks0 : (wave == 1 ? ks1 : (wave == 2 ? vt0 : vt1)));
#pragma unroll
    for (int j = 0; j < NQG; ++j) {
        const float inv = 1.0f / (l_run[j][0] + 1e-6f);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const __half2 lo = __floats2half2_rn(acc[j][dt][0] * inv, acc[j][dt][1] * inv);
            const __half2 hi = __floats2half2_rn(acc[j][dt][2] * inv, acc[j][dt][3] * inv);
            uint2         w;
            w.x = __builtin_bit_cast(uint32_t, lo);
            w.y = __builtin_bit_cast(uint32_t, hi);
            *reinterpret_cast<uint2 *>(&stg[(j * 16 + c) * OP + 16 * dt + 4 * qg]) = w;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
        const int k = u * 64 + lane, rr = k / PPR, pc = k - rr * PPR;
        const int r = rt * ROWS + wave * R + rr;
        if (r < rows)
            *reinterpret_cast<uint4 *>(a.out + row_of(r) + 8 * pc) = *reinterpret_cast<const uint4 *>(&stg[rr * OP + 8 * pc]);
    }
}

constexpr int kMergeThreads = 256;

// The chunks of the entries that have several.  A thread has four dims of a row and
// every groups-th chunk (groups: a power of two, up to what a workgroup holds of a
// row), their sums meet in LDS.  128 chunks of 32 rows x 8 heads, one thread for all
// chunks: 64 us, so: 7.
template <int ROWS> __global__ __launch_bounds__(kMergeThreads) void cross_merge_kernel(CrossArgs a, int D, int groups) {
    __shared__ f32x4 s_o[kMergeThreads];
    __shared__ float s_ml[kMergeThreads][2];
    const int ei = blockIdx.z, g = blockIdx.y;
    const int nch = a.e[ei].nch, rows = a.e[ei].nq << a.lg;
    const int per = D / 4, tid = threadIdx.x;
    const int grp = tid / per % groups, d = 4 * (tid % per);
    const int r = blockIdx.x * (kMergeThreads / (per * groups)) + tid / (per * groups);
    if (nch == 1 || (int)blockIdx.x * (kMergeThreads / (per * groups)) >= rows) return; // (the whole workgroup)
    const int     rc = min(r, rows - 1), rt = rc / ROWS;
    const int64_t p0 = ((int64_t)(a.e[ei].item0 + rt * nch) * a.Hkv + g) * ROWS + rc % ROWS, step = (int64_t)a.Hkv * ROWS;
    float         m = -INFINITY, l = 0.0f;
    f32x4         o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int ch = grp; ch < nch; ch += groups) m = fmaxf(m, a.part_ml[(p0 + ch * step) * 2]);
#pragma unroll 4
    for (int ch = grp; ch < nch; ch += groups) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + (p0 + ch * step) * 2);
        const float  w = __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(ml.y, w, l);
        o += w * *reinterpret_cast<const f32x4 *>(a.part_o + (p0 + ch * step) * D + d);
    }
    if (groups > 1) {
        s_o[tid] = o;
        s_ml[tid][0] = m;
        s_ml[tid][1] = l;
        __syncthreads();
        if (grp > 0) return;
        float mx = m;
        for (int k = 1; k < groups; ++k) mx = fmaxf(mx, s_ml[tid + k * per][0]);
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        l = 0.0f;
        for (int k = 0; k < groups; ++k) {
            const float w = __builtin_amdgcn_exp2f(s_ml[tid + k * per][0] - mx); // (0 for a group without chunks)
            l = fmaf(s_ml[tid + k * per][1], w, l);
            o += w * s_o[tid + k * per];
        }
    }
    if (r >= rows) return;
    const float   inv = 1.0f / (l + 1e-6f);
    const __half2 lo = __floats2half2_rn(o[0] * inv, o[1] * inv), hi = __floats2half2_rn(o[2] * inv, o[3] * inv);
    uint2         w;
    w.x = __builtin_bit_cast(uint32_t, lo);
    w.y = __builtin_bit_cast(uint32_t, hi);
    *reinterpret_cast<uint2 *>(a.out + ((int64_t)(a.e[ei].tok0 + (r >> a.lg)) * a.Hq + (g << a.lg) + (r & ((1 << a.lg) - 1))) * D + d) = w;
}

constexpr int kZeroRanges = 256, kZeroThreads = 256;
struct ZeroArgs {
    __half *out;
    int     row, n;
    int2    range[kZeroRanges]; // first token, tokens
};

// Workgroups (x, range): 16 bytes a lane and step.
__global__ __launch_bounds__(kZeroThreads) void cross_zero_kernel(ZeroArgs a) {
    const int2    r = a.range[blockIdx.y];
    const int64_t pieces = (int64_t)r.y * a.row / 8;
    uint4        *out = reinterpret_cast<uint4 *>(a.out + (int64_t)r.x * a.row);
    for (int64_t i = (int64_t)blockIdx.x * kZeroThreads + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * kZeroThreads)
        out[i] = make_uint4(0u, 0u, 0u, 0u);
}

template <int D, int NW> void launch_dw(const CrossArgs &a, int items, bool paged, hipStream_t stream) {
    const dim3 grid((unsigned)items * (unsigned)a.Hkv), block(NW * 64);
    if (paged) hipLaunchKernelGGL((attn_cross_kernel<D, true, NW>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((attn_cross_kernel<D, false, NW>), grid, block, 0, stream, a);
}
template <int D> void launch_d(const CrossArgs &a, int items, bool paged, int waves, hipStream_t stream) {
    if constexpr (cross_wide(D)) {
        if (waves == 8) {
            launch_dw<D, 8>(a, items, paged, stream);
            return;
        }
    }
    launch_dw<D, 4>(a, items, paged, stream);
}

} // namespace

size_t cross_workspace_floats(const CrossPlan &plan, int Hkv, int D) {
    size_t most = 0;
    for (const auto &l : plan.launches)
        if (l.split) most = std::max(most, (size_t)l.items * Hkv * cross_rows(D, plan.waves) * (D + 2));
    return most;
}

void launch_attn_cross(const CrossCall &c, const KvView &kv, const CrossPlan &plan, float *workspace,
                       hipStream_t stream) {
    CrossArgs a;
    a.q = c.q;
    a.out = c.out;
    a.kv = kv;
    // (0: so small that every score is 0 beside a masked one's -infinity)
    a.scale_log2 = c.scale == 0.0f ? 1e-37f : std::fabs(c.scale) * 1.4426950408889634f;
    a.negate = c.scale < 0.0f;
    a.Hq = c.Hq;
    a.Hkv = c.Hkv;
    a.lg = __builtin_ctz((unsigned)(c.Hq / c.Hkv));
    const bool paged = kv.block_table != nullptr;
    const int  tile = cross_rows(c.D, plan.waves);
    for (const auto &l : plan.launches) {
        if (l.items == 0) continue;
        a.n = l.n;
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(CrossEntry) * (size_t)l.n);
        a.part_ml = workspace;
        a.part_o = workspace + (size_t)l.items * c.Hkv * tile * 2;
        profile_begin(KernelId::AttnCross, stream);
        switch (c.D) {
        case 32: launch_d<32>(a, l.items, paged, plan.waves, stream); break;
        case 64: launch_d<64>(a, l.items, paged, plan.waves, stream); break;
        case 128: launch_d<128>(a, l.items, paged, plan.waves, stream); break;
        case 256: launch_d<256>(a, l.items, paged, plan.waves, stream); break;
        default: throw std::invalid_argument("attention: unsupported head_dim");
        }
        HIP_CHECK(hipGetLastError());
        if (l.split) {
            int64_t rows = 0;
            int     chunks = 1, groups = 1;
            for (int i = l.first; i < l.first + l.n; ++i) {
                const CrossEntry &e = plan.entries[(size_t)i];
                chunks = std::max(chunks, (int)e.nch);
                if (e.nch > 1) rows = std::max(rows, (int64_t)e.nq << a.lg);
            }
            while (2 * groups <= chunks && 2 * groups * (c.D / 4) <= kMergeThreads) groups *= 2;
            const int  per_block = kMergeThreads / (groups * (c.D / 4)); // rows
            const dim3 grid((unsigned)((rows + per_block - 1) / per_block), (unsigned)c.Hkv, (unsigned)l.n);
            switch (tile) {
            case 64: hipLaunchKernelGGL((cross_merge_kernel<64>), grid, dim3(kMergeThreads), 0, stream, a, c.D, groups); break;
            case 128: hipLaunchKernelGGL((cross_merge_kernel<128>), grid, dim3(kMergeThreads), 0, stream, a, c.D, groups); break;
            default: hipLaunchKernelGGL((cross_merge_kernel<256>), grid, dim3(kMergeThreads), 0, stream, a, c.D, groups); break;
            }
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::AttnCross, stream);
    }
}

void launch_cross_zeros(__half *out, int row, const std::vector<std::pair<int32_t, int32_t>> &ranges, hipStream_t stream) {
    ZeroArgs a;
    a.out = out;
    a.row = row;
    for (size_t i = 0; i < ranges.size();) {
        int32_t most = 0;
        for (a.n = 0; i < ranges.size() && a.n < kZeroRanges; ++i, ++a.n) {
            a.range[a.n] = make_int2(ranges[i].first, ranges[i].second);
            most = std::max(most, ranges[i].second);
        }
        const int64_t blocks = ((int64_t)most * row / 8 + 4 * kZeroThreads - 1) / (4 * kZeroThreads);
        profile_begin(KernelId::AttnCross, stream);
        hipLaunchKernelGGL(cross_zero_kernel, dim3((unsigned)std::min<int64_t>(blocks, 4096), (unsigned)a.n), dim3(kZeroThreads),
                           0, stream, a);
        HIP_CHECK(hipGetLastError());
        profile_end(KernelId::AttnCross, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
