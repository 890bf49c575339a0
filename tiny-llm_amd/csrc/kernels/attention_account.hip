// The account of a prompt's attention weights over a KV view, for gfx950.
//
// For every cached token t of a sequence and kv head g, over the last w of its new
// tokens j and the query heads h of g, causal (token j attends to t <= p0 + j):
//   account_out[t] = (t < p0 ? account_in[t] : 0) + sum_{h, j} P_hj(t),
//   P_hj(t) = exp(s_hjt - m_hj) / l_hj,  s = (q . k) * scale
// A column sum of a softmax over rows: a weight needs its row's maximum and sum
// over all keys first, so q . k is computed twice.  Bound by the matrix and
// exponential rates for many rows, by K's bytes for few.  Scores, sums and
// weights are fp32 throughout.
//
// account_stats_kernel: every row's maximum m and the inverse of its sum l, so that a weight
// is a multiply-add, an exponential and a multiply-add, 2^(s * scale * log2(e) - m) / l.  (In
// one number, m + log2 l, its rounding would enter the weights, 2^-24 |m| of each.)  A workgroup
// has 128 rows, 32 per wave in registers, and a chunk of the keys, whose tiles of 64
// pass through LDS (DMA, two buffers).  S^T = K Q^T on v_mfma_f32_16x16x32_f16 as in
// the prefill kernel: a lane has 16 keys of its row column per tile, and a running
// maximum of its own.
// account_sum_kernel: a workgroup has 256 keys, 64 per wave in registers, and passes
// a chunk of the rows that see them through LDS, 64 at a time (DMA, two buffers); a
// lane adds its row column's weights to 16 keys' sums, and the 16 columns are added
// at the end.
// account_merge_kernel joins the rows' chunks of keys where rows are few (very few:
// account_sum_kernel does so itself while its keys are on their way, a launch less),
// account_join_kernel adds the keys' chunks of rows.  No atomics: every sum has one
// order.
//
// Measured, 8 kv heads of 128, group 4: 4 x 1700..2048 new tokens on prefixes to 600,
// 125 us for the statistics (matrix unit busy 28% of the cycles, VALU 45%) and 119 for
// the sums (30%, 26%), no bank conflicts: the phases of a step follow each other, and
// the registers leave room for two to four waves a SIMD to fill the gaps.  The last 32
// tokens of 8192: 9 + 14 us, two launches' latency and K's 17 MB each.  (A row in one
// number: 217 and 22.0 us the two calls, in two 220 and 22.3.)
#include "account.h"

#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <stdexcept>
#include <type_traits>

namespace tiny_llm {
namespace detail {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));

constexpr int   kThreads = 256;
constexpr int   kVmcnt0 = 0x0F70; // s_waitcnt vmcnt(0)
constexpr int   kTile = kStreamTile;
constexpr float kNone = -1e30f;  // a maximum over no score

struct AccountArgs {
    const __half *q;
    const float  *w_in;
    float        *w_out;
    float        *rows;  // (m, 1 / l) [lse0 * Hkv + g * rows + r]
    float        *stats; // (m, l) [stat0 * Hkv + (chunk * Hkv + g) * rows + r]
    float        *parts; // [part0 * Hkv + (chunk * Hkv + g) * blocks * 256 + t]
    KvView        kv;
    int64_t       room;
    float         scale_log2;
    int           Hq, Hkv, lg, n; // lg: log2 of the query heads per kv head
    int           fold;           // no account_merge_kernel ran
    int           nt, nb;         // pieces of row tiles, of key blocks
    AccountPiece  tiles[kAccountPieces], blocks[kAccountPieces];
    AccountEntry  e[kAccountBatch];
};
static_assert(sizeof(AccountArgs) <= 4096, "kernel arguments");

// A launch's pieces, one per lane, so that a look-up is a ballot and lane reads
// instead of a chain of loads (2 to 7 us a call of few rows).
struct Pieces {
    AccountPiece p;
    int          n;
    __device__ __forceinline__ Pieces(const AccountPiece *all, int count) : n(count) {
        static_assert(kAccountPieces <= 64, "a lane per piece");
        p = all[min((int)(threadIdx.x & 63), count - 1)];
    }
    // The piece of work item `item`: the last whose first item is at most that.
    __device__ __forceinline__ AccountPiece of_item(int item) const {
        return at(__popcll(__ballot((int)(threadIdx.x & 63) < n && p.item0 <= item)) - 1);
    }
    // Chunks of tile (block) x, the same for the whole wave, of entry ei.
    __device__ __forceinline__ int chunks(int ei, int x) const {
        const uint64_t hit = __ballot((int)(p.what & 255u) == ei && p.first <= x && x < p.last);
        return (int)((uint32_t)__builtin_amdgcn_readlane((int)p.what, __ffsll((unsigned long long)hit) - 1) >> 8);
    }
    __device__ __forceinline__ AccountPiece at(int i) const {
        i = __builtin_amdgcn_readfirstlane(i);
        AccountPiece c;
        c.item0 = __builtin_amdgcn_readlane(p.item0, i);
        c.first = __builtin_amdgcn_readlane(p.first, i);
        c.last = __builtin_amdgcn_readlane(p.last, i);
        c.what = (uint32_t)__builtin_amdgcn_readlane((int)p.what, i);
        return c;
    }
};

// Byte offset of token t's row in a kv head's K.
template <bool PAGED> __device__ __forceinline__ int64_t key_off(const KvView &v, int row, int t) {
    if constexpr (PAGED) {
        const int blk = v.block_table[(int64_t)row * v.bt_stride + (t >> v.log2_blk)];
        return ((int64_t)blk * v.blk_stride + (int64_t)(t & ((1 << v.log2_blk) - 1)) * v.tok_stride) * 2;
    }
    return ((int64_t)row * v.blk_stride + (int64_t)t * v.tok_stride) * 2;
}

// 16-byte piece x of LDS row r at slot x ^ swz(r): 8 or 16 rows' same piece on
// distinct banks.
template <int KP> __device__ __forceinline__ int swz(int r) {
    if constexpr (KP <= 4) return r & (KP - 1);
    const int f = ((r & 3) << 1) ^ (((r >> 2) & 1) * 9) ^ (((r >> 3) & 1) << 3);
    return f & (KP - 1);
}

// Of a row's sum of weights; a row without any (its scores are all -infinite) counts nothing.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

__device__ __forceinline__ int account_blocks_dev(int keys) { return (keys + kAccountKeys - 1) / kAccountKeys; }

__device__ __forceinline__ void lds_dma(const void *src, uint16_t *dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
}

template <int D, bool PAGED>
__global__ __launch_bounds__(kThreads, 2) void account_stats_kernel(AccountArgs a) {
    constexpr int KS = D / 32, KP = D / 8;
    constexpr int NKI = kTile * KP / kThreads; // K pieces per thread
    __shared__ __align__(16) uint16_t ks0[kTile * D], ks1[kTile * D];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    const AccountPiece piece = Pieces(a.tiles, a.nt).of_item(item);
    const int          ei = (int)(piece.what & 255u), nch = (int)(piece.what >> 8);
    const int row = a.e[ei].row, p0 = a.e[ei].p0, n = a.e[ei].n, w = a.e[ei].w;
    const int rel = item - piece.item0, ch = rel % nch, rt = piece.first + rel / nch;
    const int rows = w << a.lg;
    const int r_lo = rt * kAccountRows, r_hi = min(rows, r_lo + kAccountRows);
    const int first = p0 + n - w;                          // position of query row 0's token
    const int kend = first + ((r_hi - 1) >> a.lg) + 1;     // keys that some row of the tile sees
    const int tiles = (kend + kTile - 1) / kTile;
    const int t_lo = (int)((int64_t)ch * tiles / nch), t_hi = (int)((int64_t)(ch + 1) * tiles / nch);
    const int c = lane & 15, qg = lane >> 4;

    f16x8 qb[2][KS];
    int   pos[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int     r = min(r_lo + wave * 32 + j * 16 + c, rows - 1);
        const __half *qp = a.q + ((int64_t)(a.e[ei].tok0 + n - w + (r >> a.lg)) * a.Hq + (g << a.lg) + (r & ((1 << a.lg) - 1))) * D;
        pos[j] = first + (r >> a.lg);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            // (a negative scale's sign goes into q: the maximum over s is then that over s * scale)
            const f16x8 v = *reinterpret_cast<const f16x8 *>(qp + 32 * s + 8 * qg);
            qb[j][s] = a.scale_log2 < 0.0f ? -v : v;
        }
    }
    const float scale = fabsf(a.scale_log2);
    const char *kb = reinterpret_cast<const char *>(a.kv.k_base) + (int64_t)g * a.kv.head_stride * 2;
    // A wave's 64 pieces of a load lie in one quarter of 16 tokens, whose offset is
    // uniform: ids has the quarters' blocks in its first lanes (paged views), asked
    // for a tile ahead.
    const uint32_t tokb = (uint32_t)(a.kv.tok_stride * 2);
    const int32_t *bt = PAGED ? a.kv.block_table + (int64_t)row * a.kv.bt_stride : nullptr;
    auto blocks = [&](int kt) -> int {
        if constexpr (PAGED) return lane < 4 ? bt[min(kt * kTile + 16 * lane, kend - 1) >> a.kv.log2_blk] : 0;
        else return 0;
    };
    uint32_t lane_off[NKI]; // in the quarter
#pragma unroll
    for (int u = 0; u < NKI; ++u) {
        const int sl = u * kThreads + (int)threadIdx.x, r = sl / KP;
        lane_off[u] = (uint32_t)(r % 16) * tokb + 16u * ((sl % KP) ^ swz<KP>(r));
    }
    auto issue = [&](int kt, int ids, uint16_t *dst) __attribute__((always_inline)) {
        const bool whole = kt * kTile + kTile <= kend;
#pragma unroll
        for (int u = 0; u < NKI; ++u) {
            const int q = (u * kThreads + wave * 64) / KP / 16; // the quarter
            const int tq = min(kt * kTile + 16 * q, kend - 1);
            int64_t   off;
            if constexpr (PAGED)
                off = ((int64_t)__builtin_amdgcn_readlane(ids, q) * a.kv.blk_stride +
                       (int64_t)(tq & ((1 << a.kv.log2_blk) - 1)) * a.kv.tok_stride) * 2;
            else off = ((int64_t)row * a.kv.blk_stride + (int64_t)tq * a.kv.tok_stride) * 2;
            uint32_t lo = lane_off[u];
            if (!whole) { // rows past the end: the last one
                const int r = (u * kThreads + (int)threadIdx.x) / KP % 16, more = kend - 1 - tq;
                lo -= (uint32_t)max(0, r - more) * tokb;
            }
            lds_dma(kb + off + lo, dst + (u * kThreads + wave * 64) * 8);
        }
    };
    float m[2] = {kNone, kNone}, l[2] = {0.0f, 0.0f};
    const int low = first + ((r_lo + wave * 32) >> a.lg); // the first position among the wave's rows
    // Straight-line code, so that one row group's matrix operations run under the
    // other's exponentials; tiles at the diagonal have code of their own.
    int  ids = 0;
    auto step = [&](auto diagonal, int kt, const uint16_t *kd, uint16_t *kn) __attribute__((always_inline)) {
        if (kt + 1 < t_hi) {
            const int now = ids;
            if (PAGED && kt + 2 < t_hi) ids = blocks(kt + 2);
            issue(kt + 1, now, kn);
        }
        f32x4 s[2][4];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int j = 0; j < 2; ++j) s[j][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const int   r = 16 * tt + c;
                const f16x8 kf = *reinterpret_cast<const f16x8 *>(&kd[(r * KP + ((4 * k + qg) ^ swz<KP>(r))) * 8]);
#pragma unroll
                for (int j = 0; j < 2; ++j) s[j][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qb[j][k], s[j][tt], 0, 0, 0);
            }
        const int tb = kt * kTile + 4 * qg;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if constexpr (diagonal) {
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (tb + 16 * tt + i > pos[j]) s[j][tt][i] = -INFINITY;
            }
            float mloc = s[j][0][0];
#pragma unroll
            for (int x = 1; x < 16; ++x) mloc = fmaxf(mloc, s[j][x / 4][x % 4]);
            const float m_new = fmaxf(m[j], mloc * scale);
            float       sum[4] = {l[j] * __builtin_amdgcn_exp2f(m[j] - m_new), 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][tt][i], scale, -m_new));
            l[j] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
            m[j] = m_new;
        }
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __syncthreads();
    };
    auto any_step = [&](int kt, const uint16_t *kd, uint16_t *kn) __attribute__((always_inline)) {
        if (kt * kTile + kTile - 1 > low) step(std::true_type(), kt, kd, kn);
        else step(std::false_type(), kt, kd, kn);
    };
    if (t_lo < t_hi) {
        issue(t_lo, blocks(t_lo), ks0);
        if (PAGED && t_lo + 1 < t_hi) ids = blocks(t_lo + 1);
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __syncthreads();
        for (int kt = t_lo; kt < t_hi; kt += 2) {
            any_step(kt, ks0, ks1);
            if (kt + 1 < t_hi) any_step(kt + 1, ks1, ks0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float mr = fmaxf(m[j], __shfl_xor(m[j], 16));
        mr = fmaxf(mr, __shfl_xor(mr, 32));
        float lr = l[j] * __builtin_amdgcn_exp2f(m[j] - mr);
        lr += __shfl_xor(lr, 16);
        lr += __shfl_xor(lr, 32);
        const int r = r_lo + wave * 32 + j * 16 + c;
        if (qg > 0 || r >= r_hi) continue;
        if (a.e[ei].nch == 1) {
            const int64_t at = (int64_t)a.e[ei].lse0 * a.Hkv + (int64_t)g * rows + r;
            *reinterpret_cast<float2 *>(a.rows + 2 * at) = make_float2(mr, inverse(lr));
        } else {
            const int64_t at = (int64_t)a.e[ei].stat0 * a.Hkv + ((int64_t)ch * a.Hkv + g) * rows + r;
            *reinterpret_cast<float2 *>(a.stats + 2 * at) = make_float2(mr, lr);
        }
    }
}

// (m, 1 / l) of row r from its nch chunks' (m, l), st: those of chunk 0, `step` floats from
// chunk to chunk.  Four lanes a row, 16 apart, take every fourth chunk, so that a
// load is of 16 neighbouring rows.
__device__ __forceinline__ float2 merged_row(const float *st, int64_t step, int nch) {
    float m = kNone, l = 0.0f;
#pragma unroll 4
    for (int ch = (threadIdx.x >> 4) & 3; ch < nch; ch += 4) {
        const float2 ml = *reinterpret_cast<const float2 *>(st + ch * step);
        const float  mn = fmaxf(m, ml.x);
        l = l * __builtin_amdgcn_exp2f(m - mn) + ml.y * __builtin_amdgcn_exp2f(ml.x - mn);
        m = mn;
    }
    float mx = fmaxf(m, __shfl_xor(m, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    l *= __builtin_amdgcn_exp2f(m - mx);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    return make_float2(mx, inverse(l));
}

// The rows of entries with several chunks of keys, where account_sum_kernel
// does not merge them itself.
__global__ __launch_bounds__(kThreads) void account_merge_kernel(AccountArgs a) {
    const int ei = blockIdx.z, g = blockIdx.y;
    const int nch = a.e[ei].nch, rows = a.e[ei].w << a.lg;
    const int r = blockIdx.x * (kThreads / 4) + (threadIdx.x >> 6) * 16 + (threadIdx.x & 15);
    const int r0 = blockIdx.x * (kThreads / 4) + (threadIdx.x >> 6) * 16; // the wave's first row
    if (nch == 1 || r0 >= rows) return;
    const float *st = a.stats + 2 * ((int64_t)a.e[ei].stat0 * a.Hkv + (int64_t)g * rows + min(r, rows - 1));
    const float2 v = merged_row(st, 2 * (int64_t)a.Hkv * rows, Pieces(a.tiles, a.nt).chunks(ei, r0 / kAccountRows));
    if ((threadIdx.x & 63) < 16 && r < rows)
        *reinterpret_cast<float2 *>(a.rows + 2 * ((int64_t)a.e[ei].lse0 * a.Hkv + (int64_t)g * rows + r)) = v;
}

template <int D, bool PAGED>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void account_sum_kernel(AccountArgs a) {
    constexpr int KS = D / 32, KP = D / 8;
    constexpr int NQI = kAccountStep * KP / kThreads; // Q pieces per thread
    constexpr int NRG = kAccountStep / 16;
    __shared__ __align__(16) uint16_t qs0[kAccountStep * D], qs1[kAccountStep * D];
    __shared__ float2 s_rows[kAccountFold];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    const Pieces       tile_pieces(a.tiles, a.nt);
    const AccountPiece piece = Pieces(a.blocks, a.nb).of_item(item);
    const int          ei = (int)(piece.what & 255u), nrc = (int)(piece.what >> 8);
    const int row = a.e[ei].row, p0 = a.e[ei].p0, n = a.e[ei].n, w = a.e[ei].w;
    const int rel = item - piece.item0, rchunk = rel % nrc, kblk = piece.first + rel / nrc;
    const int k_lo = kblk * kAccountKeys, keys = p0 + n;
    const int rows = w << a.lg, first = keys - w;
    // The chunk's rows, of the steps from the first one whose tokens see the block's first key.
    const int sees = (max(0, k_lo - first) << a.lg) / kAccountStep;
    const int steps = (rows + kAccountStep - 1) / kAccountStep - sees;
    const int r_lo = (sees + (int)((int64_t)rchunk * steps / nrc)) * kAccountStep;
    const int r_hi = min(rows, (sees + (int)((int64_t)(rchunk + 1) * steps / nrc)) * kAccountStep);
    const int c = lane & 15, qg = lane >> 4;
    const int wk = k_lo + wave * 64; // the wave's first key

    const float2 *row_stats = reinterpret_cast<const float2 *>(a.rows) + (int64_t)a.e[ei].lse0 * a.Hkv + (int64_t)g * rows;
    const __half *qbase = a.q + ((int64_t)(a.e[ei].tok0 + n - w) * a.Hq + (g << a.lg)) * D;
    // (a step's rows begin at a whole token: 64 rows hold 64 >> lg tokens)
    uint32_t lane_off[NQI];
#pragma unroll
    for (int u = 0; u < NQI; ++u) {
        const int sl = u * kThreads + (int)threadIdx.x, r = sl / KP;
        lane_off[u] = ((uint32_t)(r >> a.lg) * (uint32_t)a.Hq + (uint32_t)(r & ((1 << a.lg) - 1))) * D + 8 * ((sl % KP) ^ swz<KP>(r));
    }
    auto issue = [&](int r0, uint16_t *dst) __attribute__((always_inline)) {
        const __half *base = qbase + (int64_t)(r0 >> a.lg) * a.Hq * D;
        if (r0 + kAccountStep <= rows) {
#pragma unroll
            for (int u = 0; u < NQI; ++u) lds_dma(base + lane_off[u], dst + (u * kThreads + wave * 64) * 8);
        } else { // rows past the end: the last one
#pragma unroll
            for (int u = 0; u < NQI; ++u) {
                const int sl = u * kThreads + (int)threadIdx.x, r = sl / KP, x = (sl % KP) ^ swz<KP>(r);
                const int qr = min(r, rows - 1 - r0);
                lds_dma(base + ((int64_t)(qr >> a.lg) * a.Hq + (qr & ((1 << a.lg) - 1))) * D + 8 * x,
                        dst + (u * kThreads + wave * 64) * 8);
            }
        }
    };
    const bool merges = a.fold && a.e[ei].nch > 1; // (the chunk has kAccountFold rows at most)
    auto load_rows = [&](int r0, float2(&x)[NRG]) __attribute__((always_inline)) {
        const float2 *p = row_stats + r0;
        const bool    whole = r0 + kAccountStep <= r_hi;
#pragma unroll
        for (int rg = 0; rg < NRG; ++rg) {
            const int r = 16 * rg + c;
            if (!merges && whole) {
                x[rg] = p[r];
            } else { // rows past the end: weights of 0
                x[rg] = make_float2(INFINITY, 0.0f);
                if (r0 + r < r_hi) x[rg] = merges ? float2(s_rows[min(r0 + r - r_lo, kAccountFold - 1)]) : float2(p[r]);
            }
        }
    };
    if (r_lo < r_hi) issue(r_lo, qs0);
    const char *kb = reinterpret_cast<const char *>(a.kv.k_base) + (int64_t)g * a.kv.head_stride * 2;
    f16x8       kf[4][KS];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        const char *p = kb + key_off<PAGED>(a.kv, row, min(wk + 16 * tt + c, keys - 1)) + 16 * qg;
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[tt][s] = *reinterpret_cast<const f16x8 *>(p + 64 * s);
    }
    f32x4 acc[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) acc[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (merges) { // while the first rows and the keys are on their way
        const float *st = a.stats + 2 * ((int64_t)a.e[ei].stat0 * a.Hkv + (int64_t)g * rows);
        for (int r0 = r_lo + 16 * wave; r0 < r_hi; r0 += kThreads / 4) {
            const int    nch = tile_pieces.chunks(ei, r0 / kAccountRows);
            const float2 v = merged_row(st + 2 * (int64_t)min(r0 + c, r_hi - 1), 2 * (int64_t)a.Hkv * rows, nch);
            if (qg == 0 && r0 + c < r_hi) s_rows[r0 + c - r_lo] = v;
        }
        __syncthreads();
    }
    float2 x[NRG];
    load_rows(r_lo, x);
    __builtin_amdgcn_s_waitcnt(kVmcnt0);
    __syncthreads();
    auto compute = [&](auto diagonal, int r0, const uint16_t *qd) __attribute__((always_inline)) {
        // One group's scores are computed under the exponentials of the one before.
        f32x4 s[2][4];
        auto  scores = [&](int rg, f32x4(&t)[4]) __attribute__((always_inline)) {
            const int rr = 16 * rg + c;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) t[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const f16x8 qf = *reinterpret_cast<const f16x8 *>(&qd[(rr * KP + ((4 * k + qg) ^ swz<KP>(rr))) * 8]);
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) t[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tt][k], qf, t[tt], 0, 0, 0);
            }
        };
        scores(0, s[0]);
#pragma unroll
        for (int rg = 0; rg < NRG; ++rg) {
            if (rg + 1 < NRG) scores(rg + 1, s[(rg + 1) & 1]);
            const int pos = first + (min(r0 + 16 * rg + c, rows - 1) >> a.lg);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rg & 1][tt][i], a.scale_log2, -x[rg].x));
                    if constexpr (diagonal) p = wk + 16 * tt + 4 * qg + i <= pos ? p : 0.0f;
                    acc[tt][i] = __builtin_fmaf(p, x[rg].y, acc[tt][i]);
                }
        }
    };
    auto any_step = [&](int r0, const uint16_t *qd, uint16_t *qn) __attribute__((always_inline)) {
        float2 y[NRG];
        if (r0 + kAccountStep < r_hi) {
            issue(r0 + kAccountStep, qn);
            load_rows(r0 + kAccountStep, y);
        }
        if (wk + 63 <= first + (r0 >> a.lg)) compute(std::false_type(), r0, qd); // every row sees every key
        else if (wk <= first + ((r0 + kAccountStep - 1) >> a.lg)) compute(std::true_type(), r0, qd);
#pragma unroll
        for (int rg = 0; rg < NRG; ++rg) x[rg] = y[rg];
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __syncthreads();
    };
    for (int r0 = r_lo; r0 < r_hi; r0 += 2 * kAccountStep) {
        any_step(r0, qs0, qs1);
        if (r0 + kAccountStep < r_hi) any_step(r0 + kAccountStep, qs1, qs0);
    }
    const int64_t base = ((int64_t)row * a.Hkv + g) * a.room;
    float        *part = a.parts + (int64_t)a.e[ei].part0 * a.Hkv +
                  ((int64_t)rchunk * a.Hkv + g) * ((int64_t)account_blocks_dev(keys) * kAccountKeys);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        f32x4 v = acc[tt];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) v[i] += __shfl_xor(v[i], o);
        const int t = wk + 16 * tt + 4 * qg;
        if (c > 0) continue;
        if (a.e[ei].nrc > 1) {
            *reinterpret_cast<f32x4 *>(part + t) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t + i < keys) a.w_out[base + t + i] = (a.w_in && t + i < p0 ? a.w_in[base + t + i] : 0.0f) + v[i];
        }
    }
}

// The accounts of entries with several chunks of rows.
__global__ __launch_bounds__(kThreads) void account_join_kernel(AccountArgs a) {
    static_assert(kThreads == kAccountKeys, "a workgroup per block");
    const int ei = blockIdx.z, g = blockIdx.y, t = blockIdx.x * kThreads + threadIdx.x;
    const int p0 = a.e[ei].p0, keys = p0 + a.e[ei].n;
    if (a.e[ei].nrc == 1 || (int)blockIdx.x * kThreads >= keys) return;
    const int     nrc = Pieces(a.blocks, a.nb).chunks(ei, blockIdx.x);
    const int64_t base = ((int64_t)a.e[ei].row * a.Hkv + g) * a.room, len = (int64_t)account_blocks_dev(keys) * kAccountKeys;
    const float  *part = a.parts + (int64_t)a.e[ei].part0 * a.Hkv + (int64_t)g * len + t;
    float         sum = a.w_in && t < p0 ? a.w_in[base + t] : 0.0f;
#pragma unroll 8
    for (int k = 0; k < nrc; ++k) sum += part[(int64_t)k * a.Hkv * len];
    if (t < keys) a.w_out[base + t] = sum;
}

template <int D> void launch_d(const AccountArgs &a, const AccountLaunch &l, bool paged, hipStream_t stream) {
    const dim3 stats((unsigned)l.items * (unsigned)a.Hkv), sums((unsigned)l.sums * (unsigned)a.Hkv), block(kThreads);
    if (paged) hipLaunchKernelGGL((account_stats_kernel<D, true>), stats, block, 0, stream, a);
    else hipLaunchKernelGGL((account_stats_kernel<D, false>), stats, block, 0, stream, a);
    HIP_CHECK(hipGetLastError());
    if (l.split_keys && !l.fold) {
        const dim3 grid((unsigned)((l.most_rows + kThreads / 4 - 1) / (kThreads / 4)), (unsigned)a.Hkv, (unsigned)l.n);
        hipLaunchKernelGGL(account_merge_kernel, grid, block, 0, stream, a);
        HIP_CHECK(hipGetLastError());
    }
    if (paged) hipLaunchKernelGGL((account_sum_kernel<D, true>), sums, block, 0, stream, a);
    else hipLaunchKernelGGL((account_sum_kernel<D, false>), sums, block, 0, stream, a);
    HIP_CHECK(hipGetLastError());
    if (l.split_rows) {
        const dim3 grid((unsigned)((l.most_keys + kThreads - 1) / kThreads), (unsigned)a.Hkv, (unsigned)l.n);
        hipLaunchKernelGGL(account_join_kernel, grid, block, 0, stream, a);
        HIP_CHECK(hipGetLastError());
    }
}

} // namespace

size_t account_workspace_floats(const AccountPlan &plan, int Hkv) {
    int64_t most = 0;
    for (const auto &l : plan.launches) most = std::max(most, 2 * l.lse + 2 * l.stats + l.parts);
    return (size_t)most * (size_t)Hkv;
}

void launch_account(const AccountCall &c, const KvView &kv, const AccountPlan &plan, float *workspace,
                    hipStream_t stream) {
    AccountArgs a;
    a.q = c.q;
    a.w_in = c.w_in;
    a.w_out = c.w_out;
    a.kv = kv;
    a.room = c.room;
    // (0: so small that every score is 0 beside a masked one's -infinity)
    a.scale_log2 = c.scale == 0.0f ? 1e-37f : c.scale * 1.4426950408889634f;
    a.Hq = c.Hq;
    a.Hkv = c.Hkv;
    a.lg = __builtin_ctz((unsigned)(c.Hq / c.Hkv));
    const bool paged = kv.block_table != nullptr;
    for (const auto &l : plan.launches) {
        if (l.n == 0 || l.items == 0) continue;
        a.n = l.n;
        a.fold = l.fold;
        a.parts = workspace; // (multiples of 256 first: their stores are of 16 bytes)
        a.stats = a.parts + l.parts * c.Hkv;
        a.rows = a.stats + 2 * l.stats * c.Hkv;
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(AccountEntry) * (size_t)l.n);
        a.nt = (int)l.tile_pieces.size();
        a.nb = (int)l.block_pieces.size();
        std::memcpy(a.tiles, l.tile_pieces.data(), sizeof(AccountPiece) * l.tile_pieces.size());
        std::memcpy(a.blocks, l.block_pieces.data(), sizeof(AccountPiece) * l.block_pieces.size());
        profile_begin(KernelId::AttnAccount, stream);
        switch (c.D) {
        case 32: launch_d<32>(a, l, paged, stream); break;
        case 64: launch_d<64>(a, l, paged, stream); break;
        case 128: launch_d<128>(a, l, paged, stream); break;
        case 256: launch_d<256>(a, l, paged, stream); break;
        default: throw std::invalid_argument("attention account: unsupported head_dim");
        }
        profile_end(KernelId::AttnAccount, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
