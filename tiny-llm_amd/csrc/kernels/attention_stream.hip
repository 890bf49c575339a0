// Attention of a few query rows over a KV view that is read once, with an account
// of every token's weight, for gfx950.
//
// An entry's query rows of kv head g (tokens x G heads, at most 16) over its S
// cached tokens:
//   s_rt = (q_r . k_t) * scale,   P_rt = exp(s_rt - max_t s_rt) / sum_t exp(...)
//   o_r  = sum_t P_rt v_t          (sum + 1e-6 in the denominator, as in decode)
//   account_out[t] = account_in[t] + sum_r P_rt
// Bound by HBM: K and V once, 4 D bytes a token and kv head.  The account needs the
// rows' maxima and sums over all tokens before its first weight, but reading K a
// second time for it would cost half of the whole, so the scores (fp32, as the sums: an
// account is compared with others of like size) wait in LDS, 4 bytes a row and token.
//
// attn_stream_kernel: a workgroup of 4 or 8 waves per (entry, chunk of tiles, kv
// head); wave w takes every 4th (8th) tile of 64 tokens (32 at head_dim 256) and keeps
// its own running maximum, sum and output; the next tile's rows are on their way
// while one is computed.  A workgroup that has a whole entry finishes it; the others
// write their chunk's scores at the end, in one go (a write among the reads costs far
// more than its bytes: scores stored tile by tile took 77-95 of 474 us).
//   S^T = K Q^T      v_mfma_f32_16x16x32_f16: A = K rows (token l%16, dims
//                    8(l/16)..+7) straight from memory, B = Q (row l%16),
//                    D = S^T (tokens 4(l/16)+i, row l%16)
//   softmax          per row column in the log2 domain, over a reference point near
//                    the maximum (kBelow), in fp32
//   O^T += V^T P^T   over 16 tokens; V^T from the wave's row-major LDS stage by
//                    the transposing ds_read_b64_tr_b16.  A weight takes part as two
//                    fp16 numbers, its rounding and that of the rest, 2^-22 of it, side
//                    by side in the instruction's 32 places beside V^T twice, so
//                    the matrix unit has no more to do than for one of them
// stream_finish_kernel: merges the outputs of entries with several chunks and turns
// their scores into the account.
//
// Measured, with accounts, 8 kv heads of 128: 64 x 8192 tokens, group 4, whole
// entries: 361 us, 6.0 TB/s of K and V (without accounts the decode kernel takes 309 on
// the same cache); 96 lognormal lengths to 16384 on blocks, group 8: 272 + 20 us for
// the finish (27 with a row's scores on their way at a time, 30 with all eight);
// 4 x 128..512 tokens, 8 heads of 64: 7.7 us, one launch's latency (with the weights in one
// part 7.4, the others level).  Two or three steps of rows on their way in registers
// were level or slower (occupancy).
#include "stream.h"

#include "../runtime.h"
#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <mutex>
#include <stdexcept>

namespace tiny_llm {
namespace detail {

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef short    s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Weights are 2^(s - ref).  The reference is 2^7 below the maximum when it moves, and
// moves on scores 2^15 above it only: weights stay below 2^15 in fp16, and those 2^-31
// of the largest are still above its smallest step.  (A reference at the maximum lost
// all weights 2^-25 below it, which a long cache of even ones feels.)
constexpr float kBelow = 7.0f, kLazyMax = 15.0f;
// The reference over no score, or over -infinite ones only: finite, so that a score of
// -infinity has the weight 0 beside it, and below every finite score.
constexpr float kNone = -3e38f;

struct StreamArgs {
    const __half *q;
    __half       *out;
    const __half *new_k, *new_v;
    const float  *w_in;
    float        *w_out;
    float        *part_o;  // [item][Hkv][16 rows at most][D]
    float        *part_ml; // [item][Hkv][rows][2]
    float        *scores;  // [tile0 * Hkv + g * tiles + tile][rows][64], tile0 counted over entries of several chunks
    KvView        kv;
    int64_t       room;
    int           fresh;
    float         scale_log2;
    int           Hq, Hkv, G, n, chunk, rows; // rows: of the partials, nq * G at most
    StreamEntry   e[kStreamBatch];
};
static_assert(sizeof(StreamArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ __attribute__((address_space(3))) s16x4 *lds_ptr(const uint16_t *p) {
    return (__attribute__((address_space(3))) s16x4 *)(p);
}

__device__ __forceinline__ void wave_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Entry of work item `item`: the last with item0 <= item (entries without tokens
// have no items).
#define STREAM_ENTRY_OF(a, item, out)                                                                                  \
    do {                                                                                                               \
        int seen_ = 0;                                                                                                 \
        for (int k_ = 0; k_ < (a).n; k_ += 64) {                                                                       \
            const int i_ = k_ + (int)(threadIdx.x & 63);                                                               \
            seen_ += __popcll(__ballot(i_ < (a).n && (a).e[min(i_, (a).n - 1)].item0 <= (item)));                      \
        }                                                                                                              \
        out = __builtin_amdgcn_readfirstlane(seen_ - 1);                                                               \
    } while (0)

// Of a row's sum of weights; a row without any (its scores are all -infinite) counts nothing.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// Four consecutive fp32 values; the rows of accounts begin at any multiple of 4 bytes.
struct __attribute__((packed, aligned(4))) Four {
    float x[4];
};

// The account of tokens [t_lo, t_hi) of entry ei and kv head g, t_lo a multiple of a
// tile, from their scores (sc: [tile][rows][64], in LDS or memory), the rows' final
// maxima and the inverse of their sums (in LDS).  U: accounts of so many fours on
// their way at once; 1 with several rows' scores (from memory).
template <int NT, int U>
__device__ __forceinline__ void account_tokens(const StreamArgs &a, int ei, int g, int rows, int t_lo, int t_hi,
                                               const float *sc, const float *m, const float *inv) {
    constexpr int ROWS = U == 1 && NT == 256 ? 4 : 1;
    const int     old = a.e[ei].S - a.fresh;
    const int64_t base = ((int64_t)a.e[ei].row * a.Hkv + g) * a.room;
    for (int t0 = t_lo + 4 * (int)threadIdx.x; t0 < t_hi; t0 += 4 * NT * U) {
        Four w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t0 + u * 4 * NT;
            w[u] = Four{};
            if (a.w_in && t + 4 <= old) w[u] = *reinterpret_cast<const Four *>(a.w_in + base + t);
            else if (a.w_in) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i < old) w[u].x[i] = a.w_in[base + t + i];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t0 + u * 4 * NT;
            if (t >= t_hi) break;
            const float *st = sc + (int64_t)((t - t_lo) / kStreamTile) * rows * kStreamTile + t % kStreamTile;
            f32x4        sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll ROWS
            for (int r = 0; r < rows; ++r) { // (scores past the end are -infinity)
                const f32x4 s = *reinterpret_cast<const f32x4 *>(st + r * kStreamTile);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(__builtin_amdgcn_exp2f(s[i] - m[r]), inv[r], sum[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) w[u].x[i] += sum[i];
            if (t + 4 <= t_hi) *reinterpret_cast<Four *>(a.w_out + base + t) = w[u];
            else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i < t_hi) a.w_out[base + t + i] = w[u].x[i];
            }
        }
    }
}

// Dynamic LDS: the waves' V stages, then with SCORES the chunk's scores.
template <int D, bool PAGED, bool SCORES, int NW>
__global__ __launch_bounds__(NW * 64, D <= 128 ? 2 : 1) void attn_stream_kernel(StreamArgs a) {
    constexpr int TK = D <= 128 ? 64 : 32; // tokens of a wave's step
    constexpr int SUB = kStreamTile / TK;  // steps per tile
    constexpr int TT = TK / 16;
    constexpr int KS = D / 32, DT = D / 16, KP = D / 8;
    constexpr int NV = TK * KP / 64;       // V pieces per lane
    constexpr int NQ = NV / TT;            // ... of 16 tokens
    constexpr int RPI = 64 / KP;           // V rows per load instruction
    constexpr int ROWS = SCORES ? kStreamRows / 2 : kStreamRows;
    constexpr int STAGE = stream_stage_bytes(D, SCORES) / 2; // halves: 16 V rows, then o[ROWS][D] fp32
    extern __shared__ __align__(16) uint16_t smem[];
    __shared__ float sm[NW][16], sl[NW][16], s_m[16], s_l[16], s_inv[16];
    // 16-byte piece x of row r at slot x ^ swz(r): the transposing reads of rows
    // 4 apart and of neighbours fall on distinct banks.
    auto swz = [](int r) {
        if constexpr (KP <= 4) return r & (KP - 1);
        const int f = ((r & 3) << 1) ^ (((r >> 2) & 1) * 9) ^ (((r >> 3) & 1) << 3);
        return f & (KP - 1);
    };
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    STREAM_ENTRY_OF(a, item, ei);
    const int row = a.e[ei].row, S = a.e[ei].S, tok0 = a.e[ei].tok0, rows = a.e[ei].nq * a.G;
    const int tiles = (S + kStreamTile - 1) / kStreamTile;
    const int nch = (tiles + a.chunk - 1) / a.chunk, ch = item - a.e[ei].item0;
    const int tile_lo = (int)((int64_t)ch * tiles / nch), tile_hi = (int)((int64_t)(ch + 1) * tiles / nch);
    const int last = min(S, tile_hi * kStreamTile) - 1; // last token of the chunk

    const int64_t  head = (int64_t)g * a.kv.head_stride * 2;
    const char    *kb = reinterpret_cast<const char *>(a.kv.k_base) + head;
    const char    *vb = reinterpret_cast<const char *>(a.kv.v_base) + head;
    const int64_t  blk_bytes = a.kv.blk_stride * 2, tokb = a.kv.tok_stride * 2;
    const int32_t *bt = PAGED ? a.kv.block_table + (int64_t)row * a.kv.bt_stride : nullptr;
    const int      mask = (1 << a.kv.log2_blk) - 1;

    if (a.new_k && ch == nch - 1) { // the new token's row, then read like any other
        if ((int)threadIdx.x < 2 * KP) {
            const int     which = threadIdx.x / KP, x = threadIdx.x - which * KP, t = S - 1;
            const __half *src = (which ? a.new_v : a.new_k) + ((int64_t)tok0 * a.Hkv + g) * D + 8 * x;
            const int64_t off = PAGED ? (int64_t)bt[t >> a.kv.log2_blk] * blk_bytes + (int64_t)(t & mask) * tokb
                                      : (int64_t)row * blk_bytes + (int64_t)t * tokb;
            char         *dst = const_cast<char *>(which ? vb : kb) + off + 16 * x;
            *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
        }
        __threadfence_block();
        __syncthreads();
    }

    const int c = lane & 15, qg = lane >> 4;
    f16x8     qb[KS]; // B operand: row c, dims 32s + 8qg .. +7
    {
        const int     r = min(c, rows - 1);
        const __half *qp = a.q + ((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const f16x8 *>(qp + 32 * s + 8 * qg);
    }
    f32x4 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kNone, l_run = 0.0f;

    // The wave's steps: step x of the chunk's tiles, tile tile_lo + x / SUB * NW + wave.
    const int steps = max(0, (tile_hi - tile_lo - wave + NW - 1) / NW) * SUB;
    auto start = [&](int x) { return (tile_lo + x / SUB * NW + wave) * kStreamTile + x % SUB * TK; };
    // Block ids of a step's quarters of 16 tokens, lane k that of quarter k (paged
    // views).  Loads complete in the order of their issue, so ids are asked for before
    // the rows that are on their way when they are needed: two steps ahead.
    auto blocks = [&](int x) -> int {
        if constexpr (PAGED) return lane < TT ? bt[min(start(x) + 16 * lane, last) >> a.kv.log2_blk] : 0;
        else return 0;
    };
    // Offset of the 16 tokens from quarter k on (its first token clamped to the last
    // one), and how many of them may be read past the first.
    auto quarter = [&](int t0, int k, int ids, int &more) __attribute__((always_inline)) -> int64_t {
        const int tq = min(t0 + 16 * k, last);
        more = min(15, last - tq);
        if constexpr (PAGED)
            return (int64_t)__builtin_amdgcn_readlane(ids, k) * blk_bytes + (int64_t)(tq & mask) * tokb;
        else return (int64_t)row * blk_bytes + (int64_t)tq * tokb;
    };
    f16x8 kf[TT][KS];
    u32x4 vr[NV];
    auto load_k = [&](int x, int ids) __attribute__((always_inline)) {
        const int t0 = __builtin_amdgcn_readfirstlane(start(x));
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            int            more;
            const char    *p = kb + quarter(t0, tt, ids, more);
            const uint32_t off = (uint32_t)min(c, more) * (uint32_t)tokb + 16 * qg;
#pragma unroll
            for (int s = 0; s < KS; ++s) kf[tt][s] = *reinterpret_cast<const f16x8 *>(p + off + 64 * s);
        }
    };
    auto load_v = [&](int x, int ids) __attribute__((always_inline)) {
        const int t0 = __builtin_amdgcn_readfirstlane(start(x));
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int      r = (u * RPI) % 16 + lane / KP; // in its quarter
            int            more;
            const char    *p = vb + quarter(t0, u * RPI / 16, ids, more);
            const uint32_t off = (uint32_t)min(r, more) * (uint32_t)tokb + 16 * (lane % KP);
            // (whole lines, read once; K's lines are read in halves, which the hint made slower)
            vr[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + off));
        }
    };
    uint16_t *vst = smem + wave * STAGE;
    float    *lsc = reinterpret_cast<float *>(smem + NW * STAGE); // [tile of the chunk][rows][64]
    const int vrow = 4 * qg + (c >> 2);
    const int vlane = vrow * KP * 8 + 4 * (c & 1), vxor = ((c & 3) >> 1) ^ swz(vrow);

    int ids = blocks(0), next = PAGED && steps > 1 ? blocks(1) : 0;
    if (steps > 0) {
        load_k(0, ids);
        load_v(0, ids);
    }
    for (int x = 0; x < steps; ++x) {
        const int  t0 = start(x);
        const bool more = x + 1 < steps;
        ids = next;
        if (PAGED && x + 2 < steps) next = blocks(x + 2);
        f32x4 s[TT];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KS; ++i) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tt][i], qb[i], s[tt], 0, 0, 0);
        }
        if (more) load_k(x + 1, ids);
        const int tb = t0 + 4 * qg;
        float     mloc = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y = s[tt][i] * a.scale_log2;
                s[tt][i] = tb + 16 * tt + i <= last ? y : -INFINITY;
                mloc = fmaxf(mloc, s[tt][i]);
            }
        if constexpr (SCORES) {
            float *dst = lsc + (t0 / kStreamTile - tile_lo) * rows * kStreamTile + t0 % kStreamTile + c * kStreamTile + 4 * qg;
            if (c < rows)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) *reinterpret_cast<f32x4 *>(dst + 16 * tt) = s[tt];
        }
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
        if (t0 + TK - 1 > last) { // rows past the end, read as the last one: 0 times its value would be NaN where that is infinite
#pragma unroll
            for (int u = 0; u < NV; ++u)
                if (t0 + u * RPI + lane / KP > last) vr[u] = u32x4{0u, 0u, 0u, 0u};
        }
        // 16 tokens at a time through the stage (a wave's LDS operations keep their order).
#pragma unroll
        for (int q = 0; q < TT; ++q) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                const int r = u * RPI + lane / KP;
                *reinterpret_cast<u32x4 *>(&vst[(r * KP + ((lane % KP) ^ swz(r))) * 8]) = vr[q * NQ + u];
            }
            f16x8 pf; // p's rounding to fp16, then that of the rest
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(s[q][i] - m_run);
                l_run += p;
                pf[i] = (_Float16)p;
                pf[4 + i] = (_Float16)(p - (float)pf[i]);
            }
            wave_sync_lds();
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const f16x4 v = __builtin_bit_cast(
                    f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr(&vst[vlane + ((2 * dt) ^ vxor) * 8])));
                // (an infinite value times a rest of 0, or of the other sign, would be NaN)
                const f16x4 most = {65504.0f16, 65504.0f16, 65504.0f16, 65504.0f16};
                const f16x4 fin = __builtin_elementwise_max(__builtin_elementwise_min(v, most), -most);
                acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(v, fin, 0, 1, 2, 3, 4, 5, 6, 7), pf,
                                                                 acc[dt], 0, 0, 0);
            }
            wave_sync_lds();
        }
        if (more) load_v(x + 1, ids);
    }

    // The waves' (m, l, o) through LDS.
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    float *so = reinterpret_cast<float *>(vst);
    if (c < ROWS)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4 *>(so + c * D + 16 * dt + 4 * qg) = acc[dt];
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
        s_m[r] = m;
        s_l[r] = l;
        s_inv[r] = inverse(l);
        if (nch > 1)
            *reinterpret_cast<float2 *>(a.part_ml + (((int64_t)item * a.Hkv + g) * a.rows + r) * 2) = make_float2(m, l);
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < rows * D; idx += NW * 64) {
        const int r = idx / D, d = idx - r * D;
        float     o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) o = fmaf(sm[w][r], reinterpret_cast<const float *>(smem + w * STAGE)[idx], o);
        if (nch == 1)
            a.out[((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D + d] = __float2half(o * (1.0f / (s_l[r] + 1e-6f)));
        else a.part_o[(((int64_t)item * a.Hkv + g) * a.rows + r) * D + d] = o;
    }
    if constexpr (SCORES) {
        if (nch == 1) {
            account_tokens<NW * 64, NW == 8 ? 1 : 8>(a, ei, g, rows, 0, S, lsc, s_m, s_inv);
        } else { // the chunk's scores in one go
            float *dst = a.scores + ((int64_t)a.e[ei].tile0 * a.Hkv + (int64_t)g * tiles + tile_lo) * a.rows * kStreamTile;
            for (int k = threadIdx.x; k < (tile_hi - tile_lo) * rows * (kStreamTile / 4); k += NW * 64)
                *reinterpret_cast<f32x4 *>(dst + 4 * k) = *reinterpret_cast<const f32x4 *>(lsc + 4 * k);
        }
    }
}

constexpr int kFinishThreads = 256;
constexpr int kFinishTokens = 1024; // tokens of a block
constexpr int kMostBlocks = 32768;  // grid.y

// Entries of several chunks (or none: zero rows).  Workgroup (entry, kv head, y):
// the rows' maxima and sums over the chunks; every gridDim.y-th block of tokens'
// account and row's output, whose chunks are spread over the threads.
__global__ __launch_bounds__(kFinishThreads) void stream_finish_kernel(StreamArgs a, int D) {
    __shared__ float s_m[kStreamRows], s_l[kStreamRows], s_inv[kStreamRows];
    __shared__ f32x4 s_o[kFinishThreads];
    const int ei = blockIdx.x / a.Hkv, g = blockIdx.x - ei * a.Hkv;
    const int S = a.e[ei].S, tok0 = a.e[ei].tok0, rows = a.e[ei].nq * a.G;
    const int tiles = (S + kStreamTile - 1) / kStreamTile;
    const int nch = (tiles + a.chunk - 1) / a.chunk;
    if (nch == 1 || ((int)blockIdx.y >= rows && (!a.w_out || (int)blockIdx.y * kFinishTokens >= S))) return;
    const int64_t p0 = ((int64_t)a.e[ei].item0 * a.Hkv + g) * a.rows; // row 0 of chunk 0
    const int64_t pc = (int64_t)a.Hkv * a.rows;                      // from chunk to chunk
    const int     lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r < rows; r += kFinishThreads / 64) {
        if (!a.w_out && r % (int)gridDim.y != (int)blockIdx.y) continue; // (an account takes every row)
        float m = -INFINITY, l = 0.0f;
        for (int ch = lane; ch < nch; ch += 64) {
            const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + (p0 + ch * pc + r) * 2);
            const float  mn = fmaxf(m, ml.x);
            l = fmaf(l, __builtin_amdgcn_exp2f(m - mn), ml.y * __builtin_amdgcn_exp2f(ml.x - mn));
            m = mn;
        }
        float mx = m;
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        l = m == -INFINITY ? 0.0f : l * __builtin_amdgcn_exp2f(m - mx);
        for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
        if (lane == 0) {
            s_m[r] = mx;
            s_l[r] = l;
            s_inv[r] = inverse(l);
        }
    }
    __syncthreads();
    const int per = D / 4, groups = kFinishThreads / per, grp = threadIdx.x / per, d = 4 * (threadIdx.x % per);
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int ch = grp; ch < nch; ch += groups) {
            const int64_t pr = p0 + ch * pc + r;
            o += __builtin_amdgcn_exp2f(a.part_ml[pr * 2] - s_m[r]) * *reinterpret_cast<const f32x4 *>(a.part_o + pr * D + d);
        }
        s_o[threadIdx.x] = o;
        __syncthreads();
        if (grp == 0) {
            for (int k = 1; k < groups; ++k) o += s_o[threadIdx.x + k * per];
            const float   inv = nch ? 1.0f / (s_l[r] + 1e-6f) : 0.0f;
            const __half2 lo = __floats2half2_rn(o[0] * inv, o[1] * inv), hi = __floats2half2_rn(o[2] * inv, o[3] * inv);
            uint2         w;
            w.x = __builtin_bit_cast(uint32_t, lo);
            w.y = __builtin_bit_cast(uint32_t, hi);
            *reinterpret_cast<uint2 *>(a.out + ((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D + d) = w;
        }
        __syncthreads();
    }
    if (a.w_out) { // (a launch with accounts has entries of one query: rows = a.rows)
        for (int64_t t = (int64_t)blockIdx.y * kFinishTokens; t < S; t += (int64_t)gridDim.y * kFinishTokens) {
            const int    t_lo = (int)t, t_hi = (int)min((int64_t)S, t + kFinishTokens);
            const float *sc = a.scores + ((int64_t)a.e[ei].tile0 * a.Hkv + (int64_t)g * tiles + t_lo / kStreamTile) * a.rows * kStreamTile;
            account_tokens<kFinishThreads, 1>(a, ei, g, rows, t_lo, t_hi, sc, s_m, s_inv);
        }
    }
}

// Floats of the partial maxima and sums, then the outputs at a multiple of 16 bytes.
size_t part_ml_floats(size_t rows) { return (2 * rows + 3) / 4 * 4; }

template <int D, bool PAGED, bool SCORES, int NW>
void launch_one(const StreamArgs &a, int items, int lds, hipStream_t stream) {
    auto                 *fn = attn_stream_kernel<D, PAGED, SCORES, NW>;
    static std::once_flag once[64]; // per device
    std::call_once(once[current_device() & 63], [&] {
        HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      kStreamLds));
    });
    hipLaunchKernelGGL(fn, dim3((unsigned)items * (unsigned)a.Hkv), dim3(NW * 64), lds, stream, a);
}
template <int D, bool SCORES> void launch_ds(const StreamArgs &a, int items, bool paged, const StreamPlan &plan, hipStream_t stream) {
    const int lds = plan.waves * stream_stage_bytes(D, SCORES) + (SCORES ? plan.most * kStreamTile * a.rows * 4 : 0);
    if constexpr (D <= 128) {
        if (plan.waves == 8) {
            if (paged) launch_one<D, true, SCORES, 8>(a, items, lds, stream);
            else launch_one<D, false, SCORES, 8>(a, items, lds, stream);
            return;
        }
    }
    if (paged) launch_one<D, true, SCORES, 4>(a, items, lds, stream);
    else launch_one<D, false, SCORES, 4>(a, items, lds, stream);
}
template <int D> void launch_d(const StreamArgs &a, int items, bool paged, const StreamPlan &plan, hipStream_t stream) {
    if (a.w_out) launch_ds<D, true>(a, items, paged, plan, stream);
    else launch_ds<D, false>(a, items, paged, plan, stream);
}

int plan_rows(const StreamPlan &plan, int first, int n, int G) {
    int nq = 1;
    for (int i = first; i < first + n; ++i) nq = std::max(nq, (int)plan.entries[(size_t)i].nq);
    return nq * G;
}

// Tiles whose scores go through memory: those of entries of several chunks.
int64_t stored_tiles(const StreamPlan &plan, const StreamLaunch &l) {
    int64_t tiles = 0;
    for (int i = l.first; i < l.first + l.n; ++i) {
        const StreamEntry &e = plan.entries[(size_t)i];
        if (stream_items(e.S, plan.chunk) > 1) tiles += stream_tiles(e.S);
    }
    return tiles;
}

} // namespace

size_t stream_workspace_floats(const StreamPlan &plan, int Hq, int Hkv, int D, bool account) {
    size_t most = 0;
    for (const auto &l : plan.launches) {
        const size_t rows = (size_t)plan_rows(plan, l.first, l.n, Hq / Hkv) * Hkv;
        size_t       f = part_ml_floats((size_t)l.items * rows) + (size_t)l.items * rows * (size_t)D;
        if (account) f += (size_t)stored_tiles(plan, l) * kStreamTile * rows;
        most = std::max(most, f);
    }
    return most;
}

void launch_attn_stream(const StreamCall &c, const KvView &kv, const StreamPlan &plan, float *workspace,
                        hipStream_t stream) {
    StreamArgs a;
    a.q = c.q;
    a.out = c.out;
    a.new_k = c.new_k;
    a.new_v = c.new_v;
    a.w_in = c.w_in;
    a.w_out = c.w_out;
    a.kv = kv;
    a.room = c.room;
    a.fresh = c.fresh;
    a.scale_log2 = c.scale * 1.4426950408889634f;
    a.Hq = c.Hq;
    a.Hkv = c.Hkv;
    a.G = c.Hq / c.Hkv;
    a.chunk = plan.chunk;
    const bool paged = kv.block_table != nullptr;
    for (const auto &l : plan.launches) {
        if (l.n == 0) continue;
        a.n = l.n;
        a.rows = plan_rows(plan, l.first, l.n, a.G);
        if (a.rows > kStreamRows) throw std::invalid_argument("attention: too many query rows per entry");
        if ((int64_t)l.items * c.Hkv > INT32_MAX) throw std::invalid_argument("attention: too many work items");
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(StreamEntry) * (size_t)l.n);
        int64_t tiles = 0; // (as stored_tiles)
        for (int i = 0; c.w_out && i < l.n; ++i) {
            if (stream_items(a.e[i].S, plan.chunk) <= 1) continue;
            a.e[i].tile0 = (int32_t)tiles;
            tiles += stream_tiles(a.e[i].S);
        }
        a.scores = workspace;
        a.part_ml = workspace + (size_t)tiles * kStreamTile * a.rows * c.Hkv;
        a.part_o = a.part_ml + part_ml_floats((size_t)l.items * c.Hkv * a.rows);
        profile_begin(KernelId::AttnStream, stream);
        if (l.items > 0) {
            switch (c.D) {
            case 32: launch_d<32>(a, l.items, paged, plan, stream); break;
            case 64: launch_d<64>(a, l.items, paged, plan, stream); break;
            case 128: launch_d<128>(a, l.items, paged, plan, stream); break;
            case 256: launch_d<256>(a, l.items, paged, plan, stream); break;
            default: throw std::invalid_argument("attention: unsupported head_dim");
            }
            HIP_CHECK(hipGetLastError());
        }
        if (l.finish) {
            const unsigned blocks = (unsigned)std::max(a.rows, c.w_out ? std::min(l.max_len / kFinishTokens + 1, kMostBlocks) : 1);
            hipLaunchKernelGGL(stream_finish_kernel, dim3((unsigned)(l.n * c.Hkv), blocks), dim3(kFinishThreads), 0, stream,
                               a, c.D);
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::AttnStream, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
