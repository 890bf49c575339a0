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
// second time for it would cost half of the whole; the scores cost 4 bytes a row and token
// written and read (group 4, D 128: 32 against 512 bytes), so they go through the
// workspace.  They and the sums are fp32: an account is compared with others of
// like size.
//
// attn_stream_kernel: a workgroup of 4 waves per (entry, chunk of tiles, kv head);
// wave w takes every fourth tile of 64 tokens (32 at head_dim 256) and keeps its own
// running maximum, sum and output; the next tile's rows are on their way while
// one is computed.
//   S^T = K Q^T      v_mfma_f32_16x16x32_f16: A = K rows (token l%16, dims
//                    8(l/16)..+7) straight from memory, B = Q (row l%16),
//                    D = S^T (tokens 4(l/16)+i, row l%16)
//   softmax          per row column in the log2 domain; the reference point
//                    moves on jumps above 2^8 only, p is at most 2^8 (fp16 for the
//                    product, a relative rounding of 2^-11 per weight; its sum
//                    stays fp32)
//   O^T += V^T P^T   over 32 tokens; V^T from the wave's row-major LDS stage by
//                    the transposing ds_read_b64_tr_b16
// stream_finish_kernel: merges the chunks' outputs and turns scores into the account.
#include "stream.h"

#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <stdexcept>

namespace tiny_llm {
namespace detail {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float    f32x4 __attribute__((ext_vector_type(4)));
typedef short    s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int   kWaves = 4;
constexpr float kLazyMax = 8.0f;

struct StreamArgs {
    const __half *q;
    __half       *out;
    const __half *new_k, *new_v;
    const float  *w_in;
    float        *w_out;
    float        *part_o;  // [item][Hkv][16 rows at most][D]
    float        *part_ml; // [item][Hkv][rows][2]
    float        *scores;  // [tile0 * Hkv + g * tiles][rows][tiles * 64]
    KvView        kv;
    int64_t       room;
    int           fresh;
    float         scale_log2;
    int           Hq, Hkv, G, n, chunk, entry0, rows; // rows: of the partials, nq * G at most
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

template <int D, bool PAGED, bool SCORES>
__global__ __launch_bounds__(kWaves * 64, D <= 128 ? 2 : 1) void attn_stream_kernel(StreamArgs a) {
    constexpr int TK = D <= 128 ? 64 : 32; // tokens of a wave's step
    constexpr int SUB = kStreamTile / TK;  // steps per tile
    constexpr int TT = TK / 16;
    constexpr int KS = D / 32, DT = D / 16, KP = D / 8;
    constexpr int NV = TK * KP / 64;       // V pieces per lane
    constexpr int RPI = 64 / KP;           // V rows per load instruction
    constexpr int STAGE = TK * D > 16 * D * 2 ? TK * D : 16 * D * 2; // halves: V rows, then o[16][D] fp32
    __shared__ __align__(16) uint16_t stage[kWaves][STAGE];
    __shared__ float sm[kWaves][16], sl[kWaves][16];
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
    auto token_off = [&](int t) -> int64_t {
        if constexpr (PAGED) return (int64_t)bt[t >> a.kv.log2_blk] * blk_bytes + (int64_t)(t & mask) * tokb;
        else return (int64_t)row * blk_bytes + (int64_t)t * tokb;
    };

    if (a.new_k && ch == nch - 1) { // the new token's row, then read like any other
        if ((int)threadIdx.x < 2 * KP) {
            const int     which = threadIdx.x / KP, x = threadIdx.x - which * KP;
            const __half *src = (which ? a.new_v : a.new_k) + ((int64_t)(a.entry0 + ei) * a.Hkv + g) * D + 8 * x;
            char         *dst = const_cast<char *>(which ? vb : kb) + token_off(S - 1) + 16 * x;
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
    float m_run = -INFINITY, l_run = 0.0f;

    // Offset of the 16 tokens from t on, and how many of them may be read past the first.
    auto quarter = [&](int t, int &more) -> int64_t {
        const int tq = min(t, last);
        more = min(15, last - tq);
        return token_off(tq);
    };
    f16x8 kf[TT][KS];
    u32x4 vr[NV];
    auto load_k = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            int            more;
            const char    *p = kb + quarter(t0 + 16 * tt, more);
            const uint32_t off = (uint32_t)min(c, more) * (uint32_t)tokb + 16 * qg;
#pragma unroll
            for (int s = 0; s < KS; ++s) kf[tt][s] = *reinterpret_cast<const f16x8 *>(p + off + 64 * s);
        }
    };
    auto load_v = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int      r = (u * RPI) % 16 + lane / KP; // in its quarter
            int            more;
            const char    *p = vb + quarter(t0 + u * RPI / 16 * 16, more);
            const uint32_t off = (uint32_t)min(r, more) * (uint32_t)tokb + 16 * (lane % KP);
            vr[u] = *reinterpret_cast<const u32x4 *>(p + off);
        }
    };
    uint16_t *vst = stage[wave];
    const int vrow = 4 * qg + (c >> 2);
    const int vxor = ((c & 3) >> 1) ^ swz(vrow);
    const int vlane = vrow * KP * 8 + 4 * (c & 1);
    auto vt_read = [&](int r0, int dt) __attribute__((always_inline)) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr(&vst[vlane + ((2 * dt) ^ vxor) * 8 + r0 * KP * 8]));
    };
    float *srow = nullptr;
    if constexpr (SCORES)
        srow = a.scores + (((int64_t)a.e[ei].tile0 * a.Hkv + (int64_t)g * tiles) * a.rows + (int64_t)c * tiles) * kStreamTile;

    // The wave's steps: step x of the chunk's tiles, tile tile_lo + x / SUB * kWaves + wave.
    const int steps = max(0, (tile_hi - tile_lo - wave + kWaves - 1) / kWaves) * SUB;
    auto start = [&](int x) { return (tile_lo + x / SUB * kWaves + wave) * kStreamTile + x % SUB * TK; };
    if (steps > 0) {
        load_k(start(0));
        load_v(start(0));
    }
    for (int x = 0; x < steps; ++x) {
        const int t0 = start(x);
        f32x4     s[TT];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tt][k], qb[k], s[tt], 0, 0, 0);
        }
        if (x + 1 < steps) load_k(start(x + 1));
        const int tb = t0 + 4 * qg;
        float     mloc = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float v = s[tt][i] * a.scale_log2;
                s[tt][i] = tb + 16 * tt + i <= last ? v : -INFINITY;
                mloc = fmaxf(mloc, s[tt][i]);
            }
        if constexpr (SCORES) {
            if (c < rows)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
                    *reinterpret_cast<f32x4 *>(srow + tb + 16 * tt) = s[tt];
        }
        if (__any(mloc > m_run + kLazyMax)) {
            mloc = fmaxf(mloc, __shfl_xor(mloc, 16));
            mloc = fmaxf(mloc, __shfl_xor(mloc, 32));
            const float m_new = fmaxf(m_run, mloc);
            const float alpha = m_run == m_new ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
            l_run *= alpha;
            m_run = m_new;
        }
        f16x8 pf[TT / 2];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = s[tt][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s[tt][i] - m_run);
                l_run += p;
                pf[tt >> 1][4 * (tt & 1) + i] = (_Float16)p;
            }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int r = u * RPI + lane / KP;
            *reinterpret_cast<u32x4 *>(&vst[(r * KP + ((lane % KP) ^ swz(r))) * 8]) = vr[u];
        }
        if (x + 1 < steps) load_v(start(x + 1));
        wave_sync_lds();
#pragma unroll
        for (int tp = 0; tp < TT / 2; ++tp)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint2 v0 = __builtin_bit_cast(uint2, vt_read(32 * tp, dt));
                const uint2 v1 = __builtin_bit_cast(uint2, vt_read(32 * tp + 16, dt));
                const f16x8 vf = __builtin_bit_cast(f16x8, make_uint4(v0.x, v0.y, v1.x, v1.y));
                acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[tp], acc[dt], 0, 0, 0);
            }
        wave_sync_lds(); // the stage is rewritten by the next step
    }

    // The waves' (m, l, o) through LDS.
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    float *so = reinterpret_cast<float *>(vst);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4 *>(so + c * D + 16 * dt + 4 * qg) = acc[dt];
    if (qg == 0) {
        sm[wave][c] = m_run;
        sl[wave][c] = l_run;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < rows * D; idx += kWaves * 64) {
        const int r = idx / D, d = idx - r * D;
        float     m = sm[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sm[w][r]);
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float wgt = sm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][r] - m);
            o = fmaf(wgt, reinterpret_cast<const float *>(stage[w])[idx], o);
            l = fmaf(wgt, sl[w][r], l);
        }
        const int64_t pr = ((int64_t)item * a.Hkv + g) * a.rows + r;
        if (nch == 1) {
            a.out[((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D + d] = __float2half(o * (1.0f / (l + 1e-6f)));
        } else {
            a.part_o[pr * D + d] = o;
        }
        if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + pr * 2) = make_float2(m, l);
    }
}

constexpr int kFinishThreads = 256;
constexpr int kFinishTokens = 1024; // tokens of a workgroup

// Workgroup (entry, kv head, block of tokens): the rows' maxima and sums over the
// entry's chunks, the account of the block's tokens, and in block 0 the
// outputs of an entry with several chunks (or none: zeros).
__global__ __launch_bounds__(kFinishThreads) void stream_finish_kernel(StreamArgs a, int D) {
    __shared__ float s_m[kStreamRows], s_l[kStreamRows], s_inv[kStreamRows];
    const int ei = blockIdx.x / a.Hkv, g = blockIdx.x - ei * a.Hkv;
    const int row = a.e[ei].row, S = a.e[ei].S, tok0 = a.e[ei].tok0, rows = a.e[ei].nq * a.G;
    const int tiles = (S + kStreamTile - 1) / kStreamTile;
    const int nch = (tiles + a.chunk - 1) / a.chunk;
    const int t_lo = blockIdx.y * kFinishTokens, t_hi = min(S, t_lo + kFinishTokens);
    const bool merge = blockIdx.y == 0 && nch != 1;
    if (t_lo >= t_hi && !merge) return;
    const int64_t p0 = ((int64_t)a.e[ei].item0 * a.Hkv + g) * a.rows; // row 0 of chunk 0
    const int64_t pc = (int64_t)a.Hkv * a.rows;                      // from chunk to chunk
    const int     lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r < rows; r += kFinishThreads / 64) {
        float m = -INFINITY, l = 0.0f;
        for (int ch = lane; ch < nch; ch += 64) m = fmaxf(m, a.part_ml[(p0 + ch * pc + r) * 2]);
        for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        for (int ch = lane; ch < nch; ch += 64) {
            const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + (p0 + ch * pc + r) * 2);
            l = fmaf(ml.y, __builtin_amdgcn_exp2f(ml.x - m), l);
        }
        for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
        if (lane == 0) {
            s_m[r] = m;
            s_l[r] = l;
            s_inv[r] = 1.0f / l;
        }
    }
    __syncthreads();
    if (a.w_out) {
        const float  *sc = a.scores + ((int64_t)a.e[ei].tile0 * a.Hkv + (int64_t)g * tiles) * a.rows * kStreamTile;
        const int64_t base = ((int64_t)row * a.Hkv + g) * a.room;
        for (int t = t_lo + (int)threadIdx.x; t < t_hi; t += kFinishThreads) {
            float w = 0.0f;
            for (int r = 0; r < rows; ++r)
                w = fmaf(__builtin_amdgcn_exp2f(sc[(int64_t)r * tiles * kStreamTile + t] - s_m[r]), s_inv[r], w);
            if (a.w_in && t < S - a.fresh) w += a.w_in[base + t];
            a.w_out[base + t] = w;
        }
    }
    if (!merge) return;
    for (int idx = threadIdx.x; idx < rows * D; idx += kFinishThreads) {
        const int r = idx / D, d = idx - r * D;
        float     o = 0.0f;
        for (int ch = 0; ch < nch; ++ch) {
            const int64_t pr = p0 + ch * pc + r;
            o = fmaf(a.part_o[pr * D + d], __builtin_amdgcn_exp2f(a.part_ml[pr * 2] - s_m[r]), o);
        }
        a.out[((int64_t)(tok0 + r / a.G) * a.Hq + g * a.G + r % a.G) * D + d] =
            __float2half(nch ? o * (1.0f / (s_l[r] + 1e-6f)) : 0.0f);
    }
}

template <int D> void launch_d(const StreamArgs &a, int items, bool paged, bool scores, hipStream_t stream) {
    const dim3 grid((unsigned)items * (unsigned)a.Hkv), block(kWaves * 64);
    if (paged) {
        if (scores) hipLaunchKernelGGL((attn_stream_kernel<D, true, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((attn_stream_kernel<D, true, false>), grid, block, 0, stream, a);
    } else {
        if (scores) hipLaunchKernelGGL((attn_stream_kernel<D, false, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((attn_stream_kernel<D, false, false>), grid, block, 0, stream, a);
    }
}

int plan_rows(const StreamPlan &plan, int first, int n, int G) {
    int nq = 1;
    for (int i = first; i < first + n; ++i) nq = std::max(nq, (int)plan.entries[(size_t)i].nq);
    return nq * G;
}

} // namespace

size_t stream_workspace_floats(const StreamPlan &plan, int Hq, int Hkv, int D, bool account) {
    size_t most = 0;
    for (const auto &l : plan.launches) {
        const size_t rows = (size_t)plan_rows(plan, l.first, l.n, Hq / Hkv) * Hkv;
        size_t       f = (size_t)l.items * rows * (size_t)(D + 2);
        if (account) f += (size_t)l.tiles * kStreamTile * rows;
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
        a.entry0 = l.first;
        a.rows = plan_rows(plan, l.first, l.n, a.G);
        if (a.rows > kStreamRows) throw std::invalid_argument("attention: too many query rows per entry");
        if ((int64_t)l.items * c.Hkv > INT32_MAX) throw std::invalid_argument("attention: too many work items");
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(StreamEntry) * (size_t)l.n);
        a.scores = workspace;
        a.part_ml = workspace + (c.w_out ? (size_t)l.tiles * kStreamTile * a.rows * c.Hkv : 0);
        a.part_o = a.part_ml + (size_t)l.items * c.Hkv * a.rows * 2;
        profile_begin(KernelId::AttnStream, stream);
        if (l.items > 0) {
            switch (c.D) {
            case 32: launch_d<32>(a, l.items, paged, c.w_out != nullptr, stream); break;
            case 64: launch_d<64>(a, l.items, paged, c.w_out != nullptr, stream); break;
            case 128: launch_d<128>(a, l.items, paged, c.w_out != nullptr, stream); break;
            case 256: launch_d<256>(a, l.items, paged, c.w_out != nullptr, stream); break;
            default: throw std::invalid_argument("attention: unsupported head_dim");
            }
            HIP_CHECK(hipGetLastError());
        }
        bool none = false;
        for (int i = l.first; i < l.first + l.n; ++i) none |= plan.entries[(size_t)i].S == 0;
        if (c.w_out || none || l.max_items > 1) {
            const unsigned blocks = c.w_out ? (unsigned)std::max(1, (l.max_len + kFinishTokens - 1) / kFinishTokens) : 1u;
            hipLaunchKernelGGL(stream_finish_kernel, dim3((unsigned)(l.n * c.Hkv), blocks), dim3(kFinishThreads), 0, stream,
                               a, c.D);
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::AttnStream, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
