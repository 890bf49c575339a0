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
// account_stats_kernel: (m, l) of every row.  A workgroup has 128 rows, 32 per wave
// in registers, and a chunk of the keys, whose tiles of 64 pass through LDS (DMA,
// two buffers).  S^T = K Q^T on v_mfma_f32_16x16x32_f16 as in the prefill kernel: a
// lane has 16 keys of its row column per tile.
// account_sum_kernel: a workgroup has 256 keys, 64 per wave in registers, and
// passes all rows that see them through LDS, 64 at a time; a lane adds its row
// column's weights to 16 keys' sums, and the 16 columns are added at the end.
// No atomics: every sum has one order.
#include "account.h"

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

constexpr int   kThreads = 256;
constexpr int   kVmcnt0 = 0x0F70; // s_waitcnt vmcnt(0)
constexpr int   kTile = kStreamTile;
constexpr int   kQRows = 64;      // rows that account_sum_kernel stages

struct AccountArgs {
    const __half *q;
    const float  *w_in;
    float        *w_out;
    float        *stats; // [(stat0 * Hkv + (chunk * Hkv + g) * rows + r)][2]
    KvView        kv;
    int64_t       room;
    float         scale_log2;
    int           Hq, Hkv, G, n;
    AccountEntry  e[kAccountBatch];
};
static_assert(sizeof(AccountArgs) <= 4096, "kernel arguments");

// The last entry whose first item is at most `item`.
#define ACCOUNT_ENTRY_OF(a, field, item, out)                                                                          \
    do {                                                                                                               \
        int seen_ = 0;                                                                                                 \
        for (int k_ = 0; k_ < (a).n; k_ += 64) {                                                                       \
            const int i_ = k_ + (int)(threadIdx.x & 63);                                                               \
            seen_ += __popcll(__ballot(i_ < (a).n && (a).e[min(i_, (a).n - 1)].field <= (item)));                      \
        }                                                                                                              \
        out = __builtin_amdgcn_readfirstlane(seen_ - 1);                                                               \
    } while (0)

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
    int       ei;
    ACCOUNT_ENTRY_OF(a, item0, item, ei);
    const int row = a.e[ei].row, p0 = a.e[ei].p0, n = a.e[ei].n, w = a.e[ei].w, nch = a.e[ei].nch;
    const int rel = item - a.e[ei].item0, ch = rel % nch, rt = rel / nch;
    const int rows = w * a.G;
    const int r_lo = rt * kAccountRows, r_hi = min(rows, r_lo + kAccountRows);
    const int first = p0 + n - w;                          // position of query row 0's token
    const int kend = first + (r_hi - 1) / a.G + 1;         // keys that some row of the tile sees
    const int tiles = (p0 + n + kTile - 1) / kTile;        // of the whole, so that chunks agree
    const int t_lo = (int)((int64_t)ch * tiles / nch);
    const int t_hi = min((int)((int64_t)(ch + 1) * tiles / nch), (kend + kTile - 1) / kTile);
    const int c = lane & 15, qg = lane >> 4;

    f16x8 qb[2][KS];
    int   pos[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int     r = min(r_lo + wave * 32 + j * 16 + c, rows - 1);
        const __half *qp = a.q + ((int64_t)(a.e[ei].tok0 + n - w + r / a.G) * a.Hq + g * a.G + r % a.G) * D;
        pos[j] = first + r / a.G;
#pragma unroll
        for (int s = 0; s < KS; ++s) qb[j][s] = *reinterpret_cast<const f16x8 *>(qp + 32 * s + 8 * qg);
    }
    const char *kb = reinterpret_cast<const char *>(a.kv.k_base) + (int64_t)g * a.kv.head_stride * 2;
    auto issue = [&](int kt, uint16_t *dst) {
#pragma unroll
        for (int u = 0; u < NKI; ++u) {
            const int sl = u * kThreads + (int)threadIdx.x;
            const int r = sl / KP, x = (sl % KP) ^ swz<KP>(r);
            const int t = min(kt * kTile + r, kend - 1);
            lds_dma(kb + key_off<PAGED>(a.kv, row, t) + 16 * x, dst + (u * kThreads + wave * 64) * 8);
        }
    };
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    auto  step = [&](int kt, const uint16_t *kd, uint16_t *kn) __attribute__((always_inline)) {
        if (kt + 1 < t_hi) issue(kt + 1, kn);
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
            float mloc = -INFINITY;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[j][tt][i] = tb + 16 * tt + i <= pos[j] ? s[j][tt][i] * a.scale_log2 : -INFINITY;
                    mloc = fmaxf(mloc, s[j][tt][i]);
                }
            // (each lane its own reference point: its keys are its own until the end)
            const float m_new = fmaxf(m[j], mloc);
            float       sum = m[j] == -INFINITY ? 0.0f : l[j] * __builtin_amdgcn_exp2f(m[j] - m_new);
            if (m_new != -INFINITY) {
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f(s[j][tt][i] - m_new);
            }
            l[j] = sum;
            m[j] = m_new;
        }
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __syncthreads();
    };
    if (t_lo < t_hi) {
        issue(t_lo, ks0);
        __builtin_amdgcn_s_waitcnt(kVmcnt0);
        __syncthreads();
        for (int kt = t_lo; kt < t_hi; kt += 2) {
            step(kt, ks0, ks1);
            if (kt + 1 < t_hi) step(kt + 1, ks1, ks0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float mr = fmaxf(m[j], __shfl_xor(m[j], 16));
        mr = fmaxf(mr, __shfl_xor(mr, 32));
        float lr = m[j] == -INFINITY ? 0.0f : l[j] * __builtin_amdgcn_exp2f(m[j] - mr);
        lr += __shfl_xor(lr, 16);
        lr += __shfl_xor(lr, 32);
        const int r = r_lo + wave * 32 + j * 16 + c;
        if (qg == 0 && r < r_hi) {
            const int64_t at = (int64_t)a.e[ei].stat0 * a.Hkv + ((int64_t)ch * a.Hkv + g) * rows + r;
            *reinterpret_cast<float2 *>(a.stats + 2 * at) = make_float2(mr, lr);
        }
    }
}

template <int D, bool PAGED>
__global__ __launch_bounds__(kThreads, D <= 128 ? 2 : 1) void account_sum_kernel(AccountArgs a) {
    constexpr int KS = D / 32, KP = D / 8;
    constexpr int NQI = kQRows * KP / kThreads; // Q pieces per thread
    __shared__ __align__(16) uint16_t qs[kQRows * D];
    __shared__ float s_m[kQRows], s_inv[kQRows];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    ACCOUNT_ENTRY_OF(a, sum0, item, ei);
    const int row = a.e[ei].row, p0 = a.e[ei].p0, n = a.e[ei].n, w = a.e[ei].w, nch = a.e[ei].nch;
    const int k_lo = (item - a.e[ei].sum0) * kAccountKeys, keys = p0 + n;
    const int rows = w * a.G, first = keys - w;
    const int c = lane & 15, qg = lane >> 4;
    const int wk = k_lo + wave * 64; // the wave's first key

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
    // Rows from the first whose token sees the workgroup's first key.
    const int r_from = max(0, k_lo - first) * a.G / kQRows * kQRows;
    for (int r0 = r_from; r0 < rows; r0 += kQRows) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NQI; ++u) {
            const int sl = u * kThreads + (int)threadIdx.x, r = sl / KP, x = sl % KP;
            const int qr = min(r0 + r, rows - 1);
            const __half *qp = a.q + ((int64_t)(a.e[ei].tok0 + n - w + qr / a.G) * a.Hq + g * a.G + qr % a.G) * D;
            *reinterpret_cast<uint4 *>(&qs[(r * KP + (x ^ swz<KP>(r))) * 8]) = *reinterpret_cast<const uint4 *>(qp + 8 * x);
        }
        if ((int)threadIdx.x < kQRows) { // the row's maximum and sum over its chunks
            const int r = r0 + (int)threadIdx.x;
            float     m = INFINITY, l = 1.0f; // a row past the end: weights of 0
            if (r < rows) {
                const float  *st = a.stats + 2 * ((int64_t)a.e[ei].stat0 * a.Hkv + (int64_t)g * rows + r);
                const int64_t step = 2 * (int64_t)a.Hkv * rows;
                m = -INFINITY;
                for (int ch = 0; ch < nch; ++ch) m = fmaxf(m, st[ch * step]);
                l = 0.0f;
                for (int ch = 0; ch < nch; ++ch) l = fmaf(st[ch * step + 1], __builtin_amdgcn_exp2f(st[ch * step] - m), l);
            }
            s_m[threadIdx.x] = m;
            s_inv[threadIdx.x] = 1.0f / l;
        }
        __syncthreads();
#pragma unroll
        for (int rg = 0; rg < kQRows / 16; ++rg) {
            const int   rr = 16 * rg + c;
            const float m = s_m[rr], inv = s_inv[rr];
            const int   pos = first + min(r0 + rr, rows - 1) / a.G;
            f32x4       s[4];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const f16x8 qf = *reinterpret_cast<const f16x8 *>(&qs[(rr * KP + ((4 * k + qg) ^ swz<KP>(rr))) * 8]);
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) s[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[tt][k], qf, s[tt], 0, 0, 0);
            }
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(s[tt][i] * a.scale_log2 - m) * inv;
                    acc[tt][i] += wk + 16 * tt + 4 * qg + i <= pos ? p : 0.0f;
                }
        }
    }
    const int64_t base = ((int64_t)row * a.Hkv + g) * a.room;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = acc[tt][i];
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o);
            const int t = wk + 16 * tt + 4 * qg + i;
            if (c == 0 && t < keys) a.w_out[base + t] = (a.w_in && t < p0 ? a.w_in[base + t] : 0.0f) + v;
        }
}

template <int D> void launch_d(const AccountArgs &a, const AccountLaunch &l, bool paged, hipStream_t stream) {
    const dim3 stats((unsigned)l.items * (unsigned)a.Hkv), sums((unsigned)l.sums * (unsigned)a.Hkv), block(kThreads);
    if (paged) {
        hipLaunchKernelGGL((account_stats_kernel<D, true>), stats, block, 0, stream, a);
        hipLaunchKernelGGL((account_sum_kernel<D, true>), sums, block, 0, stream, a);
    } else {
        hipLaunchKernelGGL((account_stats_kernel<D, false>), stats, block, 0, stream, a);
        hipLaunchKernelGGL((account_sum_kernel<D, false>), sums, block, 0, stream, a);
    }
    HIP_CHECK(hipGetLastError());
}

} // namespace

size_t account_workspace_floats(const AccountPlan &plan, int Hkv) {
    int64_t most = 0;
    for (const auto &l : plan.launches) most = std::max(most, l.stats);
    return 2 * (size_t)most * (size_t)Hkv;
}

void launch_account(const AccountCall &c, const KvView &kv, const AccountPlan &plan, float *workspace,
                    hipStream_t stream) {
    AccountArgs a;
    a.q = c.q;
    a.w_in = c.w_in;
    a.w_out = c.w_out;
    a.stats = workspace;
    a.kv = kv;
    a.room = c.room;
    a.scale_log2 = c.scale * 1.4426950408889634f;
    a.Hq = c.Hq;
    a.Hkv = c.Hkv;
    a.G = c.Hq / c.Hkv;
    const bool paged = kv.block_table != nullptr;
    for (const auto &l : plan.launches) {
        if (l.n == 0 || l.items == 0) continue;
        if ((int64_t)std::max(l.items, l.sums) * c.Hkv > INT32_MAX)
            throw std::invalid_argument("attention account: too many work items");
        a.n = l.n;
        std::memcpy(a.e, plan.entries.data() + l.first, sizeof(AccountEntry) * (size_t)l.n);
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
