// Eviction from the cache by accumulated attention weight, for gfx950.
//
// Per sequence and kv head, of n tokens with accounts w_t and positions p_t the
// `keep` first in the order
//   (newest: p_t >= n + gone - recent) before (the rest, by falling w_t),
// equal ones by rising t, stay.  The cache row keeps its first `keep` places:
// the i-th place there that became free (rising) takes the i-th kept token from
// behind them (rising), so only those tokens move -- a stable compaction would
// move every token behind the first free place -- and no place is read and
// written by the same launch.  Attention does not depend on the order of cached
// keys; the positions are kept beside the accounts.
//
// evict_select_kernel: one workgroup per (sequence, kv head).  The account's
// bits, mapped so that unsigned order is the floats' order, go through a radix
// selection of 11 + 11 + 10 bits: a histogram in LDS, the bin in which the
// keep-th largest lies, the next digit within that bin.  Then one pass in index
// order ranks the free places and the movers, writes their pairs, and brings
// accounts and positions up to date.
// evict_move_kernel: the K and V rows of the pairs, 16 bytes a lane.
#include "evict.h"

#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

namespace tiny_llm {
namespace detail {

namespace {

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;      // 11 bits of the key
constexpr int kMoveThreads = 256;
constexpr int kMovePairs = 32;   // pairs of a workgroup of evict_move_kernel
constexpr uint32_t kNewest = 0xFFFFFFFFu; // above every account's key

struct EvictArgs {
    KvView     kv;
    EvictState st;
    int32_t   *pairs; // (from, to) of the entries' lists, then their lengths
    int32_t   *counts;
    int        recent, Hkv, D, n;
    EvictEntry e[kEvictBatch];
};
static_assert(sizeof(EvictArgs) <= 4096, "kernel arguments");

// Unsigned order of the keys = order of the accounts; NaN counts as the smallest,
// the two zeros are equal.
__device__ __forceinline__ uint32_t account_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// Sum over the workgroup of each thread's v; every thread gets it.
template <int NT> __device__ __forceinline__ uint32_t block_sum(uint32_t v, uint32_t *lds) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t s = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += lds[w];
    return s;
}

// Number of set flags in the threads before this one; `total`: in the workgroup.
template <int NT> __device__ __forceinline__ uint32_t block_rank(bool flag, uint32_t *lds, uint32_t &total) {
    const uint64_t b = __ballot(flag);
    const int      lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 0) lds[wave] = __popcll(b);
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const uint32_t c = lds[w];
        before += w < wave ? c : 0u;
        total += c;
    }
    return before + __popcll(b & ((1ull << lane) - 1ull));
}

template <int NT> __global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t lds[NT / 64];
    __shared__ uint32_t pick[3];
    const int        tid = threadIdx.x;
    const int        ei = blockIdx.x / a.Hkv, g = blockIdx.x - ei * a.Hkv;
    const EvictEntry e = a.e[ei];
    const int64_t    base = ((int64_t)e.row * a.Hkv + g) * a.st.room;
    const float     *w_in = a.st.w_in + base;
    const int32_t   *p_in = a.st.pos_in + base;
    float           *w_out = a.st.w_out + base;
    int32_t         *p_out = a.st.pos_out + base;
    const int        newest = e.len + e.gone - a.recent; // positions from here on stay
    auto position = [&](int i) { return i < e.base ? p_in[i] : i + e.gone; };
    auto key_of = [&](int i) { return position(i) >= newest ? kNewest : account_key(w_in[i]); };
    const int cap = min(e.len - e.keep, e.keep);
    int2     *pairs = reinterpret_cast<int2 *>(a.pairs) + (int64_t)e.list * a.Hkv + (int64_t)g * cap;

    // The threshold: the key of the keep-th token, and how many tokens with it stay.
    uint32_t thr = 0u, need = (uint32_t)e.keep, equal = 0u;
    if (e.keep < e.len) {
        uint32_t mine = 0;
        for (int i = tid; i < e.len; i += NT) mine += key_of(i) == kNewest;
        const uint32_t held = block_sum<NT>(mine, lds);
        if (held >= need) {
            thr = kNewest;
            equal = held;
        } else {
            need -= held;
            int shift = 32;
            for (int pass = 0; pass < 3; ++pass) {
                const int bits = pass < 2 ? 11 : 10, lo = shift - bits;
                for (int b = tid; b < kBins; b += NT) hist[b] = 0u;
                __syncthreads();
                for (int i = tid; i < e.len; i += NT) {
                    const uint32_t k = key_of(i);
                    if (k != kNewest && (shift == 32 || (k >> shift) == (thr >> shift)))
                        atomicAdd(&hist[(k >> lo) & ((1u << bits) - 1u)], 1u);
                }
                __syncthreads();
                // Bins from the top: thread t sums bins kBins-1 - t*P .. - P + 1.
                constexpr int P = kBins / NT;
                uint32_t      own = 0;
#pragma unroll
                for (int u = 0; u < P; ++u) own += hist[kBins - 1 - (tid * P + u)];
                uint32_t       inc = own; // inclusive over the wave
                const int      lane = tid & 63, wave = tid >> 6;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t v = __shfl_up(inc, o);
                    inc += lane >= o ? v : 0u;
                }
                if (lane == 63) lds[wave] = inc;
                __syncthreads();
                uint32_t above = inc - own;
                for (int w = 0; w < wave; ++w) above += lds[w];
#pragma unroll
                for (int u = 0; u < P; ++u) {
                    const int      b = kBins - 1 - (tid * P + u);
                    const uint32_t c = hist[b];
                    if (above < need && need <= above + c) { // one bin
                        pick[0] = (uint32_t)b;
                        pick[1] = need - above;
                        pick[2] = c;
                    }
                    above += c;
                }
                __syncthreads();
                thr |= pick[0] << lo;
                need = pick[1];
                equal = pick[2];
                shift = lo;
                __syncthreads();
            }
        }
    }

    // In index order: which stay, the free places and the movers.
    uint32_t ties = 0, done = 0; // so far: tokens at the threshold, free places and movers
    uint32_t free_places = 0;
    for (int i0 = 0; i0 < e.len; i0 += NT) {
        const int      i = i0 + tid;
        const bool     in = i < e.len;
        const uint32_t k = in ? key_of(i) : 0u;
        bool           stays = in && (e.keep == e.len || k > thr);
        if (e.keep < e.len) {
            const bool at = in && k == thr;
            if (equal == need) {
                stays |= at;
            } else {
                uint32_t       total;
                const uint32_t r = block_rank<NT>(at, lds, total);
                stays |= at && ties + r < need;
                ties += total;
            }
            const bool     flag = in && (i < e.keep ? !stays : stays);
            uint32_t       total;
            const uint32_t r = done + block_rank<NT>(flag, lds, total);
            // Free places come first in index order, as many as movers.
            const uint32_t nf = block_sum<NT>(flag && i < e.keep, lds);
            free_places += nf;
            if (flag && i < e.keep && r < (uint32_t)cap) pairs[r].y = i;
            if (flag && i >= e.keep && r - free_places < (uint32_t)cap) pairs[r - free_places].x = i;
            done += total;
        }
        if (in && i < e.keep && stays) {
            if (w_out != w_in) w_out[i] = w_in[i];
            if (p_out != p_in || i >= e.base) p_out[i] = position(i);
        }
    }
    if (e.keep == e.len) return;
    if (tid == 0) a.counts[(int64_t)ei * a.Hkv + g] = (int32_t)free_places;
    __threadfence_block();
    __syncthreads();
    for (uint32_t r = tid; r < free_places; r += NT) {
        const int2 p = pairs[r];
        w_out[p.y] = w_in[p.x];
        p_out[p.y] = position(p.x);
    }
}

__device__ __forceinline__ int64_t row_off(const KvView &v, int row, int t) {
    if (v.block_table) {
        const int blk = v.block_table[(int64_t)row * v.bt_stride + (t >> v.log2_blk)];
        return (int64_t)blk * v.blk_stride + (int64_t)(t & ((1 << v.log2_blk) - 1)) * v.tok_stride;
    }
    return (int64_t)row * v.blk_stride + (int64_t)t * v.tok_stride;
}

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
    const int        ei = blockIdx.x / a.Hkv, g = blockIdx.x - ei * a.Hkv;
    const EvictEntry e = a.e[ei];
    const int        cap = min(e.len - e.keep, e.keep);
    const int        first = blockIdx.y * kMovePairs;
    if (first >= cap) return; // (before the count: none of the entry's workgroups behind its list reads it)
    const int   cnt = a.counts[(int64_t)ei * a.Hkv + g];
    const int2 *pairs = reinterpret_cast<const int2 *>(a.pairs) + (int64_t)e.list * a.Hkv + (int64_t)g * cap;
    const int   pieces = a.D / 8;
    const int   last = min(first + kMovePairs, cnt);
    for (int x = threadIdx.x; x < (last - first) * 2 * pieces; x += kMoveThreads) {
        const int     piece = x % pieces, which = x / pieces & 1;
        const int2    p = pairs[first + x / (2 * pieces)];
        __half       *b = const_cast<__half *>(which ? a.kv.v_base : a.kv.k_base) + (int64_t)g * a.kv.head_stride + 8 * piece;
        const uint4   v = *reinterpret_cast<const uint4 *>(b + row_off(a.kv, e.row, p.x));
        *reinterpret_cast<uint4 *>(b + row_off(a.kv, e.row, p.y)) = v;
    }
}

} // namespace

size_t evict_workspace_words(std::vector<EvictEntry> &entries, int Hkv) {
    int64_t pairs = 0;
    for (auto &e : entries) {
        e.list = (int32_t)pairs;
        pairs += std::min(e.len - e.keep, e.keep);
    }
    return 2 * (size_t)pairs * Hkv + entries.size() * (size_t)Hkv;
}

void launch_evict(const KvView &kv, const std::vector<EvictEntry> &entries, const EvictState &st, int recent, int Hkv,
                  int D, int32_t *workspace, hipStream_t stream) {
    const bool copies = st.w_in != st.w_out || st.pos_in != st.pos_out;
    int64_t    pairs = 0;
    for (const auto &e : entries) pairs += std::min(e.len - e.keep, e.keep);
    EvictArgs a;
    a.kv = kv;
    a.st = st;
    a.pairs = workspace;
    a.recent = recent;
    a.Hkv = Hkv;
    a.D = D;
    size_t launched = 0;
    for (size_t i = 0; i < entries.size();) {
        a.n = 0;
        int cap = 0;
        a.counts = workspace + 2 * pairs * Hkv + (int64_t)launched * Hkv;
        for (; i < entries.size() && a.n < kEvictBatch; ++i) {
            const EvictEntry &e = entries[i];
            if (e.keep == e.len && !copies) continue; // all stays, where it is
            a.e[a.n++] = e;
            cap = std::max(cap, std::min(e.len - e.keep, e.keep));
        }
        if (a.n == 0) break;
        launched += (size_t)a.n;
        profile_begin(KernelId::Evict, stream);
        hipLaunchKernelGGL((evict_select_kernel<kSelThreads>), dim3((unsigned)(a.n * Hkv)), dim3(kSelThreads), 0, stream, a);
        HIP_CHECK(hipGetLastError());
        if (cap > 0) {
            const dim3 grid((unsigned)(a.n * Hkv), (unsigned)((cap + kMovePairs - 1) / kMovePairs));
            hipLaunchKernelGGL(evict_move_kernel, grid, dim3(kMoveThreads), 0, stream, a);
            HIP_CHECK(hipGetLastError());
        }
        profile_end(KernelId::Evict, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
