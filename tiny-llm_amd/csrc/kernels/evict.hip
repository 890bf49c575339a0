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
// evict_move_kernel: the K and V rows of the pairs, 16 bytes a lane, every row on
// its way before the first is written: 8 x 8192 tokens to 2048 (8 heads of 128,
// 100 MB read and written) 17 us.
// evict_select_any_kernel: more than 32768 tokens, the limit of the registers; a
// (sequence, kv head)'s one workgroup reads its accounts anew in every pass, so it is slow:
// 131072 tokens to 16384, 8 heads of 128, 393 us with the moves.
// evict_one_kernel: sequences that lose one token, in one launch: 16 x 32 heads of
// 1025 tokens 25.5 -> 6.4 us against the two launches above.
#include "evict.h"

#include "tiny_llm/hip_utils.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>

namespace tiny_llm {
namespace detail {

namespace {

constexpr int kBins = 2048;      // 11 bits of the key
constexpr int kMoveThreads = 256;
constexpr int kMovePairs = 32;   // pairs that a workgroup of evict_move_kernel moves at once
constexpr int kMostBlocks = 32768; // grid.y
constexpr int kOneThreads = 256;
constexpr int kList = 2048;      // candidates at least that the second digit finds in a list
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

template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
// Sum over the wave's lanes up to this one (row_shr 1, 2, 4, 8, then the rows' last
// lanes to the rows behind them).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

// Four consecutive words; the rows of accounts begin at any multiple of 4 bytes.
struct __attribute__((packed, aligned(4))) Words {
    uint32_t x[4];
};
__device__ __forceinline__ Words load4(const void *p, int i, int n) { // words past the end: 0
    const uint32_t *w = static_cast<const uint32_t *>(p);
    if (i + 4 <= n) return *reinterpret_cast<const Words *>(w + i);
    Words r;
#pragma unroll
    for (int u = 0; u < 4; ++u) r.x[u] = i + u < n ? w[i + u] : 0u;
    return r;
}

// The addresses of one (sequence, kv head).
struct Head {
    EvictEntry     e;
    int            ei, g, newest;
    const float   *w_in;
    const int32_t *p_in;
    float         *w_out;
    int32_t       *p_out;
    __device__ __forceinline__ int position(int i) const { return i < e.base ? p_in[i] : i + e.gone; }
    __device__ __forceinline__ uint32_t key(int i) const { return position(i) >= newest ? kNewest : account_key(w_in[i]); }
};
#define EVICT_HEAD(a, h)                                                                                               \
    Head h;                                                                                                            \
    do {                                                                                                               \
        h.ei = blockIdx.x / (a).Hkv;                                                                                   \
        h.g = blockIdx.x - h.ei * (a).Hkv;                                                                             \
        h.e = (a).e[h.ei];                                                                                             \
        h.newest = h.e.len + h.e.gone - (a).recent; /* positions from here on stay */                                  \
        const int64_t base_ = ((int64_t)h.e.row * (a).Hkv + h.g) * (a).st.room;                                        \
        h.w_in = (a).st.w_in + base_;                                                                                  \
        h.p_in = (a).st.pos_in + base_;                                                                                \
        h.w_out = (a).st.w_out + base_;                                                                                \
        h.p_out = (a).st.pos_out + base_;                                                                              \
    } while (0)

// The bin, of kBins from the top, in which the need-th largest lies: pick = {bin, how
// many of it, its count}.  `hist` is complete (a barrier before the call); the waves'
// sums have words of their own, which no wave may still be reading here.
template <int NT> __device__ __forceinline__ void pick_bin(const uint32_t *hist, uint32_t need, uint32_t *pick) {
    constexpr int P = kBins / NT;
    __shared__ uint32_t sums[NT / 64];
    const int     tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t      c[P], own = 0;
#pragma unroll
    for (int u = 0; u < P; ++u) {
        c[u] = hist[kBins - 1 - (tid * P + u)];
        own += c[u];
    }
    const uint32_t inc = wave_scan(own);
    if (lane == 63) sums[wave] = inc;
    __syncthreads();
    uint32_t above = inc - own;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) above += w < wave ? sums[w] : 0u;
#pragma unroll
    for (int u = 0; u < P; ++u) {
        if (above < need && need <= above + c[u]) { // one bin
            pick[0] = (uint32_t)(kBins - 1 - (tid * P + u));
            pick[1] = need - above;
            pick[2] = c[u];
        }
        above += c[u];
    }
    __syncthreads();
}

// Up to NT * 4 * IT tokens, their keys in registers: thread t has tokens (it * NT + t)
// * 4 .. + 3.  Where the first digit leaves up to kList candidates, the next ones are
// found among a list of them.  Bound by the instructions of the one workgroup that
// a (sequence, kv head) has, not by memory.  Four tokens a step, with one scan per
// step, instead of one with its ballots, no token looked at again after the first
// digit, and movers from an ordered list instead of from their steps: 8192 tokens
// 14.4 -> 10.1 us, 32768 39.8 -> 20.8.  Accounts in registers beside or instead of the
// keys cost more instructions than they saved (34 us).
template <int NT, int IT> __global__ __launch_bounds__(NT) void evict_select_kernel(EvictArgs a) {
    constexpr int NW = NT / 64;
    static_assert(IT <= 8, "a bit per token");
    // Histogram and list, then the free places and behind them the movers, by index.
    constexpr int kBuf = kBins + kList > NT * IT * 2 ? kBins + kList : NT * IT * 2, kListed = kBuf - kBins;
    static_assert(NT * IT * 4 <= 1 << 16, "an index of 16 bits, two a word");
    __shared__ __align__(4) uint32_t buf[kBuf];
    uint32_t *const hist = buf, *const list = buf + kBins;
    uint16_t *const order = reinterpret_cast<uint16_t *>(buf);
    __shared__ uint32_t lds[NW];
    __shared__ uint32_t pick[3];
    __shared__ uint32_t before[IT * NW]; // flags of step it's wave w, then of those before it
    __shared__ uint32_t s_total, s_listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    EVICT_HEAD(a, h);
    const EvictEntry &e = h.e;
    const int cap = min(e.len - e.keep, e.keep);
    int2     *pairs = reinterpret_cast<int2 *>(a.pairs) + (int64_t)e.list * a.Hkv + (int64_t)h.g * cap;
    // (Computed anew at each use: kept for all steps from phase to phase, the tokens'
    // addresses pushed keys out of the registers.)
    auto token = [&](int it) __attribute__((always_inline)) {
        int t = tid;
        if (IT > 4) asm volatile("" : "+v"(t));
        return (it * NT + t) * 4;
    };

    // The keys stay in registers: 0 past the end, which is below or equal to every
    // other and last in order.
    uint32_t keys[IT][4], held = 0;
    for (int b = tid; b < kBins; b += NT) hist[b] = 0u;
    if (tid == 0) s_listed = 0;
    __syncthreads();
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const Words x = load4(h.w_in, token(it), e.len);
#pragma unroll
        for (int u = 0; u < 4; ++u) keys[it][u] = x.x[u];
    }
    if (IT > 4) __builtin_amdgcn_sched_barrier(0); // (few registers are left: no positions loaded with these)
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        const int i = token(it);
        if (i < e.len) {
            Words p = {};
            if (i < e.base) p = load4(h.p_in, i, e.base);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int pos = i + u < e.base ? (int)p.x[u] : i + u + e.gone;
                uint32_t  k = account_key(__uint_as_float(keys[it][u]));
                k = pos >= h.newest ? kNewest : k;
                k = i + u < e.len ? k : 0u;
                keys[it][u] = k;
                held += k == kNewest;
                if (k != kNewest) atomicAdd(&hist[k >> 21], 1u);
            }
        }
    }
    held = block_sum<NT>(held, lds); // (its barriers also order hist)

    // The threshold: the tokens with keys above it stay, and of the `equal` ones that
    // agree with it down to bit `shift`, `need`.
    uint32_t thr = kNewest, need = (uint32_t)e.keep, equal = held;
    int      shift = 0;
    if (held < need) {
        need -= held;
        pick_bin<NT>(hist, need, pick);
        thr = pick[0] << 21;
        need = pick[1];
        equal = pick[2];
        shift = 21;
        const bool     listed = equal <= (uint32_t)kListed;
        const uint32_t n = equal;
        if (listed && equal != need) {
#pragma unroll
            for (int it = 0; it < IT; ++it)
                if (token(it) < e.len) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (keys[it][u] - thr < 1u << 21) list[atomicAdd(&s_listed, 1u)] = keys[it][u];
                }
        }
        while (shift > 0 && equal != need) { // (all of a bin stay: no need to look into it)
            const int bits = min(11, shift), lo = shift - bits;
            __syncthreads();
            for (int b = tid; b < kBins; b += NT) hist[b] = 0u;
            __syncthreads();
            auto count = [&](uint32_t k) {
                if ((k >> shift) == (thr >> shift)) atomicAdd(&hist[(k >> lo) & ((1u << bits) - 1u)], 1u);
            };
            if (listed) {
                for (uint32_t x = tid; x < n; x += NT) count(list[x]);
            } else {
#pragma unroll
                for (int it = 0; it < IT; ++it)
                    if (token(it) < e.len) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) count(keys[it][u]);
                    }
            }
            __syncthreads();
            pick_bin<NT>(hist, need, pick);
            thr |= pick[0] << lo;
            need = pick[1];
            equal = pick[2];
            shift = lo;
        }
    }

    // Flags of all tokens -> before[]: how many precede a step's wave; s_total.
    uint32_t scan[IT]; // flags in the wave's lanes before this one
    auto     rank_all = [&](auto &&flags) __attribute__((always_inline)) {
        __syncthreads();
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const uint32_t c = __popc(flags(it)), inc = wave_scan(c);
            scan[it] = inc - c;
            if (lane == 63) before[it * NW + wave] = inc;
        }
        __syncthreads();
        if (wave == 0) {
            constexpr int N = IT * NW, P = (N + 63) / 64;
            uint32_t      c[P], own = 0;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                c[u] = lane * P + u < N ? before[lane * P + u] : 0u;
                own += c[u];
            }
            const uint32_t inc = wave_scan(own);
            uint32_t       run = inc - own;
            if (lane == 63) s_total = inc;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                if (lane * P + u < N) before[lane * P + u] = run;
                run += c[u];
            }
        }
        __syncthreads();
    };
    // (all of the bin stay, or none of it yet; not all tokens do, so thr is above 0 then)
    const uint32_t limit = equal == need ? thr - 1u : thr;
    uint32_t       stays = 0; // bit 4 it + u: token(it) + u stays
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int u = 0; u < 4; ++u) stays |= (uint32_t)(keys[it][u] > limit) << (4 * it + u);
    if (equal != need) { // the first `need` tokens at the threshold
        auto at = [&](int it) {
            uint32_t f = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) f |= (uint32_t)(keys[it][u] == thr) << u;
            return f;
        };
        rank_all(at);
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            uint32_t f = at(it);
            for (uint32_t r = before[it * NW + wave] + scan[it]; f && r < need; ++r) {
                stays |= (f & -f) << 4 * it;
                f &= f - 1;
            }
        }
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) // tokens past the end do not stay
        stays &= ~((token(it) < e.len ? ~(0xFu >> max(0, token(it) + 4 - e.len)) & 0xFu : 0xFu) << 4 * it);

    // What stays in place, and the free places and movers in index order.
    auto moving = [&](int it) { // free places below keep, kept tokens from there on
        const int      i = token(it);
        const uint32_t low = i >= e.keep ? 0u : 0xFu >> max(0, i + 4 - e.keep);
        return ((stays >> 4 * it) ^ low) & 0xFu; // below keep: those that go, behind it: those that stay
    };
    rank_all(moving);
    const uint32_t moved = s_total / 2; // as many free places as movers
    const bool     copy_w = h.w_out != h.w_in, copy_p = h.p_out != h.p_in;
    // The accounts of a step's tokens from their keys; of the newest, whose keys do
    // not hold them, from memory.
    auto accounts = [&](int it) __attribute__((always_inline)) {
        Words x;
        bool  any = false;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t k = keys[it][u];
            x.x[u] = k == 0u ? 0x7FC00000u : k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu);
            any |= k == kNewest;
        }
        if (any) x = load4(h.w_in, token(it), e.len);
        return x;
    };
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        uint32_t r = before[it * NW + wave] + scan[it];
        for (uint32_t f = moving(it); f; f &= f - 1) order[r++] = (uint16_t)(token(it) + __builtin_ctz(f));
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
        if (IT > 4) __builtin_amdgcn_sched_barrier(0);
        const int      i = token(it);
        const uint32_t f = moving(it);
        if (i >= e.keep) continue;
        Words p = {}, x = {};
        if (copy_w) x = accounts(it);
        if (copy_p && i < e.base) p = load4(h.p_in, i, e.base);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i + u >= e.keep || (f >> u & 1)) continue;
            if (copy_w) h.w_out[i + u] = __uint_as_float(x.x[u]);
            if (i + u >= e.base) h.p_out[i + u] = i + u + e.gone;
            else if (copy_p) h.p_out[i + u] = (int32_t)p.x[u];
        }
    }
    if (tid == 0) a.counts[(int64_t)h.ei * a.Hkv + h.g] = (int32_t)moved;
    __syncthreads();
    for (uint32_t r0 = tid; r0 < moved; r0 += 4 * NT) { // four on their way at once
        int     from[4];
        float   w[4];
        int32_t p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            from[u] = order[moved + min(r0 + u * NT, moved - 1)];
            w[u] = h.w_in[from[u]];
            p[u] = h.position(from[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t r = r0 + u * NT;
            if (r >= moved) break;
            const int to = order[r];
            pairs[r] = make_int2(from[u], to);
            h.w_out[to] = w[u];
            h.p_out[to] = p[u];
        }
    }
}

// The same for any number of tokens, their keys computed anew in every pass.
template <int NT> __global__ __launch_bounds__(NT) void evict_select_any_kernel(EvictArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t lds[NT / 64];
    __shared__ uint32_t pick[3];
    const int tid = threadIdx.x;
    EVICT_HEAD(a, h);
    const EvictEntry &e = h.e;
    const int cap = min(e.len - e.keep, e.keep);
    int2     *pairs = reinterpret_cast<int2 *>(a.pairs) + (int64_t)e.list * a.Hkv + (int64_t)h.g * cap;
    uint32_t  mine = 0;
    for (int i = tid; i < e.len; i += NT) mine += h.key(i) == kNewest;
    const uint32_t held = block_sum<NT>(mine, lds);
    uint32_t       thr = kNewest, need = (uint32_t)e.keep, equal = held;
    int            shift = 0;
    if (held < need) {
        need -= held;
        thr = 0u;
        shift = 32;
        do {
            const int bits = min(11, shift), lo = shift - bits;
            for (int b = tid; b < kBins; b += NT) hist[b] = 0u;
            __syncthreads();
            for (int i = tid; i < e.len; i += NT) {
                const uint32_t k = h.key(i);
                if (k != kNewest && (shift == 32 || (k >> shift) == (thr >> shift)))
                    atomicAdd(&hist[(k >> lo) & ((1u << bits) - 1u)], 1u);
            }
            __syncthreads();
            pick_bin<NT>(hist, need, pick);
            thr |= pick[0] << lo;
            need = pick[1];
            equal = pick[2];
            shift = lo;
            __syncthreads();
        } while (shift > 0 && equal != need);
    }
    uint32_t done = 0, ties = 0, moved = 0;
    for (int i0 = 0; i0 < e.len; i0 += NT) {
        const int      i = i0 + tid;
        const bool     in = i < e.len;
        const uint32_t k = in ? h.key(i) : 0u;
        const bool     at = in && (k >> shift) == (thr >> shift);
        bool           stay = in && k > thr;
        uint32_t       total;
        if (equal == need) {
            stay |= at;
        } else {
            const uint32_t r = block_rank<NT>(at, lds, total);
            stay |= at && ties + r < need;
            ties += total;
        }
        const bool     flag = in && (i < e.keep ? !stay : stay);
        const uint32_t r = done + block_rank<NT>(flag, lds, total);
        moved += block_sum<NT>(flag && i < e.keep, lds); // free places come first
        if (flag && i < e.keep) pairs[r].y = i;
        if (flag && i >= e.keep) pairs[r - moved].x = i;
        done += total;
        if (i < e.keep && stay) {
            if (h.w_out != h.w_in) h.w_out[i] = h.w_in[i];
            if (h.p_out != h.p_in || i >= e.base) h.p_out[i] = h.position(i);
        }
    }
    if (tid == 0) a.counts[(int64_t)h.ei * a.Hkv + h.g] = (int32_t)moved;
    __threadfence_block();
    __syncthreads();
    for (uint32_t r = tid; r < moved; r += NT) {
        const int2 p = pairs[r];
        h.w_out[p.y] = h.w_in[p.x];
        h.p_out[p.y] = h.position(p.x);
    }
}

__device__ __forceinline__ int64_t row_off(const KvView &v, int row, int t) {
    if (v.block_table) {
        const int blk = v.block_table[(int64_t)row * v.bt_stride + (t >> v.log2_blk)];
        return (int64_t)blk * v.blk_stride + (int64_t)(t & ((1 << v.log2_blk) - 1)) * v.tok_stride;
    }
    return (int64_t)row * v.blk_stride + (int64_t)t * v.tok_stride;
}

// Sequences that lose one token, as a bounded cache does at every step (or none): the
// smallest key goes, of equal ones the last; its place, unless it is the last one,
// takes the last token, whose row is on its way before the search ends.  One
// launch, no lists.
__global__ __launch_bounds__(kOneThreads) void evict_one_kernel(EvictArgs a) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __shared__ uint64_t s_min[kOneThreads / 64];
    const int tid = threadIdx.x;
    EVICT_HEAD(a, h);
    const EvictEntry &e = h.e;
    const int last = e.len - 1, pieces = a.D / 8; // a K or V row's 16-byte pieces, 32 at most
    int       gone = e.len;                       // no token
    if (e.len > e.keep) {
        __half *b = const_cast<__half *>(tid >= pieces ? a.kv.v_base : a.kv.k_base) + (int64_t)h.g * a.kv.head_stride +
                    8 * (tid % pieces);
        u32x4   v = {0u, 0u, 0u, 0u};
        if (tid < 2 * pieces) v = *reinterpret_cast<const u32x4 *>(b + row_off(a.kv, e.row, last));
        uint64_t best = ~0ull;
        for (int i = 4 * tid; i < e.len; i += 4 * kOneThreads) {
            const Words w = load4(h.w_in, i, e.len);
            Words       p = {};
            if (i < e.base) p = load4(h.p_in, i, e.base);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int      pos = i + u < e.base ? (int)p.x[u] : i + u + e.gone;
                const uint32_t key = pos >= h.newest ? kNewest : account_key(__uint_as_float(w.x[u]));
                const uint64_t k = (uint64_t)key << 32 | (uint32_t)(0x7FFFFFFF - (i + u));
                best = i + u < e.len && k < best ? k : best;
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const uint64_t k = __shfl_xor(best, o);
            best = k < best ? k : best;
        }
        if ((tid & 63) == 0) s_min[tid >> 6] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kOneThreads / 64; ++w) best = s_min[w] < best ? s_min[w] : best;
        gone = 0x7FFFFFFF - (int)(uint32_t)best;
        if (tid < 2 * pieces && gone < last) *reinterpret_cast<u32x4 *>(b + row_off(a.kv, e.row, gone)) = v;
    }
    if (h.w_out == h.w_in && h.p_out == h.p_in) { // in place: the mover, and the positions that are new
        for (int i = e.base + tid; i < e.keep; i += kOneThreads)
            if (i != gone) h.p_out[i] = i + e.gone;
        if (tid == 0 && gone < last) {
            h.w_out[gone] = h.w_in[last];
            h.p_out[gone] = h.position(last);
        }
        return;
    }
    for (int i = tid; i < e.keep; i += kOneThreads) {
        const int from = i == gone ? last : i;
        if (h.w_out != h.w_in || from != i) h.w_out[i] = h.w_in[from];
        if (h.p_out != h.p_in || from != i || i >= e.base) h.p_out[i] = h.position(from);
    }
}

template <int D> __global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
    constexpr int PIECES = D / 8;
    constexpr int N = kMovePairs * 2 * PIECES / kMoveThreads; // pieces per thread
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int        ei = blockIdx.x / a.Hkv, g = blockIdx.x - ei * a.Hkv;
    const EvictEntry e = a.e[ei];
    const int        cap = min(e.len - e.keep, e.keep);
    if ((int)blockIdx.y * kMovePairs >= cap) return; // (before the count: no workgroup behind the list reads it)
    const int   cnt = a.counts[(int64_t)ei * a.Hkv + g];
    const int2 *pairs = reinterpret_cast<const int2 *>(a.pairs) + (int64_t)e.list * a.Hkv + (int64_t)g * cap;
    for (int first = blockIdx.y * kMovePairs; first < cap; first += gridDim.y * kMovePairs) {
        u32x4   v[N];
        __half *to[N];
#pragma unroll
        for (int u = 0; u < N; ++u) { // every row on its way before the first is written
            const int x = u * kMoveThreads + (int)threadIdx.x;
            const int r = first + x / (2 * PIECES);
            to[u] = nullptr;
            const int2 p = pairs[min(r, cap - 1)]; // (on its way with the count)
            if (r < cnt) {
                __half    *b = const_cast<__half *>(x / PIECES & 1 ? a.kv.v_base : a.kv.k_base) + (int64_t)g * a.kv.head_stride +
                            8 * (x % PIECES);
                v[u] = *reinterpret_cast<const u32x4 *>(b + row_off(a.kv, e.row, p.x));
                to[u] = b + row_off(a.kv, e.row, p.y);
            }
        }
#pragma unroll
        for (int u = 0; u < N; ++u)
            if (to[u]) *reinterpret_cast<u32x4 *>(to[u]) = v[u];
    }
}

template <int NT, int IT> void launch_select(const EvictArgs &a, dim3 grid, hipStream_t stream) {
    hipLaunchKernelGGL((evict_select_kernel<NT, IT>), grid, dim3(NT), 0, stream, a);
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
    // Entries that lose at most one token, then the others.
    for (const bool one : {true, false})
        for (size_t i = 0; i < entries.size();) {
            a.n = 0;
            int cap = 0, len = 0;
            a.counts = workspace + 2 * pairs * Hkv + (int64_t)launched * Hkv;
            for (; i < entries.size() && a.n < kEvictBatch; ++i) {
                const EvictEntry &e = entries[i];
                if ((e.len - e.keep <= 1) != one) continue;
                if (e.keep == e.len && (!copies || e.len == 0)) continue; // all stays, where it is
                a.e[a.n++] = e;
                cap = std::max(cap, std::min(e.len - e.keep, e.keep));
                len = std::max(len, e.len);
            }
            if (a.n == 0) break;
            launched += (size_t)a.n;
            profile_begin(KernelId::Evict, stream);
            const dim3 heads((unsigned)(a.n * Hkv));
            if (one) {
                hipLaunchKernelGGL(evict_one_kernel, heads, dim3(kOneThreads), 0, stream, a);
                HIP_CHECK(hipGetLastError());
                profile_end(KernelId::Evict, stream);
                continue;
            }
            if (len <= 1024) launch_select<256, 1>(a, heads, stream);
            else if (len <= 2048) launch_select<256, 2>(a, heads, stream);
            else if (len <= 4096) launch_select<512, 2>(a, heads, stream);
            else if (len <= 8192) launch_select<1024, 2>(a, heads, stream);
            else if (len <= 16384) launch_select<1024, 4>(a, heads, stream);
            else if (len <= 32768) launch_select<1024, 8>(a, heads, stream);
            else hipLaunchKernelGGL((evict_select_any_kernel<1024>), heads, dim3(1024), 0, stream, a);
            HIP_CHECK(hipGetLastError());
            const dim3 grid(heads.x, (unsigned)std::min((cap + kMovePairs - 1) / kMovePairs, kMostBlocks));
            switch (D) {
            case 32: hipLaunchKernelGGL((evict_move_kernel<32>), grid, dim3(kMoveThreads), 0, stream, a); break;
            case 64: hipLaunchKernelGGL((evict_move_kernel<64>), grid, dim3(kMoveThreads), 0, stream, a); break;
            case 128: hipLaunchKernelGGL((evict_move_kernel<128>), grid, dim3(kMoveThreads), 0, stream, a); break;
            default: hipLaunchKernelGGL((evict_move_kernel<256>), grid, dim3(kMoveThreads), 0, stream, a); break;
            }
            HIP_CHECK(hipGetLastError());
            profile_end(KernelId::Evict, stream);
        }
}

} // namespace detail
} // namespace tiny_llm
