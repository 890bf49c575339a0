// Writing a cache in 8 bits and reading it back, for gfx950 (layout: quant.h).
//
// A group of 32 tokens of one kv head is rounded once, when its last token comes, from the
// fp16 rows that wait in the slot's open tile:
//   s = cut_11_bits(max |x| / 127),  stored = round_half_even(x / s) + 128
// so the cached bytes do not depend on how the tokens came (one by one, in chunks, at
// once).  Bound by HBM: 4 D bytes of new rows in and 2 D out per token and kv head, 2 D in and 4
// D out to read back.
//
// quant_append_kernel: a workgroup per (entry, group, kv head).  Rows of a group that stays open go
// straight into its open tile.  Those of one that closes meet in LDS as the pieces of a tile (V's
// tokens side by side: the transposition that its matrix operand needs), then 16 bytes a lane
// go out in order.  32768 tokens, 8 heads of 128, 201 MB: 38-46 us, 4.4-5.3 TB/s by how much of the
// last call is still being written back (a copy by the library: 5.1).  Four tokens of 32 sequences: 5 us.
// The V rows' 2-byte stores to LDS meet in its banks (40% of the cycles), which is hidden: four tokens
// at a time, transposed in registers, swizzled, took as long.
// quant_append_one_kernel: a decode step's token; 31 of 32 times only its row.  2.8 us, the launch.
// quant_gather_kernel: a workgroup per (entry, kv head, group), through LDS to rows.  The same 201
// MB: 31 us, 6.5 TB/s.
#include "quant_device.h"

#include "../runtime.h"
#include "kv_kernels.h"
#include "tiny_llm/hip_utils.h"

#include <algorithm>
#include <climits>
#include <cstring>
#include <stdexcept>

namespace tiny_llm {
namespace detail {

namespace {

using namespace quant;

constexpr int     kThreads = 256;
constexpr int64_t kMostBlocks = (int64_t(1) << 32) / kThreads - 1; // a grid has fewer than 2^32 threads

struct AppendArgs {
    QuantView       v;
    QuantLayerSteps steps;
    const uint16_t *new_k, *new_v;
    int             Hkv, n;
    QuantAppend     e[kQuantBatch];
};
static_assert(sizeof(AppendArgs) <= 4096, "kernel arguments");

template <int D> __global__ __launch_bounds__(kThreads) void quant_append_kernel(AppendArgs a) {
    constexpr int KP = D / 8; // pieces of a row
    __shared__ __align__(16) uint16_t s_open[64 * D];
    __shared__ uint32_t               red[2 * kThreads / 64];
    const int item = blockIdx.x / a.Hkv, g = blockIdx.x - item * a.Hkv;
    int       ei;
    QUANT_ENTRY_OF(a, item, ei);
    const int row = a.e[ei].row, p0 = a.e[ei].p0, n = a.e[ei].n, tok0 = a.e[ei].tok0;
    const int first = a.e[ei].first_last & 1, last = a.e[ei].first_last >> 1;
    const int group = p0 / kGroup + item - a.e[ei].item0, t0 = group * kGroup;
    const int r_lo = max(0, p0 - t0), r_hi = min(kGroup, p0 + n - t0); // new rows of the group
    const bool opens = t0 <= p0; // the group in which the append begins
    uint16_t  *tile0 = open_of<D>(a.v, a.Hkv, row, first, g);

    constexpr int PER = (kGroup * KP + kThreads - 1) / kThreads; // pieces of a thread
    const int     pieces = (r_hi - r_lo) * KP;
    u32x4         k[PER], v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int x = threadIdx.x + i * kThreads;
        if (x >= pieces) break;
        const int64_t src = ((int64_t)(tok0 + t0 + r_lo + x / KP - p0) * a.Hkv + g) * D + 8 * (x % KP);
        k[i] = *reinterpret_cast<const u32x4 *>(a.new_k + src);
        v[i] = *reinterpret_cast<const u32x4 *>(a.new_v + src);
    }
    auto put = [&](uint16_t *tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int x = threadIdx.x + i * kThreads, r = r_lo + x / KP, o = x % KP;
            if (x >= pieces) break;
            reinterpret_cast<u32x4 *>(tile)[k_piece(r, o)] = k[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[32 * D + v_half(r, 8 * o + j)] = (uint16_t)(v[i][j / 2] >> (16 * (j & 1)));
        }
    };
    if (r_hi < kGroup) { // (behind its last row a tile holds anything)
        put(opens ? tile0 : open_of<D>(a.v, a.Hkv, row, last, g));
        return;
    }
    u32x4 *s16 = reinterpret_cast<u32x4 *>(s_open);
    if (r_lo > 0) { // its earlier rows
        for (int p = threadIdx.x; p < 8 * D; p += kThreads) s16[p] = reinterpret_cast<const u32x4 *>(tile0)[p];
        __syncthreads();
    }
    put(s_open);
    if (opens) put(tile0);
    __syncthreads();
    const int64_t at = tile_of(a.v, a.Hkv, row, g, group);
    close_group<D, kThreads>(s_open, a.v.tiles + at * (64 * D), a.v.scales + at, red);
}

// A wave per (entry, kv head) and layer.
template <int D> __global__ __launch_bounds__(64) void quant_append_one_kernel(AppendArgs a) {
    const int     i = blockIdx.x / a.Hkv, g = blockIdx.x - i * a.Hkv, layer = blockIdx.y;
    const int     row = a.e[i].row, p = a.e[i].p0;
    const int64_t at = tile_of(a.v, a.Hkv, row, g, p / kGroup);
    // (rows of a launch's entries follow each other; item0: the entries of the call)
    const int64_t src = (((int64_t)layer * a.e[i].item0 + a.e[i].tok0) * a.Hkv + g) * D;
    GroupRegs<D>  group;
    uint16_t     *open = open_of<D>(a.v, a.Hkv, row, a.e[i].first_last & 1, g) + layer * a.steps.open;
    const bool    closes = p % kGroup == kGroup - 1;
    if (closes) group.load(open);
    group.fetch(p % kGroup, a.new_k + src, a.new_v + src);
    group.append(open, p % kGroup);
    if (closes) group.close(a.v.tiles + layer * a.steps.tiles + at * (64 * D), a.v.scales + layer * a.steps.scales + at);
}

struct ZeroArgs {
    QuantView v;
    int       Hkv;
    QuantRows e[kQuantBatch];
};
static_assert(sizeof(ZeroArgs) <= 4096, "kernel arguments");

// A wave per (entry, kv head).
template <int D> __global__ __launch_bounds__(64) void quant_zero_rows_kernel(ZeroArgs a) {
    const int i = blockIdx.x / a.Hkv, g = blockIdx.x - i * a.Hkv;
    uint16_t *tile = open_of<D>(a.v, a.Hkv, a.e[i].row, a.e[i].tile, g);
    for (int r = a.e[i].lo; r < a.e[i].hi; ++r) {
        if (threadIdx.x < D / 8) reinterpret_cast<u32x4 *>(tile)[k_piece(r, (int)threadIdx.x)] = u32x4{0u, 0u, 0u, 0u};
        for (int d = threadIdx.x; d < D; d += 64) tile[32 * D + v_half(r, d)] = 0;
    }
}

struct GatherArgs {
    QuantView  v;
    uint16_t  *k_out, *v_out;
    int        Hkv, n, first, s_max;
    QuantEntry e[kQuantBatch];
};
static_assert(sizeof(GatherArgs) <= 4096, "kernel arguments");

// Two halves of whole numbers times the scale, rounded to fp16 once (the product is exact in fp32).
__device__ __forceinline__ uint32_t scaled2(uint32_t two, float s) {
    const f16x2   x = __builtin_bit_cast(f16x2, two);
    const __half2 y = __floats2half2_rn((float)x[0] * s, (float)x[1] * s);
    return __builtin_bit_cast(uint32_t, y);
}

// blockIdx.y: 0 K, 1 V (or the one that is asked for).
template <int D> __global__ __launch_bounds__(kThreads) void quant_gather_kernel(GatherArgs a) {
    constexpr int KP = D / 8, PITCH = D + 8;
    __shared__ __align__(16) uint16_t rows[kGroup * PITCH];
    const int  groups = (a.s_max + kGroup - 1) / kGroup;
    const int  group = blockIdx.x % groups, eg = blockIdx.x / groups, g = eg % a.Hkv, ei = eg / a.Hkv;
    const bool is_v = a.k_out == nullptr || blockIdx.y == 1;
    const int  row = a.e[ei].row, S = a.e[ei].S, t0 = group * kGroup;
    const int  valid = min(kGroup, S - t0), wanted = min(kGroup, a.s_max - t0);
    if (valid > 0) {
        // A thread has the pieces 2 p and 2 p + 1.
        const bool   is_open = a.e[ei].open >= 0 && t0 + kGroup > S;
        const int64_t at = is_open ? 0 : tile_of(a.v, a.Hkv, row, g, group);
        const float2 sc = is_open ? make_float2(1.0f, 1.0f) : a.v.scales[at];
        const float  s = is_v ? sc.y : sc.x;
        for (int p = threadIdx.x; p < 2 * D; p += kThreads) {
            u32x4 x[2];
            if (is_open) {
                const u32x4 *src = reinterpret_cast<const u32x4 *>(open_of<D>(a.v, a.Hkv, row, a.e[ei].open, g) + (is_v ? 32 * D : 0));
                x[0] = src[2 * p];
                x[1] = src[2 * p + 1];
            } else {
                const u32x4 w = reinterpret_cast<const u32x4 *>(a.v.tiles + at * (64 * D) + (is_v ? 32 * D : 0))[p];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    x[h] = __builtin_bit_cast(u32x4, whole8(w[2 * h], w[2 * h + 1]));
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[h][i] = scaled2(x[h][i], s);
                }
            }
            const int lane = p & 63, q = lane >> 4, c = lane & 15, s32 = 32 * (p >> 6);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!is_v) {
                    *reinterpret_cast<u32x4 *>(&rows[(16 * h + c) * PITCH + s32 + 8 * q]) = x[h];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        rows[(16 * (i >> 2) + 4 * q + (i & 3)) * PITCH + s32 + 16 * h + c] = (uint16_t)(x[h][i / 2] >> (16 * (i & 1)));
                }
            }
        }
        __syncthreads();
    }
    uint16_t *out = (is_v ? a.v_out : a.k_out) + (((int64_t)(a.first + ei) * a.Hkv + g) * a.s_max + t0) * D;
    for (int x = threadIdx.x; x < wanted * KP; x += kThreads) {
        const int r = x / KP, o = x % KP;
        const u32x4 y = r < valid ? *reinterpret_cast<const u32x4 *>(&rows[r * PITCH + 8 * o]) : u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4 *>(out + (int64_t)r * D + 8 * o) = y;
    }
}

} // namespace

void launch_quant_zero_rows(const QuantView &v, const std::vector<QuantRows> &entries, int Hkv, int D, hipStream_t stream) {
    ZeroArgs a{};
    a.v = v;
    a.Hkv = Hkv;
    for (size_t i = 0; i < entries.size();) {
        const size_t n = std::min<size_t>(kQuantBatch, entries.size() - i);
        std::memcpy(a.e, entries.data() + i, sizeof(QuantRows) * n);
        i += n;
        for_head_dim(D, [&](auto d) {
            hipLaunchKernelGGL(quant_zero_rows_kernel<decltype(d)::value>, dim3((unsigned)(n * (size_t)Hkv)), dim3(64), 0, stream, a);
        });
        HIP_CHECK(hipGetLastError());
    }
}

void launch_quant_append(const QuantView &v, std::vector<QuantAppend> &entries, int Hkv, int D, const __half *new_k,
                         const __half *new_v, hipStream_t stream) {
    AppendArgs a{};
    a.v = v;
    a.new_k = reinterpret_cast<const uint16_t *>(new_k);
    a.new_v = reinterpret_cast<const uint16_t *>(new_v);
    a.Hkv = Hkv;
    for (size_t i = 0; i < entries.size();) {
        int64_t items = 0;
        a.n = 0;
        for (; i < entries.size() && a.n < kQuantBatch; ++i, ++a.n) {
            if (a.n && (items + entries[i].groups()) * Hkv > kMostBlocks) break;
            entries[i].item0 = (int32_t)items;
            items += entries[i].groups();
            a.e[a.n] = entries[i];
        }
        if (items * Hkv > kMostBlocks) throw std::invalid_argument("8-bit cache: too many groups in one append");
        profile_begin(KernelId::KvAppend, stream);
        for_head_dim(D, [&](auto d) {
            hipLaunchKernelGGL(quant_append_kernel<decltype(d)::value>, dim3((unsigned)(items * Hkv)), dim3(kThreads), 0, stream, a);
        });
        HIP_CHECK(hipGetLastError());
        profile_end(KernelId::KvAppend, stream);
    }
}

void launch_quant_append_one(const QuantView &v, const QuantLayerSteps &steps, const std::vector<QuantAppend> &entries,
                             int num_layers, int Hkv, int D, const __half *new_k, const __half *new_v,
                             hipStream_t stream) {
    AppendArgs a{};
    a.v = v;
    a.steps = steps;
    a.new_k = reinterpret_cast<const uint16_t *>(new_k);
    a.new_v = reinterpret_cast<const uint16_t *>(new_v);
    a.Hkv = Hkv;
    for (size_t i = 0; i < entries.size(); i += (size_t)a.n) {
        a.n = (int)std::min<size_t>(kQuantBatch, entries.size() - i);
        for (int k = 0; k < a.n; ++k) {
            a.e[k] = entries[i + (size_t)k];
            a.e[k].item0 = (int32_t)entries.size();
        }
        profile_begin(KernelId::KvAppend, stream);
        for_head_dim(D, [&](auto d) {
            hipLaunchKernelGGL(quant_append_one_kernel<decltype(d)::value>, dim3((unsigned)(a.n * Hkv), (unsigned)num_layers),
                               dim3(64), 0, stream, a);
        });
        HIP_CHECK(hipGetLastError());
        profile_end(KernelId::KvAppend, stream);
    }
}

void launch_quant_gather(const QuantView &v, const std::vector<QuantEntry> &entries, int Hkv, int D, int s_max,
                         __half *k_out, __half *v_out, hipStream_t stream) {
    if (!k_out && !v_out) return;
    GatherArgs a{};
    a.v = v;
    a.k_out = reinterpret_cast<uint16_t *>(k_out);
    a.v_out = reinterpret_cast<uint16_t *>(v_out);
    a.Hkv = Hkv;
    a.s_max = s_max;
    const int64_t groups = (s_max + (int64_t)kGroup - 1) / kGroup;
    const int64_t most = std::max<int64_t>(1, kMostBlocks / (groups * Hkv)); // entries of a launch
    if (groups * Hkv > kMostBlocks) throw std::invalid_argument("8-bit cache: s_max too large for one gather");
    for (size_t i = 0; i < entries.size(); i += (size_t)a.n) {
        a.first = (int)i;
        a.n = (int)std::min<size_t>((size_t)std::min<int64_t>(kQuantBatch, most), entries.size() - i);
        std::memcpy(a.e, entries.data() + i, sizeof(QuantEntry) * (size_t)a.n);
        profile_begin(KernelId::KvGather, stream);
        for_head_dim(D, [&](auto d) {
            hipLaunchKernelGGL(quant_gather_kernel<decltype(d)::value>, dim3((unsigned)(groups * Hkv * a.n), k_out && v_out ? 2u : 1u),
                               dim3(kThreads), 0, stream, a);
        });
        HIP_CHECK(hipGetLastError());
        profile_end(KernelId::KvGather, stream);
    }
}

} // namespace detail
} // namespace tiny_llm
