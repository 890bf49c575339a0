// Layout of a cache in 8 bits and the launch interface of its kernels
// (quant_copy.hip, attention_quant.hip, prefill_quant.hip).
//
// A group is 32 consecutive tokens of one kv head.  Its tile is 64 D bytes, 32 D of K and
// then 32 D of V, whole numbers x + 128, in the order in which the matrix instructions take
// their operands (v_mfma_f32_16x16x32_f16), so that a wave's loads are of 16 bytes a
// lane, back to back, and go into registers as they are:
//   K   piece (token r, dims 8 o .. 8 o + 7), 8 bytes, at k_piece(r, o)
//   V   piece (dim d, tokens 4 q .. 4 q + 3 and 16 + 4 q .. 16 + 4 q + 3), at v_piece(q, d):
//       the tokens of which a lane has the weights after the first product
// and one scale for K and one for V: the value is (stored byte - 128) * scale.
// The group that a sequence has not filled yet is an open tile of the slot: the same
// pieces in fp16, 16 bytes each.  A slot has two, so that the group in which an append
// begins and the one in which it ends are both there until the lengths advance.
#pragma once

#include "../quant_plan.h"

#include <hip/hip_fp16.h>
#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>
#include <vector>

namespace tiny_llm {
namespace detail {

// One layer of the cache.  Tile of group i of a sequence: block table[row * bt_stride +
// (i >> lg)], tiles + (((block * Hkv + g) << lg) + (i & (2^lg - 1))) * 64 D bytes; scales by the
// same index; open tile w of slot `row`: open + ((row * 2 + w) * Hkv + g) * 64 D halves.
struct QuantView {
    uint8_t       *tiles = nullptr;
    float2        *scales = nullptr; // (K, V)
    __half        *open = nullptr;
    const int32_t *table = nullptr;
    int            bt_stride = 0;
    int            lg = 0; // log2 of the groups per block
};

// n tokens of slot `row` from position p0 on, rows tok0 .. of the call's.  first: the open
// tile of group p0 / 32, last: the one for group (p0 + n) / 32 where that is another.  item0:
// groups of the entries before it in its launch.
struct QuantAppend {
    int32_t row, p0, n, tok0, first_last, item0;
    int     groups() const { return (p0 + n + kGroup - 1) / kGroup - p0 / kGroup; }
};

// Zeros for the rows lo .. hi - 1 of an open tile that nobody brought, so that they have no part in the scale of
// the group's others.
struct QuantRows {
    int32_t row, tile, lo, hi;
};
void launch_quant_zero_rows(const QuantView &v, const std::vector<QuantRows> &entries, int Hkv, int D, hipStream_t stream);
// Appends new_k / new_v [tokens][Hkv][D]; sets the entries' item0.
void launch_quant_append(const QuantView &v, std::vector<QuantAppend> &entries, int Hkv, int D, const __half *new_k,
                         const __half *new_v, hipStream_t stream);
// One token per entry (n = 1) into num_layers layers: rows [layer][entry][Hkv][D]; from a
// layer to the next the view's tiles, scales and open tiles are `steps` further (in elements).
struct QuantLayerSteps {
    int64_t tiles = 0, scales = 0, open = 0;
};
void launch_quant_append_one(const QuantView &v, const QuantLayerSteps &steps, const std::vector<QuantAppend> &entries,
                             int num_layers, int Hkv, int D, const __half *new_k, const __half *new_v,
                             hipStream_t stream);
// k_out / v_out (either may be null) [entry][Hkv][s_max][D]: what the cache stands for, zeros
// behind the entry's S.
void launch_quant_gather(const QuantView &v, const std::vector<QuantEntry> &entries, int Hkv, int D, int s_max,
                         __half *k_out, __half *v_out, hipStream_t stream);

struct QuantCall {
    const __half *q = nullptr; // [tokens][Hq][D]
    __half       *out = nullptr;
    // Entries of one query: the token at S - 1 comes from here ([token][Hkv][D]) and is
    // appended; `open` of the entries is then the tile of its group, closed or not.
    const __half *new_k = nullptr, *new_v = nullptr;
    float         scale = 1.0f;
    int           Hq = 0, Hkv = 0, D = 0;
};
size_t quant_workspace_floats(const QuantPlan &plan, int Hkv, int D);
void   launch_attn_quant(const QuantCall &c, const QuantView &v, const QuantPlan &plan, float *workspace, hipStream_t stream);
size_t quant_prefill_workspace_floats(const QuantPrefillPlan &plan, int Hkv, int D);
void   launch_quant_prefill(const QuantCall &c, const QuantView &v, const QuantPrefillPlan &plan, float *workspace,
                            hipStream_t stream);

} // namespace detail
} // namespace tiny_llm
