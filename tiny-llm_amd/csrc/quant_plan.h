// The cache in 8 bits: its constants, and how the work of attn_quant_kernel
// (kernels/attention_quant.hip) and quant_prefill_kernel (kernels/prefill_quant.hip) is
// cut.  Plain C++, unit-tested on the host.
#pragma once

#include <cstdint>
#include <utility>
#include <vector>

namespace tiny_llm {
namespace detail {

constexpr int kGroup = 32;      // tokens that share a scale
constexpr int kQuantTile = 64;  // tokens of a step of the attention kernels: two groups
constexpr int kQuantRows = 16;  // query rows (tokens x heads of one kv head) of an entry of attn_quant_kernel at most
constexpr int kQuantBatch = 144; // entries per launch: they travel in the kernel arguments
constexpr int kQuantPrefillBatch = 112;

// The open group of a slot: which of its two tiles is the current one, the groups whose rows
// they hold (-1: none), where the last append ended, and where the one that went furthest did.
struct OpenGroup {
    int group[2] = {-1, -1};
    int cur = 0;
    int end = 0;
    int far = 0;

    // The tiles of an append of n tokens behind len: that of the group it begins in, and that of the
    // group it ends in (the other one where that is another group).
    std::pair<int, int> tiles(int len, int n) const { return {cur, len / kGroup == (len + n) / kGroup ? cur : 1 - cur}; }
    void                append(int len, int n) {
        end = len + n;
        far = end > far ? end : far;
        group[cur] = len / kGroup;
        group[1 - cur] = end / kGroup != len / kGroup && end % kGroup != 0 ? end / kGroup : -1;
    }
    // Tokens that are there, those behind len included, and the tile of their last group.
    std::pair<int, int> held(int len) const { return {end > len ? end : len, end > len ? tiles(len, end - len).second : cur}; }
    // Whether length `to` leaves the group that the last append ended in, whose rows wait in fp16 for those
    // that complete it: nothing would read them there any more.
    bool leaves_rows(int to) const { return end % kGroup != 0 && to / kGroup > end / kGroup; }
    // Whether it is beyond the last append, where an earlier one had brought more: its rows there may
    // have made room for the last one's.
    bool replaced(int to) const { return to > end && far > end; }
    // Whether the layers, whose last appends ended at ends[], can all go from length len to length `to`: the tiles are
    // told apart by the last append to any of them, so what was appended behind len has to be alike in those that
    // have some, and the others must not leave rows behind either.
    bool alike(const int *ends, int layers, int len, int to) const {
        for (int l = 0; l < layers; ++l)
            if (ends[l] != end && (ends[l] > len || (ends[l] % kGroup != 0 && to / kGroup > ends[l] / kGroup))) return false;
        return true;
    }
    // From length len to length `to`; false (and no change) where that leaves rows behind, or shows
    // replaced ones, or lies inside what one append brought and the rows that would be open again are gone.
    bool advance(int len, int to) {
        const int g = to / kGroup;
        if (leaves_rows(to) || replaced(to)) return false;
        if (g != len / kGroup && group[1 - cur] == g) {
            cur = 1 - cur;
        } else if (to % kGroup != 0 && to < end && (g != len / kGroup || group[cur] != g)) {
            return false;
        } else if (g != len / kGroup) {
            // Nothing is open at a group's first token; what was never appended is whatever is there.
            group[cur] = to % kGroup != 0 ? g : -1;
        }
        return true;
    }
};

// Query tokens tok0 .. tok0 + nq - 1 attend to the first S tokens of slot `row`, the last
// one to all of them, the others causally.  open: the tile (0 or 1) that holds the
// tokens from S / 32 * 32 on in fp16, or -1: every attended token is in 8 bits.  item0: work
// items of the entries before it in its launch.
struct QuantEntry {
    int32_t row, S, tok0, nq, open, item0;
    int     closed() const { return open < 0 ? S : S / kGroup * kGroup; }
};
struct QuantLaunch {
    int  first, n, items, rows; // rows: of the entry with the most
    bool finish;                // some entry has several chunks, or no tokens
};
// Entry e has ceil(tiles / chunk) work items of equal size (in tiles, to one).
struct QuantPlan {
    std::vector<QuantEntry>  entries;
    std::vector<QuantLaunch> launches;
    int                      chunk = 1; // tiles
    bool                     small = false; // workgroups of kQuantSmallWaves waves
    void                     clear() { entries.clear(), launches.clear(); }
};
// Waves of a workgroup: for most, and for many entries of a few tiles.
constexpr int quant_waves(int D) { return D <= 128 ? 8 : 4; }
constexpr int kQuantSmallWaves = 2;
inline int quant_tiles(int S) { return S / kQuantTile + (S % kQuantTile != 0); }
inline int quant_items(int S, int chunk) { return (quant_tiles(S) + chunk - 1) / chunk; }
// Sets item0 of plan.entries (and orders them, longest first), the launches and the chunk length.
void plan_quant(QuantPlan &plan, int G, int Hkv, int D, int cus);

// The same for more query rows: rt row tiles (of tokens x heads of one kv head) x nch chunks
// of the keys that a tile sees; the work items of an entry are its tiles from the last,
// which sees the most, to the first, times nch.
struct QuantPrefillEntry {
    int32_t row, S, tok0, nq, open, nch, item0;
};
struct QuantPrefillLaunch {
    int first, n, items;
    int parts; // items up to the last of an entry of several chunks, 0: there is none
};
struct QuantPrefillPlan {
    std::vector<QuantPrefillEntry>  entries;
    std::vector<QuantPrefillLaunch> launches;
    void                            clear() { entries.clear(), launches.clear(); }
};
// Waves and rows of a workgroup, workgroups a CU, and the tokens of a key tile.  Four waves and two workgroups at
// head_dim 128, eight waves elsewhere, two workgroups where 128 registers do (1 x 8192, 4 x 500 over 3000 .. 6000; 8 heads,
// groups of 4, eight waves against four: 128 611, 221 against 598, 190 us; 256 1288, 420 against 2704, 825; 64
// 321, 114 against 338, 121; 32 232, 87 against 240, 89.  One workgroup of eight at 64 394, 152, at 32 304, 117).
constexpr int quant_prefill_waves(int D) { return D == 128 ? 4 : 8; }
constexpr int quant_prefill_rows(int D) { return quant_prefill_waves(D) * (D <= 128 ? 32 : 16); }
constexpr int quant_prefill_per_cu(int D) { return D <= 128 ? 2 : 1; }
constexpr int quant_prefill_tile(int D) { return D <= 128 ? 64 : 32; }
// Sets nch and item0 of plan.entries and the launches (and orders the
// entries, longest items first).  False when a launch would have more than 2^32 threads.
constexpr int64_t kQuantMostItems = (1 << 23) - 1;
bool plan_quant_prefill(QuantPrefillPlan &plan, int D, int G, int Hkv, int cus);

} // namespace detail
} // namespace tiny_llm
