// How the work of attn_stream_kernel (kernels/attention_stream.hip), of the prompt's
// account (kernels/attention_account.hip) and of attn_cross_kernel
// (kernels/attention_cross.hip) is cut: plain C++, unit-tested on the host.
#pragma once

#include <cstdint>
#include <vector>

namespace tiny_llm {
namespace detail {

constexpr int kStreamTile = 64;    // keys
constexpr int kStreamWhole = 12;   // tiles that one workgroup takes whatever else there is (a quarter at head_dim 256)
constexpr int kStreamRows = 16;    // query rows (tokens x heads of one kv head) of an entry at most
constexpr int kStreamBatch = 144;  // entries per launch: they travel in the kernel arguments

// Query tokens tok0 .. tok0 + nq - 1 attend to the first S tokens of cache row
// `row`.  item0, tile0: work items and tiles of the entries before it in its
// launch (in the kernels' arguments tile0 counts entries of several chunks only).
struct StreamEntry {
    int32_t row, S, tok0, nq, item0, tile0;
};

// Launch `first`..: n entries, `items` work items (per kv head), `tiles` tiles.
// Entry e has ceil(tiles_e / chunk) work items of equal size (in tiles, to one).
struct StreamLaunch {
    int     first, n, items, max_len;
    bool    finish; // some entry has several chunks, or no tokens
    int64_t tiles;
};
struct StreamPlan {
    std::vector<StreamEntry>  entries;
    std::vector<StreamLaunch> launches;
    int                       chunk = 1; // tiles
    int                       most = 0;  // tiles of the longest work item
    int                       waves = 4; // per workgroup
    void                      clear() { entries.clear(), launches.clear(); }
};

// LDS of a workgroup: at most kStreamLds of dynamic memory (160 KB a CU, less the
// kernel's own arrays).  Per wave, a stage of 16 V rows that later holds the rows'
// fp32 outputs (half of kStreamRows rows where scores are kept); with scores, also 4
// bytes for each token and row of the work item.
constexpr int kStreamLds = 160 * 1024 - 2048;
constexpr int stream_stage_bytes(int D, bool scores) { return kStreamRows / (scores ? 2 : 1) * D * 4; }
constexpr int stream_most_tiles(int D, int waves, int rows) { // with scores
    return (kStreamLds - waves * stream_stage_bytes(D, true)) / (kStreamTile * rows * 4);
}

inline int stream_tiles(int S) { return S / kStreamTile + (S % kStreamTile != 0); }
inline int stream_items(int S, int chunk) { return (stream_tiles(S) + chunk - 1) / chunk; }

// Sets item0 and tile0 of plan.entries (and orders them, longest first), the
// launches, the waves and the chunk length.  account_rows: query rows of every entry
// when their scores are kept (at most kStreamRows / 2), 0: they are not.
void plan_stream(StreamPlan &plan, int Hkv, int D, int account_rows, int cus);

constexpr int kAccountRows = 128;  // query rows of a workgroup of account_stats_kernel
constexpr int kAccountKeys = 256;  // keys of a workgroup of account_sum_kernel
constexpr int kAccountStep = 64;   // rows that it stages at a time
constexpr int kAccountBatch = 44;  // entries per launch
constexpr int kAccountPieces = 64; // pieces per launch and kernel
constexpr int kAccountFold = 256;  // rows of a chunk whose statistics account_sum_kernel merges,
constexpr int kAccountFoldParts = 8192; // and their partial results at most

// The last w of the n new tokens of cache row `row` (positions p0 .. p0 + n - 1; tok0:
// the first one's index in the call's tokens) attend causally: w * G query rows per
// kv head.  account_stats_kernel cuts them into tiles and the keys that a tile sees into
// nch chunks at most; account_sum_kernel cuts the keys into blocks and the rows that see
// a block into nrc chunks at most.  lse0, stat0, part0: rows of results, rows of partial
// results and tokens of partial sums of the entries before.
struct AccountEntry {
    int32_t row, p0, n, w, tok0, nch, lse0, stat0, nrc, part0;
};
// Tiles (blocks) first .. last - 1 of an entry, each in `chunks` equal chunks, some of
// them empty where it has less: work items item0 .. of the launch.
struct AccountPiece {
    int32_t  item0, first, last;
    uint32_t what; // entry of the launch | chunks << 8
    int      entry() const { return (int)(what & 255u); }
    int      chunks() const { return (int)(what >> 8); }
};
struct AccountLaunch {
    int     first, n, items, sums;
    bool    split_keys, split_rows;   // some nch, nrc is above 1
    bool    fold;                     // account_sum_kernel merges the key chunks' statistics itself
    int     most_rows, most_keys;     // of an entry that is split
    int64_t lse, stats, parts;        // per kv head
    std::vector<AccountPiece> tile_pieces, block_pieces; // longest items first
};
struct AccountPlan {
    std::vector<AccountEntry>  entries;
    std::vector<AccountLaunch> launches;
    int                        window = -1;
    void                       clear() { entries.clear(), launches.clear(), window = -1; }
};

inline int account_blocks(int keys) { return keys / kAccountKeys + (keys % kAccountKeys != 0); }
// Key tiles that row tile rt sees, and the first of the row steps that see key block kb.
inline int account_seen(const AccountEntry &e, int G, int rt) {
    const int64_t rows = (int64_t)e.w * G, r_hi = rows < (int64_t)(rt + 1) * kAccountRows ? rows : (int64_t)(rt + 1) * kAccountRows;
    return stream_tiles((int)(e.p0 + e.n - e.w + (r_hi - 1) / G + 1));
}
inline int account_sees(const AccountEntry &e, int G, int kb) {
    const int64_t behind = (int64_t)kb * kAccountKeys - (e.p0 + e.n - e.w);
    return behind > 0 ? (int)(behind * G / kAccountStep) : 0;
}

// Sets the rest of plan.entries, and the launches.  False when a launch's rows or
// items do not fit 31 bits.
bool plan_account(AccountPlan &plan, int G, int Hkv, int cus);

// Query tokens tok0 .. tok0 + nq - 1 attend to the first S >= 1 tokens of cache row
// `row`: row tiles (of tokens x heads of one kv head) x nch chunks of its keys are
// the work items of attn_cross_kernel, item0 those of the entries before it in its
// launch.
constexpr int kCrossBatch = 144;
struct CrossEntry {
    int32_t row, S, tok0, nq, nch, item0;
};
struct CrossLaunch {
    int  first, n, items;
    bool split; // some entry has several chunks
};
struct CrossPlan {
    std::vector<CrossEntry>  entries;
    std::vector<CrossLaunch> launches;
    int                      waves = 4; // per workgroup
    void                     clear() { entries.clear(), launches.clear(); }
};
// Whether 8 waves are an option (64: level with 4).
constexpr bool cross_wide(int D) { return D == 32 || D == 128; }
// Rows of a workgroup: 32 per wave up to head_dim 128, 16 at 256.
constexpr int cross_rows(int D, int waves) { return waves * (D <= 128 ? 32 : 16); }

// Sets the waves, nch and item0 of plan.entries and the launches (and orders the
// entries, longest items first).  False when a launch's items exceed 31 bits.
bool plan_cross(CrossPlan &plan, int D, int G, int Hkv, int cus);

} // namespace detail
} // namespace tiny_llm
