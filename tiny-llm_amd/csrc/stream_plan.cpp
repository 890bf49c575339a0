#include "stream_plan.h"

#include <algorithm>
#include <climits>
#include <utility>

namespace tiny_llm {
namespace detail {

void plan_stream(StreamPlan &plan, int Hkv, int D, int account_rows, int cus) {
    int64_t total = 0, some = 0, longest = 0;
    for (const auto &e : plan.entries) {
        total += stream_tiles(e.S);
        some += e.S > 0;
        longest = std::max<int64_t>(longest, stream_tiles(e.S));
    }
    total *= Hkv;
    const int64_t n = std::max(1, cus);
    int64_t       chunk;
    const int64_t share = (total + n - 1) / n, half = (total + 2 * n - 1) / (2 * n); // of a CU, of one of two workgroups
    const bool    few = some * Hkv <= n;
    // An entry in one chunk is finished by its own workgroup: no partial results, no
    // second launch, and its scores never leave the LDS.  Short entries are left whole
    // (16 x 300 tokens with accounts, 8 heads of 64: 7.2 us, 11.6 split), with eight waves
    // where they have so many tiles.  Work that is little for the chip is spread over
    // as many workgroups as it has pieces of four tiles (1 x 4096, 8 heads of 128: 14.0 us,
    // 16.8 in pieces of 8 on eight waves, 30 of 32).  Where a CU has several tiles to itself,
    // eight waves and fewer pieces are better (4 x 2048: 17.6 against 19.0 us; 1 x 32768:
    // 33.0, 34.5), and whole entries are while they fill half of the chip and none is much
    // longer than a CU's share (30 x 4096: 96 us, 112; 20 x 1500, 8 heads of 64: 17.5, 21;
    // but 8 x 1024: 19.3, 16.9).
    if (few && longest <= (D <= 128 ? kStreamWhole : kStreamWhole / 4)) {
        plan.waves = D <= 128 && longest > 4 ? 8 : 4;
        chunk = longest;
    } else if (few && total < (account_rows > 0 ? 4 : 8) * n) {
        plan.waves = 4;
        chunk = std::max<int64_t>(4, half);
    } else if (few && D <= 128) {
        plan.waves = 8;
        chunk = std::max<int64_t>(8, share);
        if (2 * some * Hkv >= n && 2 * longest <= 5 * chunk) chunk = longest;
    } else {
        plan.waves = 4;
        chunk = longest <= std::max<int64_t>(32, 2 * half + half / 2) ? longest : std::max<int64_t>(8, half);
    }
    if (account_rows > 0) {
        const int64_t fits = stream_most_tiles(D, plan.waves, account_rows);
        if (chunk > fits) // (equal chunks)
            chunk = std::min(fits, (longest + (longest + fits - 1) / fits - 1) / std::max<int64_t>(1, (longest + fits - 1) / fits));
    }
    plan.chunk = (int)std::max<int64_t>(1, std::min<int64_t>(chunk, 1 << 24));
    plan.most = 0;
    for (const auto &e : plan.entries) {
        const int t = stream_tiles(e.S), k = stream_items(e.S, plan.chunk);
        if (k) plan.most = std::max(plan.most, (t + k - 1) / k);
    }
    // Longest work items first.
    auto item_tiles = [&](const StreamEntry &e) {
        const int k = stream_items(e.S, plan.chunk);
        return k ? (stream_tiles(e.S) + k - 1) / k : 0;
    };
    std::stable_sort(plan.entries.begin(), plan.entries.end(),
                     [&](const StreamEntry &x, const StreamEntry &y) { return item_tiles(x) > item_tiles(y); });
    plan.launches.clear();
    for (size_t i = 0; i < plan.entries.size();) {
        StreamLaunch l{(int)i, 0, 0, 0, false, 0};
        for (; i < plan.entries.size() && l.n < kStreamBatch; ++i, ++l.n) {
            StreamEntry &e = plan.entries[i];
            const int    items = stream_items(e.S, plan.chunk);
            e.item0 = l.items;
            e.tile0 = (int32_t)l.tiles;
            l.items += items;
            l.tiles += stream_tiles(e.S);
            l.finish |= items != 1;
            if (items > 1) l.max_len = std::max(l.max_len, e.S);
        }
        plan.launches.push_back(l);
    }
}

bool plan_account(AccountPlan &plan, int G, int Hkv, int cus) {
    // Work items take about a third of a CU's share of all key tiles (or row steps), in the
    // order of their length: a whole prompt's row tiles see from one key tile to all of
    // them, and its key blocks are seen by all rows to few (8 heads of 128, groups of 4: 4 x
    // 1700..2048 on prefixes 214 us, whole tiles entry by entry 246; 1 x 2048 69 and 80).
    // Row tiles that are fewer than CUs: half of a share (the last 32 of 4 x 8192: 46.9
    // against 49.3).  Chunks have two key tiles at least (1 x 4096 tokens, the last
    // one's account: 15.4 us, of four 17.4), and four row steps (1 x 1000: 38.5 us, of two
    // 41.5) or, where those are fewer than CUs, two (1 x 300: 21.9 against 24.7).
    const int64_t n = std::max(1, cus);
    int64_t       seen = 0, steps = 0, all = 0; // key tiles of all row tiles, row steps of all key blocks, row tiles
    for (const auto &e : plan.entries) {
        const int64_t rows = (int64_t)e.w * G;
        if (rows > INT32_MAX / 2) return false;
        const int64_t rt = (rows + kAccountRows - 1) / kAccountRows, kb = account_blocks(e.p0 + e.n);
        const int64_t st = (rows + kAccountStep - 1) / kAccountStep;
        all += rt;
        seen += rt * (account_seen(e, G, 0) + account_seen(e, G, (int)rt - 1)) / 2;
        steps += kb * st - std::min(kb, (e.w + kAccountKeys - 1) / (int64_t)kAccountKeys) * st / 2;
    }
    auto          ceil_div = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    const int64_t keys_each = std::max<int64_t>(2, ceil_div(seen * Hkv, (all * Hkv < n ? 2 : 3) * n));
    const int64_t rows_each = std::max<int64_t>(steps * Hkv >= 4 * n ? 4 : 2, ceil_div(steps * Hkv, 3 * n));
    // Pieces in the order of their items' lengths (cost), with their item0; the number of items.
    auto order = [&](std::vector<std::pair<int64_t, AccountPiece>> &cost, std::vector<AccountPiece> &out) {
        std::stable_sort(cost.begin(), cost.end(), [](const auto &x, const auto &y) { return x.first > y.first; });
        int64_t items = 0;
        for (auto &c : cost) {
            c.second.item0 = (int32_t)std::min<int64_t>(items, INT32_MAX);
            items += (int64_t)(c.second.last - c.second.first) * c.second.chunks();
            out.push_back(c.second);
        }
        return items;
    };
    plan.launches.clear();
    std::vector<std::pair<int64_t, AccountPiece>> tiles, blocks;
    for (size_t i = 0; i < plan.entries.size();) {
        AccountLaunch l{};
        l.first = (int)i;
        l.n = (int)std::min<size_t>(kAccountBatch, plan.entries.size() - i);
        l.fold = true;
        tiles.clear(), blocks.clear();
        const int pieces = kAccountPieces / l.n; // of an entry
        int64_t   fold_rows = 0, fold_parts = 0;
        for (int k = 0; k < l.n; ++k, ++i) {
            AccountEntry &e = plan.entries[i];
            const int     keys = e.p0 + e.n, rows = e.w * G;
            const int     rt = (rows + kAccountRows - 1) / kAccountRows, kb = account_blocks(keys);
            const int     st = (rows + kAccountStep - 1) / kAccountStep;
            e.nch = e.nrc = 1;
            for (int x = 0, lo = 0; x < pieces; ++x) {
                const int hi = (int)((int64_t)(x + 1) * rt / pieces);
                if (hi == lo) continue;
                const int64_t most = account_seen(e, G, hi - 1), c = ceil_div(most, keys_each);
                tiles.push_back({ceil_div(most, c), {0, lo, hi, (uint32_t)k | (uint32_t)c << 8}});
                e.nch = std::max(e.nch, (int)c);
                lo = hi;
            }
            int64_t chunk_rows = 0;
            for (int x = 0, lo = 0; x < pieces; ++x) {
                const int hi = (int)((int64_t)(x + 1) * kb / pieces);
                if (hi == lo) continue;
                const int64_t most = st - account_sees(e, G, lo), c = ceil_div(most, rows_each);
                blocks.push_back({ceil_div(most, c), {0, lo, hi, (uint32_t)k | (uint32_t)c << 8}});
                e.nrc = std::max(e.nrc, (int)c);
                chunk_rows = std::max(chunk_rows, ceil_div(most, c) * kAccountStep);
                lo = hi;
            }
            e.lse0 = (int32_t)l.lse;
            e.stat0 = (int32_t)l.stats;
            e.part0 = (int32_t)l.parts;
            l.lse += rows;
            if (e.nch > 1) l.stats += (int64_t)rows * e.nch;
            if (e.nrc > 1) l.parts += (int64_t)kb * kAccountKeys * e.nrc;
            if (std::max({l.lse, l.stats, l.parts}) > INT32_MAX) return false;
            l.split_keys |= e.nch > 1;
            l.split_rows |= e.nrc > 1;
            if (e.nch > 1) {
                l.most_rows = std::max(l.most_rows, rows);
                fold_rows = std::max(fold_rows, chunk_rows);
                fold_parts = std::max(fold_parts, chunk_rows * e.nch);
            }
            if (e.nrc > 1) l.most_keys = std::max(l.most_keys, keys);
        }
        l.fold = fold_rows <= kAccountFold && fold_parts <= kAccountFoldParts;
        const int64_t items = order(tiles, l.tile_pieces), sums = order(blocks, l.block_pieces);
        if (std::max(items, sums) * Hkv > INT32_MAX) return false;
        l.items = (int)items;
        l.sums = (int)sums;
        plan.launches.push_back(std::move(l));
    }
    return true;
}

bool plan_cross(CrossPlan &plan, int D, int G, int Hkv, int cus) {
    // 8 waves share a key tile among 256 rows and have a CU to themselves, 4 waves waste
    // fewer rows of a short entry, two workgroups to a CU.  Measured, 8 heads of 128, groups of 4,
    // 8 against 4 waves: 2 x 2048 queries over 8192 544 us, 584; 1 x 500 over 4096 55.6, 60.3;
    // 16 x 64 over 2048 61, 67.  One full round of large workgroups and a part of
    // another is worse: 4 x 512 over 2048 105, 77; 3 x 1024 over 4096 245, 229.  Level at 64.
    const int64_t n = std::max(1, cus);
    int64_t       rows = 0, large = 0;
    for (const auto &e : plan.entries) {
        rows += (int64_t)e.nq * G;
        large += ((int64_t)e.nq * G + cross_rows(D, 8) - 1) / cross_rows(D, 8);
    }
    const bool wide = cross_wide(D) && !plan.entries.empty() && rows >= 256 * (int64_t)plan.entries.size() &&
                      (large * Hkv < n || large * Hkv >= 2 * n);
    plan.waves = wide ? 8 : 4;
    const int tile = cross_rows(D, plan.waves);
    int64_t   tiles = 0;
    for (const auto &e : plan.entries) tiles += ((int64_t)e.nq * G + tile - 1) / tile;
    // Row tiles that do not fill the chip have their keys split, into chunks of at least
    // three tiles, once per CU (4 x 32 queries over 8192, 8 heads of 128, groups of 4:
    // 44.6 us, twice per CU 47.9; 500 over 4096: 57 against 79): a chunk's partial outputs
    // are written and read again.  Twice pays where half of a tile's rows are empty
    // (16 x 32 over 1500, 8 heads of 64: 18.5 against 20.3) or chunks stay long (64 over
    // 32768: 65.7 against 68.5).
    const int64_t work = std::max<int64_t>(1, tiles * Hkv);
    const int64_t once = std::max<int64_t>(1, n / work), twice = std::max<int64_t>(1, 2 * n / work);
    const bool    sparse = 2 * rows <= tiles * tile;
    for (auto &e : plan.entries) {
        const int64_t t = stream_tiles(e.S);
        e.nch = (int)std::max<int64_t>({1, std::min<int64_t>(once, t / 3), sparse ? std::min<int64_t>(twice, t / 4) : t >= 16 * twice ? twice : 1});
    }
    std::stable_sort(plan.entries.begin(), plan.entries.end(), [](const CrossEntry &x, const CrossEntry &y) {
        return (int64_t)x.S * y.nch > (int64_t)y.S * x.nch;
    });
    plan.launches.clear();
    for (size_t i = 0; i < plan.entries.size();) {
        CrossLaunch l{(int)i, 0, 0, false};
        int64_t     items = 0;
        for (; i < plan.entries.size() && l.n < kCrossBatch; ++i, ++l.n) {
            CrossEntry &e = plan.entries[i];
            e.item0 = (int32_t)items;
            items += ((int64_t)e.nq * G + tile - 1) / tile * e.nch;
            l.split |= e.nch > 1;
            if (items * Hkv > INT32_MAX) return false;
        }
        l.items = (int)items;
        plan.launches.push_back(l);
    }
    return true;
}

} // namespace detail
} // namespace tiny_llm
