// How the work of the account and cross attention kernels is cut
// (tiny-llm_amd/csrc/stream_plan.cpp), and the block allocator's shrink, on random
// and extreme inputs under the address and undefined-behaviour sanitizers (built by
// tests/test_retention_cpu.py with g++, no GPU).
#include "block_allocator.h"
#include "stream_plan.h"

#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

using namespace tiny_llm::detail;

#define CHECK(c)                                                                                                       \
    do {                                                                                                               \
        if (!(c)) {                                                                                                    \
            std::fprintf(stderr, "check failed: %s (%s:%d)\n", #c, __FILE__, __LINE__);                              \
            std::abort();                                                                                              \
        }                                                                                                              \
    } while (0)

static void stream_random() {
    std::mt19937_64 rng(1);
    for (int it = 0; it < 500; ++it) {
        StreamPlan p;
        const int  n = (int)(rng() % 400), most = 1 << (rng() % 17);
        for (int i = 0; i < n; ++i) p.entries.push_back({i, rng() % 9 ? (int32_t)(rng() % most) : 0, i, 1, -1, -1});
        if (it % 50 == 0 && n) p.entries[0].S = INT32_MAX;
        const int D = 32 << (rng() % 4);
        const int rows = (int)(rng() % 2) ? 1 << (rng() % 4) : 0;
        plan_stream(p, 1 << (rng() % 6), D, rows, 1 + (int)(rng() % 300));
        CHECK(p.chunk >= 1 && (p.waves == 4 || (p.waves == 8 && D <= 128)));
        auto length = [&](const StreamEntry &e) {
            const int k = stream_items(e.S, p.chunk);
            return k ? (stream_tiles(e.S) + k - 1) / k : 0;
        };
        for (size_t i = 1; i < p.entries.size(); ++i) CHECK(length(p.entries[i]) <= length(p.entries[i - 1]));
        size_t next = 0;
        for (const auto &l : p.launches) {
            CHECK((size_t)l.first == next && l.n > 0 && l.n <= kStreamBatch);
            int     items = 0, longest = 0;
            bool    finish = false;
            int64_t tiles = 0;
            for (int i = l.first; i < l.first + l.n; ++i) {
                const StreamEntry &e = p.entries[(size_t)i];
                const int          t = stream_tiles(e.S), k = stream_items(e.S, p.chunk);
                CHECK(e.item0 == items && e.tile0 == tiles);
                CHECK((int64_t)t * kStreamTile >= e.S && (int64_t)(t - 1) * kStreamTile < e.S);
                CHECK((k == 0) == (e.S == 0));
                // the kernel's chunks: every tile once, none empty
                int64_t at = 0;
                for (int c = 0; c < std::min(k, 50); ++c) {
                    const int64_t lo = (int64_t)c * t / k, hi = (int64_t)(c + 1) * t / k;
                    CHECK(lo == at && hi > lo && hi - lo <= p.chunk);
                    at = hi;
                }
                if (k <= 50) CHECK(at == t);
                items += k;
                tiles += t;
                if (k > 1) longest = std::max(longest, (int)e.S);
                finish |= k != 1;
            }
            // the kernel's search: the last entry that starts at or before the item
            for (int item = 0; item < std::min(items, 200); ++item) {
                int found = -1;
                for (int j = l.first; j < l.first + l.n; ++j)
                    if (p.entries[(size_t)j].item0 <= item) found = j;
                const StreamEntry &e = p.entries[(size_t)found];
                CHECK(item - e.item0 >= 0 && item - e.item0 < stream_items(e.S, p.chunk));
            }
            CHECK(l.items == items && l.tiles == tiles && l.max_len == longest && l.finish == finish);
            next += (size_t)l.n;
        }
        CHECK(next == p.entries.size());
        // what the kernel keeps in LDS fits
        int item = 0;
        for (const auto &e : p.entries) {
            const int64_t t = stream_tiles(e.S), k = stream_items(e.S, p.chunk);
            for (int64_t c = 0; c < std::min<int64_t>(k, 50); ++c) item = std::max(item, (int)((c + 1) * t / k - c * t / k));
        }
        CHECK(item <= p.most && p.most <= p.chunk);
        if (rows) CHECK((int64_t)p.waves * stream_stage_bytes(D, true) + (int64_t)p.most * kStreamTile * rows * 4 <= kStreamLds);
    }
    std::puts("ok stream_random");
}

static void account_random() {
    std::mt19937_64 rng(2);
    for (int it = 0; it < 500; ++it) {
        AccountPlan p;
        const int   n = (int)(rng() % 150), most = 1 << (rng() % 14), G = 1 << (rng() % 4);
        for (int i = 0; i < n; ++i) {
            const int    nt = 1 + (int)(rng() % most), w = rng() % 2 ? nt : 1 + (int)(rng() % nt);
            AccountEntry e{};
            e.row = i, e.p0 = (int32_t)(rng() % most), e.n = nt, e.w = w;
            p.entries.push_back(e);
        }
        CHECK(plan_account(p, G, 1 << (rng() % 6), 1 + (int)(rng() % 300)));
        size_t next = 0;
        for (const auto &l : p.launches) {
            CHECK((size_t)l.first == next && l.n > 0 && l.n <= kAccountBatch);
            CHECK((int)l.tile_pieces.size() <= kAccountPieces && (int)l.block_pieces.size() <= kAccountPieces);
            int64_t items = 0, sums = 0, stats = 0, lse = 0, parts = 0;
            bool    keys_split = false, rows_split = false;
            for (int i = 0; i < l.n; ++i) {
                const AccountEntry &e = p.entries[next + (size_t)i];
                const int           keys = e.p0 + e.n, rows = e.w * G;
                CHECK(e.stat0 == stats && e.lse0 == lse && e.part0 == parts);
                // every row tile and every key block in one piece
                std::vector<int> tile(((size_t)rows + kAccountRows - 1) / kAccountRows), block((size_t)account_blocks(keys));
                int              nch = 1, nrc = 1;
                for (const auto &c : l.tile_pieces) {
                    if (c.entry() != i) continue;
                    CHECK(c.first >= 0 && c.first < c.last && c.last <= (int)tile.size());
                    CHECK(c.chunks() >= 1 && c.chunks() <= account_seen(e, G, c.last - 1));
                    for (int x = c.first; x < c.last; ++x) ++tile[(size_t)x];
                    nch = std::max(nch, c.chunks());
                }
                for (const auto &c : l.block_pieces) {
                    if (c.entry() != i) continue;
                    CHECK(c.first >= 0 && c.first < c.last && c.last <= (int)block.size());
                    const int steps = (rows + kAccountStep - 1) / kAccountStep - account_sees(e, G, c.first);
                    CHECK(c.chunks() >= 1 && c.chunks() <= steps);
                    CHECK(!l.fold || e.nch == 1 || (steps + c.chunks() - 1) / c.chunks() * kAccountStep <= kAccountFold);
                    for (int x = c.first; x < c.last; ++x) ++block[(size_t)x];
                    nrc = std::max(nrc, c.chunks());
                }
                for (int x : tile) CHECK(x == 1);
                for (int x : block) CHECK(x == 1);
                CHECK(e.nch == nch && e.nrc == nrc);
                lse += rows;
                if (e.nch > 1) stats += (int64_t)rows * e.nch;
                CHECK(e.nch == 1 || rows <= l.most_rows);
                if (e.nrc > 1) parts += (int64_t)account_blocks(keys) * kAccountKeys * e.nrc;
                CHECK(e.nrc == 1 || keys <= l.most_keys);
                keys_split |= e.nch > 1;
                rows_split |= e.nrc > 1;
            }
            for (const auto &c : l.tile_pieces) {
                CHECK(c.item0 == items);
                items += (int64_t)(c.last - c.first) * c.chunks();
            }
            for (const auto &c : l.block_pieces) {
                CHECK(c.item0 == sums);
                sums += (int64_t)(c.last - c.first) * c.chunks();
            }
            CHECK(l.items == items && l.sums == sums && l.stats == stats && l.lse == lse && l.parts == parts);
            CHECK(l.split_keys == keys_split && l.split_rows == rows_split);
            next += (size_t)l.n;
        }
        CHECK(next == p.entries.size());
    }
    AccountPlan big; // rows that do not fit 31 bits
    for (int i = 0; i < 5; ++i) {
        AccountEntry e{};
        e.row = i, e.n = e.w = 1 << 26;
        big.entries.push_back(e);
    }
    CHECK(!plan_account(big, 8, 8, 256));
    std::puts("ok account_random");
}

static void cross_random() {
    std::mt19937_64 rng(4);
    const int       dims[] = {32, 64, 128, 256};
    for (int it = 0; it < 500; ++it) {
        CrossPlan p;
        const int n = (int)(rng() % 300), most = 1 << (rng() % 17), longest = 1 << (rng() % 12);
        const int G = 1 << (rng() % 4), D = dims[rng() % 4], hkv = 1 << (rng() % 6);
        for (int i = 0; i < n; ++i)
            p.entries.push_back({i, 1 + (int32_t)(rng() % most), i, 1 + (int32_t)(rng() % longest), -1, -1});
        CHECK(plan_cross(p, D, G, hkv, 1 + (int)(rng() % 300)));
        CHECK(p.waves == 4 || (p.waves == 8 && D <= 128));
        std::set<int> rows;
        size_t        next = 0;
        for (const auto &l : p.launches) {
            CHECK((size_t)l.first == next && l.n > 0 && l.n <= kCrossBatch);
            int64_t items = 0;
            bool    split = false;
            for (int i = l.first; i < l.first + l.n; ++i) {
                const CrossEntry &e = p.entries[(size_t)i];
                CHECK(rows.insert(e.row).second && e.tok0 == e.row);
                CHECK(e.item0 == items && e.nch >= 1 && e.nch <= stream_tiles(e.S)); // no chunk is empty
                if (i > 0) {
                    const CrossEntry &b = p.entries[(size_t)i - 1];
                    CHECK((int64_t)b.S * e.nch >= (int64_t)e.S * b.nch);
                }
                const int tile = cross_rows(D, p.waves);
                items += ((int64_t)e.nq * G + tile - 1) / tile * e.nch;
                split |= e.nch > 1;
            }
            CHECK(l.items == items && l.split == split);
            next += (size_t)l.n;
        }
        CHECK(next == p.entries.size());
    }
    CrossPlan big;
    for (int i = 0; i < 3; ++i) big.entries.push_back({i, 1, 0, 1 << 28, 1, 0});
    CHECK(!plan_cross(big, 256, 8, 1024, 256));
    std::puts("ok cross_random");
}

static void allocator_shrink() {
    std::mt19937_64 rng(3);
    BlockAllocator  a(5, 9, 20);
    for (int it = 0; it < 4000; ++it) {
        const int row = (int)(rng() % 7) - 1, k = (int)(rng() % 11) - 1;
        const int had = row >= 0 && row < 5 ? a.mapped(row) : 0, free_before = a.freeBlocks();
        if (rng() % 2) {
            a.shrink(row, k);
            const bool acts = row >= 0 && row < 5 && k >= 0 && k < had;
            CHECK(a.freeBlocks() == free_before + (acts ? had - k : 0));
            if (row >= 0 && row < 5) CHECK(a.mapped(row) == (acts ? k : had));
        } else {
            a.ensure(row, k);
        }
        std::set<int32_t> used;
        for (int r = 0; r < 5; ++r)
            for (int j = 0; j < 9; ++j) {
                const int32_t b = a.table()[(size_t)(r * 9 + j)];
                if (j < a.mapped(r)) CHECK(b >= 0 && b < 20 && used.insert(b).second);
                else CHECK(b == a.spare());
            }
        CHECK((int)used.size() + a.freeBlocks() == 20);
        // the device copy follows by the updates alone
        static std::vector<int32_t> copy(45, a.spare());
        for (const auto &u : a.takeUpdates()) copy[(size_t)u.first] = u.second;
        CHECK(copy == a.table());
    }
    std::puts("ok allocator_shrink");
}

int main() {
    stream_random();
    account_random();
    cross_random();
    allocator_shrink();
    return 0;
}
