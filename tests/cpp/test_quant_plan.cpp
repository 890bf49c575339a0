// The cache in 8 bits on the host, under sanitizers: the plans of its attention kernels cover
// every tile once, and the open group's tiles always hold the rows that are read or kept.
#include "quant_plan.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

using namespace tiny_llm::detail;

#define CHECK(c)                                                                                   \
    do {                                                                                           \
        if (!(c)) {                                                                                \
            std::fprintf(stderr, "check failed: %s (%s:%d)\n", #c, __FILE__, __LINE__);          \
            std::abort();                                                                          \
        }                                                                                          \
    } while (0)

static std::mt19937_64 rng(8);
static int             upto(int n) { return (int)(rng() % (uint64_t)(n + 1)); }

static void stream_random() {
    for (int it = 0; it < 2000; ++it) {
        const int D = 32 << upto(3), Hkv = 1 << upto(5), G = 1 << upto(3), cus = 1 + upto(300);
        const int n = it % 7 == 0 ? 0 : 1 + upto(it % 5 == 0 ? 400 : 40);
        QuantPlan p;
        for (int i = 0; i < n; ++i) {
            const int S = it % 3 == 0 ? upto(200000) : upto(700);
            p.entries.push_back({i, S, i, 1 + upto(kQuantRows / G - 1), S % kGroup ? 0 : -1, 0});
        }
        plan_quant(p, G, Hkv, D, cus);
        CHECK(p.chunk >= 1);
        std::vector<int> seen((size_t)n, 0);
        int              next = 0, longest = 1 << 30;
        for (const auto &l : p.launches) {
            CHECK(l.first == next && l.n <= kQuantBatch);
            next += l.n;
            int  items = 0;
            bool finish = false;
            for (int i = l.first; i < l.first + l.n; ++i) {
                const QuantEntry &e = p.entries[(size_t)i];
                seen[(size_t)e.row]++;
                const int tiles = quant_tiles(e.S), k = quant_items(e.S, p.chunk);
                CHECK(e.item0 == items && e.nq * G <= l.rows && l.rows <= kQuantRows);
                CHECK((k == 0) == (e.S == 0) && k <= tiles);
                int covered = 0;
                for (int ch = 0; ch < k; ++ch) {
                    const int lo = (int)((int64_t)ch * tiles / k), hi = (int)((int64_t)(ch + 1) * tiles / k);
                    CHECK(lo == covered && hi > lo && hi - lo <= p.chunk);
                    covered = hi;
                }
                CHECK(covered == tiles);
                if (k) {
                    CHECK((tiles + k - 1) / k <= longest);
                    longest = (tiles + k - 1) / k;
                }
                items += k;
                finish |= k != 1;
            }
            CHECK(items == l.items && finish == l.finish);
        }
        CHECK(next == n);
        for (int s : seen) CHECK(s == 1);
    }
    std::puts("ok stream_random");
}

static void prefill_random() {
    for (int it = 0; it < 2000; ++it) {
        const int D = 32 << upto(3), Hkv = 1 << upto(5), G = 1 << upto(3), cus = 1 + upto(300);
        const int n = it % 7 == 0 ? 0 : 1 + upto(it % 5 == 0 ? 300 : 20);
        QuantPrefillPlan p;
        for (int i = 0; i < n; ++i) {
            const int nq = 1 + upto(it % 3 == 0 ? 20000 : 300), S = nq + (it % 2 ? upto(100000) : 0);
            p.entries.push_back({i, S, i, nq, S % kGroup ? 1 : -1, 1, 0});
        }
        CHECK(plan_quant_prefill(p, D, G, Hkv, cus));
        const int        rows = quant_prefill_rows(D);
        std::vector<int> seen((size_t)n, 0);
        int              next = 0;
        for (const auto &l : p.launches) {
            CHECK(l.first == next && l.n <= kQuantPrefillBatch);
            next += l.n;
            int64_t items = 0;
            int64_t parts = 0;
            for (int i = l.first; i < l.first + l.n; ++i) {
                const QuantPrefillEntry &e = p.entries[(size_t)i];
                seen[(size_t)e.row]++;
                CHECK(e.item0 == items && e.nch >= 1);
                items += ((int64_t)e.nq * G + rows - 1) / rows * e.nch;
                if (e.nch > 1) parts = items;
            }
            CHECK(items == l.items && parts == l.parts);
        }
        CHECK(next == n);
        for (int s : seen) CHECK(s == 1);
    }
    QuantPrefillPlan p;
    p.entries.push_back({0, 1 << 30, 0, 1 << 30, -1, 1, 0});
    CHECK(!plan_quant_prefill(p, 128, 8, 128, 256)); // more threads than a launch has
    std::puts("ok prefill_random");
}

// What the kernels do with the tiles, by stamps of the rows.
struct Slot {
    OpenGroup        open;
    int              len = 0;
    std::vector<int> want;                                // stamp of every held token
    int              tile[2][kGroup], group[2] = {-1, -1}; // stamps in the tiles
    std::vector<int> closed;                              // stamps of the closed groups' tokens
};

static void append(Slot &s, int n, int stamp) {
    const auto [first, last] = s.open.tiles(s.len, n);
    const int end = s.len + n;
    s.want.resize((size_t)s.len);
    for (int t = s.len; t < end; ++t) s.want.push_back(stamp + t);
    s.closed.resize((size_t)std::max<size_t>(s.closed.size(), (size_t)(end / kGroup * kGroup)), -1);
    for (int g = s.len / kGroup; g * kGroup < end; ++g) {
        int rows[kGroup];
        std::fill(rows, rows + kGroup, -1);
        if (g == s.len / kGroup && s.len % kGroup) {
            std::copy(s.tile[first], s.tile[first] + kGroup, rows);
            CHECK(s.group[first] == g);
        }
        for (int r = 0; r < kGroup; ++r)
            if (g * kGroup + r >= s.len && g * kGroup + r < end) rows[r] = stamp + g * kGroup + r;
        const bool opens = g == s.len / kGroup, whole = (g + 1) * kGroup <= end;
        if (opens || !whole) {
            const int w = opens ? first : last;
            std::copy(rows, rows + kGroup, s.tile[w]);
            s.group[w] = g;
        }
        if (whole) std::copy(rows, rows + kGroup, s.closed.begin() + g * kGroup);
    }
    s.open.append(s.len, n);
}

// Every token up to S as a read finds it, `held` tokens being there and the last group in `tile`.
static void check_read(const Slot &s, int S, int held, int tile) {
    for (int t = 0; t < S; ++t) {
        if (t < held / kGroup * kGroup) {
            if (t / kGroup * kGroup + kGroup <= s.len || S > s.len) CHECK(s.closed[(size_t)t] == s.want[(size_t)t]);
        } else {
            CHECK(s.group[tile] == t / kGroup && s.tile[tile][t % kGroup] == s.want[(size_t)t]);
        }
    }
}

static void open_group_random() {
    int refused = 0, cut = 0;
    for (int it = 0; it < 3000; ++it) {
        Slot s;
        for (int step = 0; step < 60; ++step) {
            const int kinds[] = {1, 1, 1, 1 + upto(8), 1 + upto(70), 32 * (1 + upto(3)), 1 + upto(300)};
            const int n = kinds[upto(6)], stamp = (step + 1) * 1000000;
            append(s, n, stamp);
            if (upto(5) == 0) append(s, n, stamp + 500000); // the same again, replaced
            const auto [held, tile] = s.open.held(s.len);
            CHECK(held == (int)s.want.size());
            check_read(s, held, held, tile);
            check_read(s, s.len, s.len, s.open.cur); // what was advanced over is still there
            for (int parts = 0; parts < 2; ++parts) {
                const int left = (int)s.want.size() - s.len;
                if (!left) break;
                const int  k = upto(2) ? left : 1 + upto(left - 1), to = s.len + k;
                OpenGroup  before = s.open;
                const bool ok = s.open.advance(s.len, to);
                const bool must = to % kGroup == 0 || to / kGroup == s.len / kGroup || to / kGroup == (int)s.want.size() / kGroup;
                if (parts == 0) CHECK(ok == must);
                if (!ok) {
                    ++refused;
                    CHECK(before.cur == s.open.cur && before.end == s.open.end && before.group[0] == s.open.group[0] &&
                          before.group[1] == s.open.group[1]);
                    continue;
                }
                cut += k < left;
                s.len = to;
                check_read(s, s.len, s.len, s.open.cur);
                const auto [h2, t2] = s.open.held(s.len);
                CHECK(h2 == (int)s.want.size());
                check_read(s, h2, h2, t2);
            }
        }
    }
    CHECK(refused > 1000 && cut > 1000);
    OpenGroup o; // beyond what was appended: any length
    CHECK(o.advance(0, 50) && o.advance(50, 51) && o.advance(51, 64) && o.advance(64, 200));
    std::puts("ok open_group_random");
}

int main() {
    stream_random();
    prefill_random();
    open_group_random();
    return 0;
}
