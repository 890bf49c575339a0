// The open group of a cache in 8 bits on the host, under sanitizers, beside what an fp16 cache holds
// after the same calls: a length that is accepted shows every token that the fp16 cache shows.
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

static std::mt19937_64 rng(9);
static int             upto(int n) { return (int)(rng() % (uint64_t)(n + 1)); }

constexpr int kRoom = 4096;

// One layer's memory, by stamps of the rows (0: never written), as the append kernels leave it.
struct Memory {
    std::vector<int> fp16 = std::vector<int>(kRoom);   // of an fp16 cache
    std::vector<int> closed = std::vector<int>(kRoom); // in 8 bits
    int              tile[2][kGroup] = {};

    // n tokens from p0 on, the open tiles of its first and of its last group as they were prepared
    void append(int p0, int n, int first, int last, int stamp) {
        const int end = p0 + n;
        for (int t = p0; t < end; ++t) fp16[(size_t)t] = stamp + t;
        for (int g = p0 / kGroup; g * kGroup < end; ++g) {
            const int lo = std::max(p0, g * kGroup), hi = std::min(end, (g + 1) * kGroup), base = g * kGroup;
            const bool opens = g == p0 / kGroup, closes = (g + 1) * kGroup <= end;
            int        rows[kGroup];
            std::copy(tile[first], tile[first] + kGroup, rows);
            for (int t = lo; t < hi; ++t) rows[t - base] = stamp + t;
            if (closes) std::copy(rows, rows + kGroup, closed.begin() + base);
            if (opens || !closes)
                for (int t = lo; t < hi; ++t) tile[opens ? first : last][t - base] = stamp + t;
        }
    }
    // The first len tokens, read as a batch of that length reads them.
    void check(int len, int cur) const {
        for (int t = 0; t < len; ++t) {
            const int got = t < len / kGroup * kGroup ? closed[(size_t)t] : tile[cur][t % kGroup];
            if (fp16[(size_t)t]) CHECK(got == fp16[(size_t)t]);
        }
    }
};

static void append(OpenGroup &o, Memory &m, int len, int n, int stamp) {
    const auto [first, last] = o.tiles(len, n);
    m.append(len, n, first, last, stamp);
    o.append(len, n);
}

static void advance_beyond_what_was_appended() {
    int kept = 0, refused = 0;
    for (int it = 0; it < 4000; ++it) {
        OpenGroup o;
        Memory    m;
        int       len = 0;
        for (int step = 0; step < 30; ++step) {
            const int n = upto(3) ? 1 + upto(60) : 32 - len % 32; // (also to a group's end)
            if (len + n + 200 > kRoom) break;
            append(o, m, len, n, (step + 1) * 10000);
            const int  end = len + n, to = end + (upto(2) ? 0 : 1 + upto(80));
            OpenGroup  before = o;
            const bool ok = o.advance(len, to);
            // Only rows that wait in fp16 can be left behind.
            CHECK(ok == (to == end || end % kGroup == 0 || to / kGroup == end / kGroup));
            if (!ok) {
                ++refused;
                CHECK(before.cur == o.cur && before.end == o.end && before.group[0] == o.group[0] && before.group[1] == o.group[1]);
                CHECK(o.advance(len, end));
                len = end;
            } else {
                kept += to > end;
                len = to;
            }
            m.check(len, o.cur);
        }
    }
    CHECK(kept > 1000 && refused > 1000);
    // 20 tokens that were advanced over, then 20 that nobody brought.
    OpenGroup o;
    o.append(0, 20);
    CHECK(o.advance(0, 20) && !o.advance(20, 40) && o.advance(20, 31) && !o.advance(31, 32));
    std::puts("ok advance_beyond_what_was_appended");
}

// Several batches append at one length, in any order, and one of them commits.
static void advance_over_another_append() {
    int ok = 0, refused = 0, replaced = 0;
    for (int it = 0; it < 40000; ++it) {
        OpenGroup o;
        Memory    m;
        int       len = upto(100), last = 0, most = 0;
        append(o, m, 0, len + 1, 1000);
        CHECK(o.advance(0, ++len));
        int n[4];
        for (int k = 0; k < 4; ++k) n[k] = upto(1) ? 1 + upto(8) : 1 + upto(90);
        for (int k = 0, count = 1 + upto(4); k < count; ++k) {
            last = n[upto(3)];
            most = std::max(most, last);
            append(o, m, len, last, (k + 2) * 10000);
        }
        const int to = len + n[upto(3)];
        // What an append brought again may be less than what was there before: the rest is gone.
        const bool gone = to > len + last && to <= len + most;
        const bool done = o.advance(len, to);
        if (gone) {
            CHECK(!done);
            ++replaced;
        }
        if (to == len + last) CHECK(done);
        if (!done) {
            ++refused;
            continue;
        }
        ++ok;
        m.check(to, o.cur);
    }
    CHECK(ok > 5000 && refused > 5000 && replaced > 5000);
    std::puts("ok advance_over_another_append");
}

// Batches that append to some of the layers only: every layer has to have had the same.
static void advance_where_layers_differ() {
    constexpr int L = 3;
    int           ok = 0, refused = 0;
    for (int it = 0; it < 40000; ++it) {
        OpenGroup o;
        Memory    m[L];
        int       ends[L] = {}, len = 1 + upto(100);
        auto      add = [&](int at, int n, unsigned layers, int stamp) {
            const auto [first, last] = o.tiles(at, n);
            for (int l = 0; l < L; ++l)
                if (layers >> l & 1) m[l].append(at, n, first, last, stamp + 1000 * l), ends[l] = at + n;
            o.append(at, n);
        };
        add(0, len + (upto(1) ? 0 : upto(90)), 7, 10000);
        if (!o.alike(ends, L, 0, len) || !o.advance(0, len)) continue; // (an inside length)
        int last = 0;
        for (int k = 0, count = 1 + upto(3); k < count; ++k) {
            last = 1 + upto(upto(1) ? 8 : 90);
            add(len, last, upto(1) ? 7u : 1u + (unsigned)upto(6), (k + 2) * 10000);
            if (upto(2) == 0) { // the same, in all of them
                add(len, last, 7, (k + 2) * 10000);
                CHECK(o.alike(ends, L, len, len + last));
            }
        }
        if (!o.alike(ends, L, len, len + last) || !o.advance(len, len + last)) {
            ++refused;
            continue;
        }
        ++ok;
        for (int l = 0; l < L; ++l) m[l].check(len + last, o.cur);
    }
    CHECK(ok > 5000 && refused > 5000);
    std::puts("ok advance_where_layers_differ");
}

int main() {
    advance_beyond_what_was_appended();
    advance_over_another_append();
    advance_where_layers_differ();
    return 0;
}
