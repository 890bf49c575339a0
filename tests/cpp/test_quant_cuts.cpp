// How plan_quant and plan_quant_prefill cut the work, on the host under sanitizers.  Prompts have their keys cut
// by one length for all of them, into no more chunks than there are tiles, within the slots where the row tiles
// are, and only where that is so; steps as was measured faster.
#include "quant_plan.h"

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>

using namespace tiny_llm::detail;

#define CHECK(c)                                                                                   \
    do {                                                                                           \
        if (!(c)) {                                                                                \
            std::fprintf(stderr, "check failed: %s (%s:%d)\n", #c, __FILE__, __LINE__);          \
            std::abort();                                                                          \
        }                                                                                          \
    } while (0)

static std::mt19937_64 rng(10);
static int             upto(int n) { return (int)(rng() % (uint64_t)(n + 1)); }

static void prefill_cuts() {
    int cut = 0, whole = 0, some = 0, fits = 0, rounds = 0;
    for (int it = 0; it < 6000; ++it) {
        const int D = 32 << upto(3), Hkv = 1 << upto(5), G = 1 << upto(3), cus = it % 2 ? 256 : 1 + upto(300);
        const int n = 1 + upto(it % 5 == 0 ? 150 : it % 5 == 1 ? 0 : 16);
        const int far = 1 << (6 + upto(12)), many = 1 << (5 + upto(7));
        QuantPrefillPlan p;
        for (int i = 0; i < n; ++i) {
            const int nq = 1 + upto(many), S = nq + upto(far);
            p.entries.push_back({i, S, i, nq, S % kGroup ? 1 : -1, 1, 0});
        }
        CHECK(plan_quant_prefill(p, D, G, Hkv, cus));
        const int64_t slots = (int64_t)cus * quant_prefill_per_cu(D);
        const int     tile = quant_prefill_tile(D), rows = quant_prefill_rows(D);
        int64_t       row_tiles = 0, items = 0, work = 0, longest = 0, shortest_cut = 0;
        int           most = 1, least = 1 << 30;
        for (const auto &e : p.entries) {
            const int64_t keys = (e.S + (int64_t)tile - 1) / tile, r = ((int64_t)e.nq * G + rows - 1) / rows;
            CHECK(e.nch >= 1 && e.nch <= keys);
            row_tiles += r * Hkv;
            items += r * e.nch * Hkv;
            work += r * keys * Hkv;
            longest = std::max(longest, keys);
            // the lengths by which this entry is cut into nch: from ceil(keys / nch) on
            shortest_cut = std::max(shortest_cut, (keys + e.nch - 1) / e.nch);
            most = std::max(most, e.nch);
            least = std::min(least, e.nch);
        }
        for (const auto &e : p.entries) { // one length does for all
            const int64_t keys = (e.S + (int64_t)tile - 1) / tile;
            CHECK((keys + shortest_cut - 1) / shortest_cut == e.nch);
        }
        if (row_tiles <= slots) {
            ++fits;
            CHECK(items <= slots);
            // Chunks a sixth of the longest entry would be cut, and those would have slots: then they are cut.
            int64_t six = 0;
            const int64_t c = std::max<int64_t>(3, longest / 6);
            for (const auto &e : p.entries)
                six += ((int64_t)e.nq * G + rows - 1) / rows * (((e.S + (int64_t)tile - 1) / tile + c - 1) / c) * Hkv;
            if (six <= slots && longest >= 12) CHECK(most > 1);
            if (longest < 9) CHECK(most == 1);
        } else {
            ++rounds;
            // No chunk is shorter than the chip's whole work, and nothing is cut that is not half as long again.
            const int64_t share = (work + slots - 1) / slots;
            if (most > 1) CHECK(longest >= share + share / 2 && longest >= share + 6);
            if (longest >= 2 * share + 6 && longest >= 9) CHECK(most > 1);
        }
        cut += most > 1;
        whole += most == 1;
        some += most > 1 && least == 1;
    }
    CHECK(cut > 1000 && whole > 1000 && some > 300 && fits > 1000 && rounds > 1000);
    std::puts("ok prefill_cuts");
}

// Decode entries of one length on 256 CUs: whole, or in so many chunks, as was measured faster.
static void decode_sides() {
    const struct { int D, Hkv, n, S, items; } sides[] = {
        {32, 8, 1, 1000, 1},   {64, 8, 1, 1000, 1},   {128, 8, 1, 1000, 1},  {256, 8, 1, 1000, 4},
        {32, 8, 1, 4000, 8},   {64, 8, 1, 4000, 8},   {128, 8, 1, 4000, 8},  {256, 8, 1, 4000, 16},
        {32, 8, 16, 1000, 1},  {64, 8, 16, 1000, 1},  {128, 8, 16, 1000, 1}, {256, 8, 16, 1000, 1},
        {32, 8, 16, 2000, 1},  {64, 8, 16, 2000, 1},  {128, 8, 16, 2000, 1}, {128, 8, 16, 4000, 1},
        {32, 8, 16, 8000, 2},  {64, 8, 16, 8000, 2},  {128, 8, 16, 8000, 2}, {256, 8, 16, 8000, 2},
        {32, 8, 28, 6000, 1},  {64, 8, 28, 6000, 1},  {128, 8, 28, 6000, 1}, {256, 8, 24, 6000, 1},
        {32, 2, 70, 3000, 1},  {128, 2, 70, 3000, 1}, {256, 2, 70, 3000, 1}, {256, 1, 100, 8000, 2},
    };
    for (const auto &x : sides) {
        QuantPlan p;
        for (int i = 0; i < x.n; ++i) p.entries.push_back({i, x.S + 1, i, 1, 0, 0});
        plan_quant(p, 4, x.Hkv, x.D, 256);
        if (quant_items(x.S + 1, p.chunk) != x.items) std::fprintf(stderr, "head_dim %d, %d x %d of %d heads\n", x.D, x.n, x.S, x.Hkv);
        CHECK(quant_items(x.S + 1, p.chunk) == x.items);
    }
    std::puts("ok decode_sides");
}

int main() {
    prefill_cuts();
    decode_sides();
    return 0;
}
