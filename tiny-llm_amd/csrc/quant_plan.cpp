#include "quant_plan.h"

#include <algorithm>

namespace tiny_llm {
namespace detail {

void plan_quant(QuantPlan &plan, int G, int Hkv, int D, int cus) {
    int64_t total = 0, longest = 0, some = 0;
    for (const auto &e : plan.entries) {
        total += quant_tiles(e.S);
        some += e.S > 0;
        longest = std::max<int64_t>(longest, quant_tiles(e.S));
    }
    // A workgroup that has a whole entry finishes it; entries in chunks need a second launch, about 3 us
    // more.  In hundredths of a us: a tile takes a CU `alone`, whether one workgroup or two are on it (what 1 x 4000
    // takes whole more than 1 x 2000), and the chip 60 of a CU's share at head_dim 128, a quarter more where half of
    // the CUs have none, a sixth more where some have one workgroup and others two.  Chunks are the shortest ones that
    // give every CU one workgroup at most, or two: a few workgroups beyond that would leave their CUs alone with twice
    // the work.  Beyond two the chip's share is all that counts.
    // Measured, 8 heads, groups of 4, caches beyond the last level's size, us whole and in the shortest chunks of at
    // most one a CU, of at most two, * what is taken (more of them: profiles/quantized_plan_sides.txt):
    //   head_dim          32                  64                  128                 256
    //   1 x 1000          7.4*  9.3  9.5      9.0* 10.7 10.9      12.5* 13.3 13.7     21.0  16.8* 17.1
    //   1 x 4000          15.1  9.9* 10.0     18.7 11.2* 11.2     27.0  13.8* 14.0    49.7  17.6* 17.7
    //   16 x 1000         8.1* 10.4 10.6      10.0* 12.4 12.5     14.9* 17.6 18.0     23.5* 26.0  32.7
    //   16 x 2000         10.7* 12.2 12.2     13.4* 14.7 14.9     20.9* 23.4 25.9     31.6  32.8* 38.0
    //   16 x 4000         15.7 14.6* 15.8     19.5 20.3* 21.5     32.3* 34.5 39.2     54.2  55.9* 60.9
    //   16 x 8000         25.9 19.6* 20.3     32.6 29.3* 29.8     52.7 49.6* 54.7     95.9  87.6* 91.3
    //   16 x 16000        45.4 30.4* 29.9     57.9 48.9* 48.3     97.4 95.0* 92.8     180   165*  167
    //   28 x 6000         21.4* -    24.3     33.7* -   35.4      62.1* -    65.8     117*  -     117
    //   40 x 600 .. 8000  26.0* -    24.6     41.7 -    38.2*     66.6 -     64.0*    134   -     131*
    //   60 x 600 .. 8000  32.7* -    35.1     53.9* -   55.3      92.6 -     95.2*    172   -     165*
    // With 28 for head_dim 32 and 64 and 112 for 256, 16 x 2000 took the chunks at 32 and 64, 16 x 1000 at 256, and
    // 70 x 3000 of 2 heads of 256 two a CU, 52.6 for 43.3.  Chunks of a CU's share, however many, and these: 10 x 100 ..
    // 30000 76, 64; head_dim 64 4 x 28000 .. 32000 34.4, 26.6; 256 16 x 500 .. 20000 133, 112.
    const int64_t n = std::max(1, cus), work = some * Hkv, waves = quant_waves(D);
    const int64_t share = (total * Hkv + n - 1) / n;
    const int64_t alone = D == 32 ? 16 : D == 64 ? 20 : D == 128 ? 28 : 72, stream = std::max<int64_t>(1, 60 * D / 128);
    int64_t       chunk = longest;
    int64_t       least = work <= n ? std::max(alone * longest, stream * total * Hkv / n * (4 * n - work) / (3 * n))
                                    : longest * std::max(alone, stream * 7 / 6);
    auto consider = [&](int64_t c, int64_t per_cu) {
        const int64_t takes = (c < longest ? 300 : 0) + std::max(alone * per_cu * c, stream * share);
        if (takes < least) {
            least = takes;
            chunk = c;
        }
    };
    for (int64_t k = 1; k <= 2 && work > 0; ++k) {
        if (work > k * n) continue;
        int64_t lo = std::min(waves, longest), hi = longest; // the shortest chunks of which there are at most k n
        while (lo < hi) {
            const int64_t c = (lo + hi) / 2;
            int64_t       items = 0;
            for (const auto &e : plan.entries) items += quant_items(e.S, (int)std::min<int64_t>(c, 1 << 24));
            if (items * Hkv <= k * n) hi = c;
            else lo = c + 1;
        }
        consider(lo, k);
    }
    if (work > 2 * n) consider(std::max(waves, share), 1);
    // More entries than workgroups of all waves fit at once (one a CU, two where registers are few), and short ones:
    // workgroups of two waves, four times as many. 33 x 32 heads of 128, to 64 tokens 13.8 us, 26.4 with eight
    // waves, to 800 38.6 and 51.7, to 1500 61.6 and 72.5, to 3000 113 and 110; 90 x 8 9.7 and 19.3, 22.9 and 34.2, 40.9
    // and 47.0, 79.9 and 74.7; 33 x 32 of 64 7.5 and 13.1, 17.4 and 24.1, 30.4 and 32.3, 61 and 53.  As many as fit: 32 x 8
    // of 128, to 300 tokens 9.9 and 8.1.
    plan.small = longest <= 20 && work > n * (D <= 64 ? 2 : 1);
    plan.chunk = (int)std::max<int64_t>(1, std::min<int64_t>(chunk, 1 << 24));
    auto item_tiles = [&](const QuantEntry &e) {
        const int k = quant_items(e.S, plan.chunk);
        return k ? (quant_tiles(e.S) + k - 1) / k : 0;
    };
    std::stable_sort(plan.entries.begin(), plan.entries.end(),
                     [&](const QuantEntry &x, const QuantEntry &y) { return item_tiles(x) > item_tiles(y); });
    plan.launches.clear();
    for (size_t i = 0; i < plan.entries.size();) {
        QuantLaunch l{(int)i, 0, 0, 1, false};
        for (; i < plan.entries.size() && l.n < kQuantBatch; ++i, ++l.n) {
            QuantEntry &e = plan.entries[i];
            const int   items = quant_items(e.S, plan.chunk);
            e.item0 = l.items;
            l.items += items;
            l.rows = std::max(l.rows, e.nq * G);
            l.finish |= items != 1;
        }
        plan.launches.push_back(l);
    }
}

bool plan_quant_prefill(QuantPrefillPlan &plan, int D, int G, int Hkv, int cus) {
    // Row tiles that leave workgroup slots empty have their keys split over them, in chunks of one length, of
    // three tiles at least, where the longest gets six shorter (8 heads of 128, groups of 4: 100 tokens over 30000
    // 98 us in 16 chunks, 122 in 8, 120 in 32; 300 alone 22 whole, 25 in 2; entries cut by the length, and each into as
    // many: 5 x 64 over 500 .. 20000 93, 114, 40 x 24 over 200 .. 3000 66, 91, head_dim 64 6 x 128 over 500 .. 20000
    // 110, 236).  A chunk's outputs are written and read again, so where slots run out, only what would take
    // half as long again as the chip's whole work is cut, to that length (longest entry 1.42 and 1.47 times that: 142
    // and 169 us whole, 154 and 177 cut; 1.62 340, 303; 2.3 498, 333; 16 x 300 58 whole, 138 in 2).
    const int64_t slots = (int64_t)std::max(1, cus) * quant_prefill_per_cu(D);
    const int     tile = quant_prefill_rows(D);
    auto          keys = [&](const QuantPrefillEntry &e) { return ((int64_t)e.S + quant_prefill_tile(D) - 1) / quant_prefill_tile(D); };
    auto          items = [&](int64_t c) { // of chunks of at most c tiles
        int64_t k = 0;
        for (const auto &e : plan.entries) k += ((int64_t)e.nq * G + tile - 1) / tile * ((keys(e) + c - 1) / c) * Hkv;
        return k;
    };
    int64_t longest = 1;
    for (const auto &e : plan.entries) longest = std::max(longest, keys(e));
    int64_t    lo = std::min<int64_t>(3, longest), hi = longest;
    const bool rounds = items(longest) > slots;
    if (rounds) {
        int64_t work = 0;
        for (const auto &e : plan.entries) work += ((int64_t)e.nq * G + tile - 1) / tile * keys(e) * Hkv;
        lo = std::clamp((work + slots - 1) / slots, lo, hi);
    } else {
        while (lo < hi) { // the shortest that all have a slot at once
            const int64_t c = (lo + hi) / 2;
            if (items(c) <= slots) hi = c;
            else lo = c + 1;
        }
    }
    const int64_t chunk = longest - lo >= (rounds ? std::max<int64_t>(6, lo / 2) : 6) ? lo : longest;
    for (auto &e : plan.entries) e.nch = (int)((keys(e) + chunk - 1) / chunk);
    std::stable_sort(plan.entries.begin(), plan.entries.end(), [](const QuantPrefillEntry &x, const QuantPrefillEntry &y) {
        return (int64_t)x.S * y.nch > (int64_t)y.S * x.nch;
    });
    // Where every workgroup has a slot at once, those behind the first half share the CUs of the first in turn:
    // the shortest with the longest (16 x 128 over 500 .. 9000: 267 us, longest first throughout 278, shortest
    // first 299).
    int64_t all = 0, before = 0;
    for (const auto &e : plan.entries) all += ((int64_t)e.nq * G + tile - 1) / tile * e.nch * Hkv;
    if (all <= slots) {
        size_t i = 0;
        for (; i < plan.entries.size() && before < slots / 2; ++i)
            before += ((int64_t)plan.entries[i].nq * G + tile - 1) / tile * plan.entries[i].nch * Hkv;
        std::reverse(plan.entries.begin() + (std::ptrdiff_t)i, plan.entries.end());
    }
    plan.launches.clear();
    for (size_t i = 0; i < plan.entries.size();) {
        QuantPrefillLaunch l{(int)i, 0, 0, 0};
        int64_t            items = 0;
        for (; i < plan.entries.size() && l.n < kQuantPrefillBatch; ++i, ++l.n) {
            QuantPrefillEntry &e = plan.entries[i];
            e.item0 = (int32_t)items;
            items += ((int64_t)e.nq * G + tile - 1) / tile * e.nch;
            if (e.nch > 1) l.parts = (int)std::min<int64_t>(items, kQuantMostItems);
            if (items * Hkv > kQuantMostItems) return false;
        }
        l.items = (int)items;
        plan.launches.push_back(l);
    }
    return true;
}

} // namespace detail
} // namespace tiny_llm
