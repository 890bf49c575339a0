// The eviction kernels (tiny-llm_amd/csrc/kernels/evict.hip) on the CPU, lane by lane
// (wave_host/), in several orders of the waves between barriers, against a plain
// selection, every place of the cache, the accounts and the positions compared.
#include "../../tiny-llm_amd/csrc/kernels/evict.hip"

#include <cmath>
#include <limits>

namespace tiny_llm {
namespace detail {
void profile_begin(KernelId, hipStream_t) {}
void profile_end(KernelId, hipStream_t) {}
} // namespace detail
} // namespace tiny_llm

using namespace tiny_llm::detail;

#define CHECK(c)                                                                                                       \
    do {                                                                                                               \
        if (!(c)) {                                                                                                    \
            std::fprintf(stderr, "check failed: %s (%s:%d)\n", #c, __FILE__, __LINE__);                              \
            std::abort();                                                                                              \
        }                                                                                                              \
    } while (0)

namespace {

constexpr int D = 32, kSpace = 64; // untouched words around every array

enum class Kind { Tail, Ties, Equal, Wild };

// An array with known words on both sides.
template <class T> struct Guarded {
    std::vector<T> v;
    Guarded(size_t n, T guard) : v(n + 2 * kSpace, guard), guard_(guard) {}
    T   *data() { return v.data() + kSpace; }
    void check() const {
        for (int i = 0; i < kSpace; ++i) CHECK(std::memcmp(&v[(size_t)i], &guard_, sizeof(T)) == 0 && std::memcmp(&v[v.size() - 1 - (size_t)i], &guard_, sizeof(T)) == 0);
    }

  private:
    T guard_;
};

struct Case {
    std::vector<int> lens, keeps;
    int              recent, hkv, block, room;
    Kind             kind;
    bool             in_place;
    std::vector<int> base, gone;
};

void run(const Case &c, std::mt19937_64 &rng) {
    const int    n = (int)c.lens.size();
    const size_t words = (size_t)n * c.hkv * c.room;
    Guarded<float>   w(words, 5.0f), w_out(words, 6.0f);
    Guarded<int32_t> pos(words, -5), pos_out(words, -6);
    auto u01 = [&] { return (double)(rng() >> 11) / 9007199254740992.0; };
    for (size_t i = 0; i < words; ++i) {
        const double u = u01();
        float        x = 0.5f;
        if (c.kind == Kind::Tail) x = u < 0.03 ? 0.0f : (float)(8 * std::pow(u, 6));
        if (c.kind == Kind::Ties) x = (float)std::floor(5 * u);
        if (c.kind == Kind::Wild) {
            const float inf = std::numeric_limits<float>::infinity();
            const float odd[] = {inf, -inf, std::numeric_limits<float>::quiet_NaN(), 0.0f, -0.0f};
            x = u < 0.3 ? odd[(size_t)(u / 0.06)] : (float)(u < 0.6 ? u - 0.45 : -u);
        }
        w.data()[i] = x;
    }
    // positions below a sequence's base: some order of what it kept then
    std::vector<EvictEntry> entries;
    for (int i = 0; i < n; ++i) {
        const int base = c.base[(size_t)i], gone = c.gone[(size_t)i];
        entries.push_back({i, c.lens[(size_t)i], c.keeps[(size_t)i], base, gone, 0});
        for (int h = 0; h < c.hkv; ++h) {
            std::vector<int32_t> all((size_t)(base + gone));
            for (int t = 0; t < base + gone; ++t) all[(size_t)t] = t;
            std::shuffle(all.begin(), all.end(), rng);
            std::copy(all.begin(), all.begin() + base, pos.data() + ((size_t)i * c.hkv + h) * c.room);
        }
    }
    // the cache: K and V rows that say where they were
    const int           blocks = c.block ? c.room / c.block : 1, per = c.block ? c.block : c.room;
    std::vector<int32_t> table((size_t)n * blocks);
    for (size_t i = 0; i < table.size(); ++i) table[i] = (int32_t)i;
    std::shuffle(table.begin(), table.end(), rng);
    const size_t     half_words = (size_t)n * c.room * c.hkv * D;
    Guarded<__half> k(half_words, __half{0x7777}), v(half_words, __half{0x7777});
    KvView           view;
    view.k_base = k.data();
    view.v_base = v.data();
    view.tok_stride = c.hkv * D;
    view.head_stride = D;
    view.blk_stride = (int64_t)per * c.hkv * D;
    if (c.block) {
        view.block_table = table.data();
        view.bt_stride = blocks;
        view.log2_blk = __builtin_ctz((unsigned)c.block);
    }
    auto at = [&](int i, int t, int h) {
        const int blk = c.block ? table[(size_t)(i * blocks + t / per)] : i;
        return ((size_t)blk * per + (size_t)(t % per)) * c.hkv * D + (size_t)h * D;
    };
    auto sign = [](int i, int t, int h, int d, int which) { return (uint16_t)((i * 31 + t * 7 + h * 5 + which) * 32 + d); };
    for (int i = 0; i < n; ++i)
        for (int t = 0; t < c.room; ++t)
            for (int h = 0; h < c.hkv; ++h)
                for (int d = 0; d < D; ++d) {
                    k.data()[at(i, t, h) + d] = {sign(i, t, h, d, 0)};
                    v.data()[at(i, t, h) + d] = {sign(i, t, h, d, 1)};
                }
    const std::vector<float>   w0 = w.v, wo0 = c.in_place ? w.v : w_out.v;
    const std::vector<int32_t> p0 = pos.v, po0 = c.in_place ? pos.v : pos_out.v;

    EvictState st;
    st.w_in = w.data();
    st.w_out = c.in_place ? w.data() : w_out.data();
    st.pos_in = pos.data();
    st.pos_out = c.in_place ? pos.data() : pos_out.data();
    st.room = c.room;
    Guarded<int32_t> work(evict_workspace_words(entries, c.hkv), -7);
    launch_evict(view, entries, st, c.recent, c.hkv, D, work.data(), nullptr);
    for (const auto *g : {&w, &w_out}) g->check();
    for (const auto *g : {&pos, &pos_out, &work}) g->check();
    for (const auto *g : {&k, &v}) g->check();

    for (int i = 0; i < n; ++i)
        for (int h = 0; h < c.hkv; ++h) {
            const int    len = c.lens[(size_t)i], keep = c.keeps[(size_t)i], base = c.base[(size_t)i], gone = c.gone[(size_t)i];
            const size_t o = ((size_t)i * c.hkv + h) * c.room;
            auto position = [&](int t) { return t < base ? p0[kSpace + o + (size_t)t] : t + gone; };
            auto weight = [&](int t) { return w0[kSpace + o + (size_t)t]; };
            std::vector<int> rank((size_t)len);
            for (int t = 0; t < len; ++t) rank[(size_t)t] = t;
            std::stable_sort(rank.begin(), rank.end(), [&](int x, int y) {
                const bool nx = position(x) >= len + gone - c.recent, ny = position(y) >= len + gone - c.recent;
                if (nx || ny) return nx && !ny;
                const float a = weight(x), b = weight(y);
                return a != a ? false : b != b ? true : a > b;
            });
            std::vector<char> stays((size_t)len, 0);
            for (int r = 0; r < keep; ++r) stays[(size_t)rank[(size_t)r]] = 1;
            int mover = keep;
            for (int t = 0; t < c.room; ++t) {
                int from = t;
                if (t < keep && !stays[(size_t)t]) {
                    while (!stays[(size_t)mover]) ++mover;
                    from = mover++;
                }
                for (int d = 0; d < D; ++d) {
                    CHECK(k.data()[at(i, t, h) + d].bits == sign(i, from, h, d, 0));
                    CHECK(v.data()[at(i, t, h) + d].bits == sign(i, from, h, d, 1));
                }
                const float   got = st.w_out[o + (size_t)t], want = t < keep ? weight(from) : wo0[kSpace + o + (size_t)t];
                const int32_t at_p = st.pos_out[o + (size_t)t];
                CHECK(got == want || (got != got && want != want));
                if (c.in_place && keep == len) CHECK(at_p == po0[kSpace + o + (size_t)t]); // nothing is taken
                else CHECK(at_p == (t < keep ? position(from) : po0[kSpace + o + (size_t)t]));
            }
        }
}

// Two sequences, the longer one of `len` tokens, through the kernel for that length.
void both(int len, int keep, int recent, Kind kind, int block, bool in_place, std::mt19937_64 &rng) {
    Case c;
    c.lens = {len, len > 3 ? len / 3 : len};
    c.keeps = {std::min(keep, len), std::max(std::min(c.lens[1], recent), std::min(c.lens[1], 1 + keep / 4))};
    c.recent = std::min({recent, c.keeps[0], c.keeps[1]});
    c.hkv = len > 4096 ? 1 : 2;
    c.block = block;
    c.room = (len + 5 + 15) / 16 * 16;
    c.kind = kind;
    c.in_place = in_place;
    const bool again = rng() % 2;
    for (const int l : c.lens) {
        c.base.push_back(again ? l / 2 : 0);
        c.gone.push_back(again ? 1 + l / 5 : 0);
    }
    run(c, rng);
}

} // namespace

int main() {
    std::mt19937_64 rng(7);
    const Kind      kinds[] = {Kind::Tail, Kind::Ties, Kind::Equal, Kind::Wild};
    const std::pair<wave_host::Order, const char *> orders[] = {
        {wave_host::Order::Rising, "rising"}, {wave_host::Order::Falling, "falling"}, {wave_host::Order::Random, "random"}};
    for (const auto &o : orders) {
        wave_host::order = o.first;
        for (const int len : {1, 2, 3, 5, 64, 65, 255, 257, 1000, 1024, 1025, 2047, 2049})
            for (int x = 0; x < 4; ++x) {
                const int keep = 1 + (int)(rng() % (uint64_t)len), recent = (int)(rng() % (uint64_t)(keep + 1));
                both(len, keep, recent, kinds[x], x % 2 ? 16 : 0, (x / 2 + len) % 2, rng);
            }
        both(1024, 300, 0, Kind::Tail, 0, true, rng);
        both(900, 899, 17, Kind::Ties, 16, false, rng);
        std::printf("ok short %s\n", o.second);
        // the other instantiations, and the kernel beyond them
        int x = 0;
        for (const int len : {2100, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769})
            both(len, len / 5, len / 50, kinds[(x + (int)o.first) % 4], x % 2 ? 0 : 16, (x / 2) % 2, rng), ++x;
        std::printf("ok long %s\n", o.second);
        std::fflush(stdout);
    }
    return 0;
}
