// Runs a kernel source on the CPU: every lane is a coroutine, a wave's lanes meet at
// its cross-lane operations, a workgroup's waves at its barriers.  Between two
// barriers the waves run one after another, in an order that the test picks, so a wave
// can be a whole phase ahead of the others: a barrier that is missing, or not reached by
// all, shows as a wrong result or as an abort here, every time.  Only what the kernels
// under test use is there.
#pragma once

#include "hip_fp16.h"
#include "hip_runtime_api.h"

#include <ucontext.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <memory>
#include <random>
#include <vector>

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
struct int2 {
    int x, y;
};
inline int2 make_int2(int x, int y) { return {x, y}; }

inline dim3 threadIdx, blockIdx, blockDim, gridDim;

namespace wave_host {

enum class Order { Rising, Falling, Random };
inline Order           order = Order::Rising;
inline std::mt19937_64 rng(1);

enum class At { Ready, Wave, Block, Done };
struct Lane {
    ucontext_t              ctx;
    std::unique_ptr<char[]> stack;
    At                      at = At::Ready;
    int                     line = 0; // of the operation that it waits in
    uint64_t                in = 0;
};
constexpr size_t                     kStack = 64 * 1024;
inline std::vector<Lane>             lanes;
inline std::vector<uint64_t>         met; // what the lanes of each wave brought to their last operation
inline ucontext_t                    scheduler;
inline int                           current = 0;
inline const std::function<void()> *body = nullptr;

[[noreturn]] inline void fail(const char *what, int line) {
    std::fprintf(stderr, "%s (source line %d, workgroup %u %u)\n", what, line, blockIdx.x, blockIdx.y);
    std::abort();
}

inline void wait(At at, int line, uint64_t in) {
    Lane &l = lanes[(size_t)current];
    l.at = at;
    l.line = line;
    l.in = in;
    swapcontext(&l.ctx, &scheduler);
}
inline void entry() {
    (*body)();
    lanes[(size_t)current].at = At::Done;
    swapcontext(&lanes[(size_t)current].ctx, &scheduler);
}

// What lane `lane` of the wave brought to the operation in which all of them met.
inline uint64_t of_lane(int lane) { return met[(size_t)((current & ~63) + lane)]; }
inline void     meet(int line, uint64_t in) { wait(At::Wave, line, in); }

// The lanes of wave w up to their next operation, where all of them have to meet.
inline At run_wave(int w) {
    for (int i = 64 * w; i < 64 * w + 64; ++i) {
        Lane &l = lanes[(size_t)i];
        l.at = At::Ready;
        current = i;
        threadIdx = dim3((unsigned)i);
        swapcontext(&scheduler, &l.ctx);
    }
    const Lane &first = lanes[(size_t)(64 * w)];
    for (int i = 64 * w; i < 64 * w + 64; ++i) {
        const Lane &l = lanes[(size_t)i];
        if (l.at != first.at || (l.at != At::Done && l.line != first.line)) fail("a wave's lanes part", l.line);
        met[(size_t)i] = l.in;
    }
    return first.at;
}

inline void workgroup(int threads) {
    if (threads % 64) fail("whole waves only", 0);
    const int waves = threads / 64;
    if (lanes.size() < (size_t)threads) lanes.resize((size_t)threads);
    met.assign((size_t)threads, 0);
    for (int i = 0; i < threads; ++i) {
        Lane &l = lanes[(size_t)i];
        if (!l.stack) l.stack.reset(new char[kStack]);
        getcontext(&l.ctx);
        l.ctx.uc_stack.ss_sp = l.stack.get();
        l.ctx.uc_stack.ss_size = kStack;
        l.ctx.uc_link = nullptr;
        makecontext(&l.ctx, entry, 0);
    }
    for (;;) { // from barrier to barrier
        std::vector<int> open((size_t)waves);
        for (int w = 0; w < waves; ++w) open[(size_t)w] = order == Order::Falling ? waves - 1 - w : w;
        while (!open.empty()) {
            const size_t k = order == Order::Random ? (size_t)(rng() % open.size()) : 0;
            if (run_wave(open[k]) != At::Wave) open.erase(open.begin() + (long)k);
        }
        for (int w = 1; w < waves; ++w) {
            const Lane &x = lanes[0], &y = lanes[(size_t)(64 * w)];
            if (x.at != y.at || (x.at == At::Block && x.line != y.line)) fail("the waves part at a barrier", y.line);
        }
        if (lanes[0].at == At::Done) return;
    }
}

inline void launch(dim3 grid, dim3 block, const std::function<void()> &f) {
    gridDim = grid;
    blockDim = block;
    body = &f;
    for (unsigned y = 0; y < grid.y; ++y)
        for (unsigned x = 0; x < grid.x; ++x) {
            blockIdx = dim3(x, y);
            workgroup((int)block.x);
        }
}

template <class T> inline T shuffle(int line, T v, int lane) {
    static_assert(sizeof(T) <= 8, "a word of 64 bits");
    uint64_t in = 0;
    std::memcpy(&in, &v, sizeof(T));
    meet(line, in);
    in = of_lane(lane);
    std::memcpy(&v, &in, sizeof(T));
    return v;
}
inline uint64_t ballot(int line, bool b) {
    meet(line, b);
    uint64_t m = 0;
    for (int i = 0; i < 64; ++i) m |= of_lane(i) << i;
    return m;
}
// row_shr 1..15 (0x110 + n), row_bcast15 (0x142), row_bcast31 (0x143); a lane whose row is
// masked, or that has no source, keeps `old`.
inline int dpp(int line, int old, int v, int ctrl, int rows) {
    meet(line, (uint32_t)v);
    const int l = current & 63, row = l / 16;
    if (!(rows >> row & 1)) return old;
    int from = -1;
    if (ctrl > 0x110 && ctrl < 0x120) from = l % 16 >= ctrl - 0x110 ? l - (ctrl - 0x110) : -1;
    else if (ctrl == 0x142) from = row ? 16 * row - 1 : -1;
    else if (ctrl == 0x143) from = row >= 2 ? 31 : -1;
    else fail("unknown row operation", line);
    return from < 0 ? old : (int)(uint32_t)of_lane(from);
}

} // namespace wave_host

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __shared__ static
#define __align__(n) __attribute__((aligned(n)))
#define __launch_bounds__(...)
#define __syncthreads() wave_host::wait(wave_host::At::Block, __LINE__, 0)
#define __threadfence_block() ((void)0)
#define __shfl_xor(v, mask) wave_host::shuffle(__LINE__, v, (int)(threadIdx.x & 63) ^ (mask))
#define __ballot(b) wave_host::ballot(__LINE__, b)
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, bound) wave_host::dpp(__LINE__, old, v, ctrl, rows)
#define __builtin_amdgcn_sched_barrier(mask) ((void)0)
#define __popc(x) __builtin_popcount(x)
#define __popcll(x) __builtin_popcountll(x)
#define hipLaunchKernelGGL(fn, grid, block, lds, stream, ...)                                                          \
    wave_host::launch(grid, block, [&] { fn(__VA_ARGS__); })

template <class T, class U> inline auto min(T a, U b) { return a < b ? a : b; }
template <class T, class U> inline auto max(T a, U b) { return a < b ? b : a; }
inline uint32_t __float_as_uint(float f) {
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return u;
}
inline float __uint_as_float(uint32_t u) {
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}
inline uint32_t atomicAdd(uint32_t *p, uint32_t v) { // (one lane runs at a time)
    const uint32_t old = *p;
    *p = old + v;
    return old;
}
