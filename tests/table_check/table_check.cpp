// The checkpoint tables of the generator streams on the CPU (hip/hip_runtime.h beside this file): what their uploads read,
// when the background thread walks ahead, and that calls of several threads get the states of the streams.
//   table_check <what> ; exit status 0: right
#include <stdio.h>
#include <unistd.h>
#include <chrono>
#include <cstdarg>
#include <string>
#include <thread>

#include "prg.hip"

int mpcx_fail(mpcx_ctx *, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfprintf(stderr, fmt, ap);
    va_end(ap);
    return 1;
}
int mpcx_ws(mpcx_ctx *, u64, void **) { return 1; }
void mpcx_parallel_memcpy(void *dst, const void *src, u64 bytes) { memcpy(dst, src, bytes); }

static int failed = 0;
#define CHECK(...)                                                  \
    do {                                                            \
        if (!(__VA_ARGS__)) {                                       \
            fprintf(stderr, "line %d: %s\n", __LINE__, #__VA_ARGS__); \
            failed = 1;                                             \
        }                                                           \
    } while (0)

static u64 checkpoints(u64 seed) { // of the host copy
    Table &T = table_of(0, seed, 0);
    CallerLock g(T);
    return T.host.size();
}
static void idle() { // the background thread has nothing left to do (at most ten seconds)
    for (int i = 0; i < 1000; i++) {
        std::this_thread::sleep_for(std::chrono::milliseconds(10));
        std::lock_guard<std::mutex> lk(reg().qmu);
        if (reg().queue.empty() && !reg().walker_busy) return;
    }
    CHECK(!"the background thread did not finish");
}
// the device copy holds the stream's states, at every checkpoint of [0, need)
static bool right(const PrgCk *dev, u64 seed, u64 need) {
    PrgCk c{seed, 0, 0};
    for (int i = 0; i < 5; i++) prv_step(c.seed, c.lcg, c.hash);
    for (u64 e = 0; e < need; e++) {
        if (memcmp(&dev[e], &c, sizeof c)) return false;
        for (u64 i = 0; i < PRG_CK; i++) prv_step(c.seed, c.lcg, c.hash);
    }
    return true;
}

// one word a call, as the norm draws it, further and further on: nothing is walked beyond the first request's spare block
static void short_advances() {
    mpcx_ctx ctx;
    const PrgCk *dev;
    CHECK(mpcx_prg_table(&ctx, 11, 0, PRG_POP_T0 + 1, &dev) == 0);
    idle();
    const u64 first = checkpoints(11);
    for (u64 pop = 1; pop < 200000; pop += 999) CHECK(mpcx_prg_table(&ctx, 11, 0, PRG_POP_T0 + pop + 1, &dev) == 0);
    idle();
    CHECK(checkpoints(11) == first);
    CHECK(right(dev, 11, first));
}
// a stream on the move is walked ahead: by one large step, and by small ones that add up
static void long_advances() {
    mpcx_ctx ctx;
    const PrgCk *dev;
    for (u64 step : {u64(1) << 20, u64(50000)}) {
        const u64 seed = 100 + step;
        u64 t = PRG_POP_T0;
        for (u64 k = 0; k < 12; k++, t += step) CHECK(mpcx_prg_table(&ctx, seed, 0, t + 1, &dev) == 0);
        idle();
        CHECK(checkpoints(seed) >= (t + (8u << 20)) / PRG_CK);
        const u64 walked = checkpoints(seed);
        CHECK(mpcx_prg_table(&ctx, seed, 0, t + 1, &dev) == 0);
        CHECK(right(dev, seed, walked < 40000 ? walked : 40000));
    }
}
// uploads, of calls and of the background thread, read pinned memory that stays: never the table's pages, which move
static void upload_sources() {
    long_advances();
    CHECK(stub().copies > 0 && stub().copied > 0);
    CHECK(stub().from_pageable == 0);
}
// several threads advance two streams at once
static void threads() {
    std::vector<std::thread> th;
    std::atomic<int> bad{0};
    for (int k = 0; k < 4; k++)
        th.emplace_back([&, k] {
            mpcx_ctx ctx;
            const u64 seed = 7 + k % 2;
            for (u64 i = 0; i < 20; i++) {
                const PrgCk *dev;
                const u64 need = (i * 30000 * (k + 1)) / PRG_CK + 1;
                if (mpcx_prg_table(&ctx, seed, 0, i * 30000 * (k + 1), &dev)) bad++;
                if (i % 5 == 4 && !right(dev, seed, need)) bad++;
            }
        });
    for (auto &t : th) t.join();
    idle();
    CHECK(bad == 0);
}

int main(int argc, char **argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "short") short_advances();
    else if (what == "long") long_advances();
    else if (what == "sources") upload_sources();
    else if (what == "threads") threads();
    else return 2;
    fflush(stderr);
    return failed;
}
