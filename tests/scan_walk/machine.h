// What camel_b200/csrc/scan_walk.cuh needs of the machine, for threads of the host: a thread is a warp (its lane 0), shared memory of a block is a piece of the
// host's, and barriers count as the PTX manual says.  What that leaves undefined is noted in `violations`: an arrival without one pending, a count of bytes out of
// its range, bytes that arrive in a block that has ended.
#pragma once

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <condition_variable>
#include <cstdint>
#include <map>
#include <mutex>
#include <set>
#include <string>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __restrict__
using std::fma;
using std::max;
using std::min;

struct double2 {
    double x, y;
};
inline double2 make_double2(double x, double y) { return {x, y}; }
struct Index {
    unsigned x;
};
inline thread_local Index threadIdx, blockIdx;

// A copy of `bytes`, which arrives after `after_ms`, or never (below 0).
struct CUtensorMap {
    int bytes  = 0;
    int after_ms = 0;
};

namespace host {

struct Barrier {
    int count = 0, pending = 0;
    int64_t bytes  = 0;
    uint32_t phase = 0;
};
inline std::mutex lock;
inline std::condition_variable changed;
inline std::map<uint32_t, Barrier> barriers;
inline std::set<std::string> violations;
inline std::vector<char *> memory; // of each block
inline std::vector<bool> ended;
inline std::vector<std::thread> copies;
inline thread_local int block; // of this thread
constexpr int kBlockBits = 24;

inline void note(const char *what) { violations.insert(what); }
inline void complete(Barrier &b) {
    if (b.pending == 0 && b.bytes == 0)
        ++b.phase, b.pending = b.count, changed.notify_all();
}
inline void add_bytes(Barrier &b, int64_t bytes) {
    b.bytes += bytes;
    if (b.bytes > (1 << 20) - 1 || b.bytes < -((1 << 20) - 1))
        note("bytes of a barrier out of range");
}
inline void arrive(uint32_t bar, int64_t bytes) {
    std::lock_guard<std::mutex> l(lock);
    Barrier &b = barriers[bar];
    add_bytes(b, bytes);
    if (b.pending == 0)
        note("an arrival at a barrier that has none pending");
    else
        --b.pending;
    complete(b);
}
inline void landed(uint32_t bar, int64_t bytes) {
    std::lock_guard<std::mutex> l(lock);
    if (ended[bar >> kBlockBits])
        note("bytes arrive in a block that has ended");
    add_bytes(barriers[bar], -bytes);
    complete(barriers[bar]);
}
inline bool wait(uint32_t bar, uint32_t parity, std::chrono::milliseconds limit) {
    std::unique_lock<std::mutex> l(lock);
    return changed.wait_for(l, limit, [&] { return (barriers[bar].phase & 1) != parity; });
}
// A barrier of all threads of the cluster.
inline int threads, waiting, turn;
inline void sync() {
    std::unique_lock<std::mutex> l(lock);
    const int mine = turn;
    if (++waiting == threads)
        waiting = 0, ++turn, changed.notify_all();
    else
        changed.wait(l, [&] { return turn != mine; });
}

} // namespace host

template <typename T> bool __all_sync(unsigned, T v) { return v; }
inline void __syncwarp() {}
inline void __syncthreads() { host::sync(); }
inline uint32_t atomicExch(uint32_t *to, uint32_t v) {
    std::lock_guard<std::mutex> l(host::lock);
    std::swap(*to, v);
    return v;
}

namespace ct {
enum FlagWord : int { FLAG_TIMEOUT = 2 };
namespace ptx {

inline uint64_t kWaitBudgetNs; // set by the program
enum WaitFor { kCta, kClusterWritten, kClusterRead };
inline uint64_t globaltimer_ns() {
    return (uint64_t)std::chrono::duration_cast<std::chrono::nanoseconds>(std::chrono::steady_clock::now().time_since_epoch()).count();
}
inline uint32_t smem_u32(const void *p) { return (uint32_t)host::block << host::kBlockBits | (uint32_t)(static_cast<const char *>(p) - host::memory[host::block]); }
inline uint32_t mapa(uint32_t addr, uint32_t rank) { return rank << host::kBlockBits | (addr & ((1u << host::kBlockBits) - 1)); }
inline uint32_t cluster_rank() { return (uint32_t)host::block; }
inline void cluster_sync() { host::sync(); }
inline void mbar_init(uint32_t bar, uint32_t count) {
    std::lock_guard<std::mutex> l(host::lock);
    host::barriers[bar]         = {};
    host::barriers[bar].count   = (int)count;
    host::barriers[bar].pending = (int)count;
}
inline void mbar_fence_init() {}
inline void mbar_arrive(uint32_t bar) { host::arrive(bar, 0); }
inline void mbar_expect_tx(uint32_t bar, uint32_t bytes) { host::arrive(bar, bytes); }
template <WaitFor FOR = kCta> bool mbar_try_wait(uint32_t bar, uint32_t parity) { return host::wait(bar, parity, std::chrono::milliseconds(1)); }
// as in tc_ptx.cuh: until the budget has run out, or another's
template <WaitFor FOR = kCta> bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*abort_flag)
            return false;
        if (globaltimer_ns() - t0 > kWaitBudgetNs) {
            *abort_flag = 1;
            return false;
        }
    }
    return true;
}
// a warp's 32 lanes together
inline void st_async_d2(uint32_t addr, uint32_t bar, double2 v) {
    *reinterpret_cast<double2 *>(host::memory[addr >> host::kBlockBits] + (addr & ((1u << host::kBlockBits) - 1))) = v;
    host::landed(bar, 512);
}
inline void copy(const void *map, uint32_t bar) {
    const CUtensorMap m = *static_cast<const CUtensorMap *>(map);
    if (m.after_ms < 0)
        return;
    if (m.after_ms == 0)
        return host::landed(bar, m.bytes);
    std::lock_guard<std::mutex> l(host::lock);
    host::copies.emplace_back([=] {
        std::this_thread::sleep_for(std::chrono::milliseconds(m.after_ms));
        host::landed(bar, m.bytes);
    });
}
inline void tma_load_2d(uint32_t, const void *map, uint32_t bar, int, int) { copy(map, bar); }
inline void tma_load_3d(uint32_t, const void *map, uint32_t bar, int, int, int) { copy(map, bar); }
inline void cp_async_4(uint32_t, const float *) {}
inline void cp_async_commit() {}
template <int PENDING> void cp_async_wait() {}

} // namespace ptx
} // namespace ct
