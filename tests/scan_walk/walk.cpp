// Walks tiles with threads of the host.  walk <tiles> <what goes wrong> [tile]: nothing; a warp that is late by many limits; a copy that never comes;
// one that comes after its limit has run out.  Prints what the machine leaves undefined and was done, the blocks that reported, and the state.
#include "scan_walk.cuh"

#include <cstdio>
#include <cstdlib>
#include <cstring>

using namespace ct;
using namespace ct::ptx;

constexpr int kBlocks = 3, kWalk = 3, S = 16, kDepth = 2;
constexpr int kBytes = 2 * S * 32 * 4; // of both arrays' boxes
using Values = Pieces<2, S, TILES, false, kDepth>;
struct Memory {
    Exchange<kWalk, true> ex;
    uint64_t arrived[kWalk][kDepth];
    float pieces[kWalk * Values::FLOATS * kDepth];
};

int main(int argc, char **argv) {
    const int tiles        = argc > 1 ? atoi(argv[1]) : 40;
    const std::string what = argc > 2 ? argv[2] : "nothing";
    const int when         = argc > 3 ? atoi(argv[3]) : 6;
    kWaitBudgetNs          = (what == "nothing" ? 20000 : 400) * 1000000ull;
    std::vector<Memory> memory(kBlocks);
    uint32_t flags[kBlocks][4] = {};
    double states[kBlocks]     = {};
    for (auto &m : memory)
        host::memory.push_back(reinterpret_cast<char *>(&m));
    host::ended.assign(kBlocks, false);
    host::threads = kBlocks * (kWalk + 1);
    auto value    = [](int piece) { return 0.25 * ((piece * 37 % 11) - 5); }; // h = h / 2 + value of a piece

    auto warp_of = [&](int block, int warp) {
        host::block = block;
        threadIdx.x = (unsigned)warp * 32, blockIdx.x = (unsigned)block;
        Memory &m = memory[block];
        Arrays<2> arrays{};
        arrays.map[0].bytes = arrays.map[1].bytes = kBytes / 2;
        Values values(m.pieces, m.arrived[std::min(warp, kWalk - 1)], &m.ex.gave_up, arrays, 32);
        walk_begin(m.ex);
        const int tile = kBlocks * kWalk * S, t0 = (block * kWalk + warp) * S;
        int last = tiles * tile;
        values.at(Chain{0, 0, last, true}, 0, 32, last, t0);
        const bool mine = block == 1 && warp == 1;
        auto fetch      = [&](int i) {
            arrays.map[1].after_ms = mine && i == when ? (what == "lost" ? -1 : what == "late" ? 640 : 0) : 0;
            values.fetch(i, t0 + i * tile, -1, last - (t0 + i * tile), last);
        };
        if (warp < kWalk)
            for (int i = 0; i < kDepth; ++i)
                fetch(i);
        struct Steps {
            int tile;
        };
        bool right         = true;
        const double state = walk<Steps>(
            m.ex, tiles, 1.0, kBlocks,
            [&](int i, Steps &s) {
                s.tile = i;
                if (t0 + i * tile >= last) {
                    fetch(i + kDepth);
                    return make_double2(1.0, 0.0);
                }
                values.wait(i, last);
                fetch(i + kDepth);
                if (what == "slow" && mine && i == when)
                    std::this_thread::sleep_for(std::chrono::milliseconds(2500));
                return make_double2(0.5, value(i * kBlocks * kWalk + block * kWalk + warp));
            },
            [&](int i, const Steps &s, float) { right &= s.tile == i; });
        walk_end(m.ex, flags[block]);
        if (warp == kWalk)
            states[block] = state;
        if (!right) {
            std::lock_guard<std::mutex> l(host::lock);
            host::note("a tile's steps are another's");
        }
    };
    std::vector<std::thread> threads;
    for (int b = 0; b < kBlocks; ++b)
        for (int w = 0; w <= kWalk; ++w)
            threads.emplace_back(warp_of, b, w);
    for (auto &t : threads)
        t.join();
    {
        std::lock_guard<std::mutex> l(host::lock);
        host::ended.assign(kBlocks, true);
    }
    for (auto &t : host::copies)
        t.join();
    double state = 1.0;
    for (int p = 0; p < tiles * kBlocks * kWalk; ++p)
        state = state * 0.5 + value(p);
    for (const auto &v : host::violations)
        printf("violation: %s\n", v.c_str());
    for (int b = 0; b < kBlocks; ++b)
        printf("block %d %s\n", b, flags[b][FLAG_TIMEOUT] ? "reported" : std::abs(states[b] - state) < 1e-12 ? "right" : "wrong");
    return 0;
}
