// How the blocks of a scan walk along the steps (gated_scan.cu): how values come into their shared memory, how the pieces of a tile meet, and what becomes of
// waits that run out.  Whatever touches the machine is behind the functions of tc_ptx.cuh, so that a test walks with threads of the host.
#pragma once

#include "common.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

#include <type_traits>

namespace ct {
namespace {

using namespace ptx;

template <int W> constexpr int kMostBlocks = W == 8 ? 15 : 8; // of a cluster; their places are shared memory that other blocks cannot have

// How the pieces of a tile meet.  Without a cluster every warp goes through the pieces of all.  In a cluster a warp of its own does, the joining one: it sends what
// the block's pieces do together to the other blocks by st.async, whose arrival a barrier counts (a cluster-wide barrier would wait until the last tile's stores to
// global memory are done), and hands each warp the state before its steps.  Meanwhile the warps work out the next tile's pieces: the state comes a tile late.
// A warp has the state of tile i - 1 when it leaves the piece of tile i + 1, so there are two places for pieces and states; a block may send tile j while another
// reads what came of tile j - 2, and four places for that.
//
// A wait that runs out is reported, and what the call computes does not count any more; until it ends no thread may do what barriers leave undefined.  A lane
// of the joining warp then sends nothing more, and lane 0 arms nothing more (an arrival at a barrier whose last phase it did not see complete may be one too
// many), so that other blocks' waits for that run out as well, each after its own limit.  A warp whose copies did not come fetches no more of them, and goes through
// its tiles as if they had no steps.
template <int W, bool CLUSTER> struct Exchange {
    double2 pieces[2][W][32]; // (a, b)
    int gave_up;              // a wait has run out, which is reported at the end; see below
};
template <int W> struct Exchange<W, true> : Exchange<W, false> {
    float before[2][W][32];
    double2 blocks[4][kMostBlocks<W + 1>][32];
    uint64_t published[2], ready[2], arrived[4];
};

// After a wait has run out: what is on its way to this block's memory lands before the block ends, or is waited for once more.
template <WaitFor FOR = kCta> __device__ __forceinline__ void land(const uint64_t &barrier, int phase) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait<FOR>(smem_u32(&barrier), phase & 1) && globaltimer_ns() - t0 < kWaitBudgetNs) {
    }
}

// Walks the tiles: first(i, steps) takes tile i into `steps`, a lane's registers, and says what they do; second(i, steps, state) goes through them from
// the state before them.  Returns the state behind all tiles.
template <typename Steps, int W, typename First, typename Second>
__device__ __forceinline__ double walk(Exchange<W, false> &e, int tiles, double state, int, First &&first, Second &&second) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Steps s;
    for (int i = 0; i < tiles; ++i) {
        e.pieces[i & 1][warp][lane] = first(i, s);
        __syncthreads();
        double before = state;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            before          = w == warp ? state : before;
            const double2 p = e.pieces[i & 1][w][lane];
            state           = fma(p.x, state, p.y);
        }
        second(i, s, (float)before);
    }
    return state;
}
template <typename Steps, int W, typename First, typename Second>
__device__ __forceinline__ double walk(Exchange<W, true> &e, int tiles, double state, int blocks, First &&first, Second &&second) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == W) {
        const int rank = (int)cluster_rank();
        bool on        = true; // this lane's waits have not run out
        for (int i = 0; i < tiles; ++i) {
            on = on && mbar_wait(smem_u32(&e.published[i & 1]), i >> 1 & 1, &e.gave_up);
            double2 p[W], all = make_double2(1.0, 0.0);
#pragma unroll
            for (int w = 0; w < W; ++w)
                p[w] = e.pieces[i & 1][w][lane];
#pragma unroll
            for (int w = 0; w < W; ++w)
                all = make_double2(all.x * p[w].x, fma(p[w].x, all.y, p[w].y));
            const uint32_t at = smem_u32(&e.blocks[i & 3][rank][lane]), bar = smem_u32(&e.arrived[i & 3]);
            if (on) {
                if (lane == 0)
                    mbar_expect_tx(bar, blocks * 512);
                for (int r = 0; r < blocks; ++r)
                    st_async_d2(mapa(at, r), mapa(bar, r), all);
                on = mbar_wait<kClusterWritten>(bar, i >> 2 & 1, &e.gave_up);
                if (!on) // (a block that sends a piece of a later tile waits for this one's: that has landed long before its own limit)
                    land<kClusterWritten>(e.arrived[i & 3], i >> 2);
            }
            auto pass = [&](int r) {
                const double2 q = e.blocks[i & 3][r][lane];
                state           = fma(q.x, state, q.y);
            };
            for (int r = 0; r < rank; ++r)
                pass(r);
            double before = state;
            for (int r = rank; r < blocks; ++r)
                pass(r);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                e.before[i & 1][w][lane] = (float)before;
                before                   = fma(p[w].x, before, p[w].y);
            }
            __syncwarp();
            if (lane == 0)
                mbar_arrive(smem_u32(&e.ready[i & 1]));
        }
        return state;
    }
    auto turn = [&](int i, Steps &now, Steps &past) {
        if (i < tiles) {
            e.pieces[i & 1][warp][lane] = first(i, now);
            __syncwarp();
            if (lane == 0)
                mbar_arrive(smem_u32(&e.published[i & 1]));
        }
        if (i > 0) {
            const int j = i - 1;
            if (!*(volatile int *)&e.gave_up)
                mbar_wait(smem_u32(&e.ready[j & 1]), j >> 1 & 1, &e.gave_up);
            second(j, past, e.before[j & 1][warp][lane]);
        }
    };
    Steps even, odd;
    for (int i = 0;; i += 2) {
        turn(i, even, odd);
        if (i == tiles)
            break;
        turn(i + 1, odd, even);
        if (i + 1 == tiles)
            break;
    }
    return state;
}
template <int W, bool CLUSTER> __device__ __forceinline__ void walk_begin(Exchange<W, CLUSTER> &e) {
    if (threadIdx.x == 0) {
        e.gave_up = 0;
        if constexpr (CLUSTER) {
            for (int i = 0; i < 4; ++i)
                mbar_init(smem_u32(&e.arrived[i]), 1);
            for (int i = 0; i < 2; ++i)
                mbar_init(smem_u32(&e.published[i]), W), mbar_init(smem_u32(&e.ready[i]), 1);
            mbar_fence_init();
        }
    }
    if (CLUSTER)
        cluster_sync();
    else
        __syncthreads();
}
template <int W, bool CLUSTER> __device__ __forceinline__ void walk_end(Exchange<W, CLUSTER> &e, uint32_t *flags) {
    if (CLUSTER)
        cluster_sync(); // nothing is on its way to a block that has ended
    else
        __syncthreads();
    if (threadIdx.x == 0 && e.gave_up)
        atomicExch(&flags[FLAG_TIMEOUT], 1u + blockIdx.x);
}

struct Chain {
    int64_t first; // of its values, at step 0
    int64_t index; // of its state
    int steps;     // that belong to the sequence; none of a chain that is not there
    bool here;
};
__device__ __forceinline__ Chain chain_of(int64_t index, int64_t chains, int64_t steps, int64_t channels, const int64_t *__restrict__ lengths) {
    Chain c;
    c.here          = index < chains;
    c.index         = c.here ? index : 0;
    const int64_t b = c.index / channels;
    c.first         = b * steps * channels + (c.index - b * channels);
    c.steps         = c.here ? (int)steps : 0;
    if (c.here && lengths) {
        const int64_t length = lengths[b];
        c.steps              = length < 0 ? 0 : (int)(length < steps ? length : steps);
    }
    return c;
}

// How values come into a block's shared memory.
//   TILES: a group is 32 channels of one sequence; a piece of an array is one box of a tensor map, whose bytes a barrier counts.  (By cp.async, 16 bytes to a
//     lane, copies and their addresses took a third of the first walk; as a bulk copy to each row, 15 clocks a row.)
//   ROWS: the same where channels are no multiple of four, and rows begin anywhere.  Four rows together do begin on 16 bytes: the map's rows are these, and
//     a piece is four boxes, of the rows 0, 4, .., those behind them, and so on, each from the multiple of four values before its first one.
//   SINGLE: a group is 32 chains that follow one another, of several sequences where they have few channels, at any address; each lane copies what it reads.
enum Source { TILES, ROWS, SINGLE };
template <int ARRAYS> struct Arrays {
    CUtensorMap map[ARRAYS]; // TILES: [batch][steps][channels]; ROWS: [batch * steps / 4][4 channels]
    const float *base[ARRAYS];
};
template <Source FROM>
__device__ __forceinline__ Chain chain_of_lane(
    int64_t group, int lane, int64_t chains, int64_t steps, int channels, const int64_t *__restrict__ lengths) {
    if (FROM == SINGLE)
        return chain_of(group * 32 + lane, chains, steps, channels, lengths);
    const int64_t per = (channels + 31) / 32, b = group / per, c = (group - b * per) * 32 + lane;
    return chain_of(c < channels ? b * channels + c : chains, chains, steps, channels, lengths);
}

// A warp's ARRAYS pieces of S rows, in DEPTH places.  Tile i + DEPTH's are fetched when tile i's have been read, a quarter of a tile's time from its beginning,
// and arrive meanwhile.  Two places are for the blocks of clusters, which do not fill the machine, from whole boxes (us in line with one and with two: 16384 steps of 16, 24 and 32 groups
// 23 and 23, 31 and 29, 37 and 35, backward 42 and 39, 56 and 53, 70 and 76: there up to as many groups as a sixth of the SMs; blocks of 4 warps, 168
// groups of 1537 steps 27 and 25, 41 and 36).  Elsewhere the second place keeps other blocks out (8 x 2048 x 2048 backward 136 and 152; 1537 steps of 175 groups by rows 27 and 35).
// The last array's rows may be those of the step before (SHIFTED).
template <int ARRAYS, int S, Source FROM, bool SHIFTED, int DEPTH> struct Pieces {
    static constexpr int BOXES = FROM == ROWS ? 4 : 1, ROW = FROM == ROWS ? 36 : 32; // values of a box's row
    static constexpr int BOX = (S / BOXES * ROW + 31) & ~31, PIECE = BOXES * BOX, FLOATS = ARRAYS * PIECE; // a box begins on 128 bytes
    float *memory;
    uint64_t *arrived;
    int *gave_up;
    const Arrays<ARRAYS> *arrays;
    int64_t first; // SINGLE: of the chain's values
    int channels, c0, batch, lane;
    int row0, in_fours; // ROWS: the sequence's first row, and how many rows are in groups of four (all but the last three at most)
    int steps;          // of the sequence, padding among them
    int skew[4];        // ROWS: how far the group lies from a multiple of four values in the rows 0, 1, 2 and 3 of any piece

    __device__ __forceinline__ Pieces(float *all, uint64_t *barriers, int *flag, const Arrays<ARRAYS> &from, int width)
        : memory(all + (threadIdx.x >> 5) * FLOATS * DEPTH), arrived(barriers), gave_up(flag), arrays(&from), channels(width), lane(threadIdx.x & 31) {
        if (FROM != SINGLE && lane == 0) {
            for (int d = 0; d < DEPTH; ++d)
                mbar_init(smem_u32(arrived + d), 1);
            mbar_fence_init();
        }
        __syncwarp();
    }
    // t: where one of the warp's pieces begins; the others do a multiple of S, and so of four, steps from there
    __device__ __forceinline__ void at(const Chain &c, int64_t group, int64_t chains, int64_t all_steps, int t) {
        const int64_t per = (channels + 31) / 32, b = group / per;
        first = c.first, steps = (int)all_steps, batch = (int)b, c0 = (int)(group - b * per) * 32;
        if (FROM == ROWS) {
            row0     = batch * steps;
            in_fours = (int)(chains / channels * all_steps) & ~3;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                skew[q] = (((row0 + t + q) & 3) * channels + c0) & 3;
        }
    }
    // The warp's piece i, which begins at step t and has the chain's steps first_row .. last_row - 1 as rows; last: what wait() may have changed.
    __device__ __forceinline__ void fetch(int i, int t, int first_row, int last_row, int last) {
        if (FROM != SINGLE && last < 0)
            return;
        float *place = memory + i % DEPTH * FLOATS;
        if (FROM == SINGLE) {
            auto copy_rows = [&](auto all) {
#pragma unroll
                for (int k = 0; k < ARRAYS; ++k) {
                    const int shift   = SHIFTED && k == ARRAYS - 1;
                    const float *from = arrays->base[k] + first + (int64_t)(t - shift) * channels;
#pragma unroll
                    for (int j = 0; j < S; ++j)
                        if (decltype(all)::value || (j >= first_row && j < last_row && (!shift || t + j > 0)))
                            cp_async_4(smem_u32(place + k * PIECE + j * 32 + lane), from + (int64_t)j * channels);
                }
            };
            if (__all_sync(0xffffffffu, first_row < 0 && last_row >= S))
                copy_rows(std::true_type{});
            else
                copy_rows(std::false_type{});
            cp_async_commit();
            return;
        }
        // what a box has outside the array is zeros; rows of other sequences are not used
        const uint32_t bar = smem_u32(arrived + i % DEPTH), to = smem_u32(place);
        if (FROM == TILES) {
            if (lane == 0) { // (by a lane to each array they would be issued one lane after the other)
                mbar_expect_tx(bar, last_row > 0 ? ARRAYS * S * ROW * 4 : 0);
                if (last_row > 0)
#pragma unroll
                    for (int k = 0; k < ARRAYS; ++k)
                        tma_load_3d(to + k * PIECE * 4, &arrays->map[k], bar, c0, t - (SHIFTED && k == ARRAYS - 1), batch);
            }
        } else if (lane < ARRAYS * BOXES) { // 16 of them are issued sooner so than by one lane (7 x 1537 x 771 backward 55 us and 59)
            const int k = lane / BOXES, row = row0 + t - (SHIFTED && k == ARRAYS - 1) + lane % BOXES;
            if (lane == 0)
                mbar_expect_tx(bar, last_row > 0 ? ARRAYS * S * ROW * 4 : 0);
            if (last_row > 0)
                tma_load_2d(to + lane * BOX * 4, &arrays->map[k], bar, ((row & 3) * channels + c0) & ~3, row >> 2);
        }
    }
    // When the wait has run out the copies that are on their way land, and `last` becomes a step before all: the warp waits for nothing more, and fetches nothing
    // more, since that would be an arrival at a barrier whose phase may not be complete.
    __device__ __forceinline__ void wait(int i, int &last) {
        if (FROM == SINGLE)
            cp_async_wait<DEPTH - 1>();
        else if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(arrived + i % DEPTH), i / DEPTH & 1, gave_up))) {
            for (int d = 0; d < DEPTH; ++d)
                land(arrived[(i + d) % DEPTH], (i + d) / DEPTH);
            last = -(1 << 30);
        }
        __syncwarp();
    }
    // The lane's values in array k of the piece that begins at step t.
    __device__ __forceinline__ void read(int i, int k, int t, float (&to)[S]) const {
        const float *from = memory + i % DEPTH * FLOATS + k * PIECE + lane;
        if (FROM == ROWS) {
            constexpr int SHIFT = SHIFTED ? 1 : 0;
            const bool shift    = SHIFT && k == ARRAYS - 1;
#pragma unroll
            for (int j = 0; j < S; ++j)
                to[j] = from[(j & 3) * BOX + j / 4 * ROW + skew[shift ? (j + 3) & 3 : j & 3]];
            const int row = row0 + t - shift;
            if (row + S > in_fours) { // the array's last rows
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (row + j >= in_fours && t + j < steps && c0 + lane < channels)
                        to[j] = arrays->base[k][(int64_t)(row + j) * channels + c0 + lane];
            }
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j)
                to[j] = from[j * ROW];
        }
    }
};

} // namespace
} // namespace ct
