// A gated linear recurrence along sequences, and its gradient.
//
//   a = sigmoid(gate), h[t] = a[t] h[t-1] + (1 - a[t]) value[t]
//   g[t] = dout[t] + a[t+1] g[t+1],  dvalue = (1 - a) g,  dgate[t] = a (1 - a) g (h[t-1] - value[t])
//
// Each channel of each sequence is a chain of its own, and both are bound by memory (12 and 24 bytes a step of one).  There are seldom
// enough chains to keep it busy, so the steps of a chain are shared: a lane has S of them in its registers, the warps of a block the pieces
// behind, and the blocks of a cluster those behind the block's.  What S steps do to a state is one multiplication and one addition: each lane works
// that out for its steps, takes what the pieces before its own do to the state of the tile's beginning, and then goes through its steps.  The next tile's values are
// on their way meanwhile.  The gradient is the same along the reversed axis, of c[t] = a[t] g[t] = a[t] (dout[t] + c[t+1]).
//
// Of a gate both a and 1 - a are taken with all their digits (sigmoids): a product of `a`s, each off by 2^-25 of 1, would be off by what 1 - a loses
// of its digits, and a state that remembers 1 / (1 - a) steps would add that up.  A lane's steps therefore do to a state h what is a product A and
// what they add, b, and their 1 - A is summed up by itself, S' = a S + (1 - a).  A is 1 - S in 64 bits, or, from where S has more than 1/2, the
// product, which is then small and has its digits.  Between pieces states are in 64 bits.
#include "common.cuh"
#include "gate.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace ct {
namespace {

using namespace ptx;

// What steps do to the state before them: a h + b.
struct Piece {
    float a = 1.0f, lost = 0.0f, b = 0.0f; // lost: 1 - a
    __device__ __forceinline__ void step(float ga, float rest, float add) {
        b    = __fmaf_rn(ga, b, add);
        lost = __fmaf_rn(ga, lost, rest);
        a    = __fmul_rn(ga, a);
    }
    __device__ __forceinline__ double2 joined() const { return make_double2(lost <= 0.5f ? 1.0 - (double)lost : (double)a, (double)b); }
};

constexpr int kMostBlocks = 8; // of a cluster

// The state before each warp's steps, from what all pieces of the tile do; `state` goes on to the tile's end.  Pieces lie in the order of warps, and
// of the cluster's blocks.  One tile after the other alternates between two places, so that a fast warp does not write over what a slow one reads.
// Blocks send what their pieces do to one another by st.async, whose arrival a barrier counts: a cluster-wide barrier would wait until the last
// tile's stores to global memory are done.
template <int W> struct Exchange {
    double2 pieces[2][W][32];
    double2 blocks[2][kMostBlocks][32];
    uint64_t arrived[2];
    int gave_up;
};
__device__ __forceinline__ void send(uint32_t at, uint32_t barrier, double2 p) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];" ::"r"(at), "d"(p.x), "d"(p.y), "r"(barrier)
                 : "memory");
}
template <int W>
__device__ __forceinline__ double exchange(Exchange<W> &e, int tile, Piece mine, double &state, int warp, int lane, int blocks, uint32_t rank) {
    const int turn             = tile & 1;
    e.pieces[turn][warp][lane] = mine.joined();
    __syncthreads();
    double before = state;
    if (blocks == 1) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            before          = w == warp ? state : before;
            const double2 p = e.pieces[turn][w][lane];
            state           = fma(p.x, state, p.y);
        }
        return before;
    }
    // what the warps before this one do, and the last warp's with it: the block's
    double a = 1.0, b = 0.0;
    const int upto = warp == W - 1 ? W : warp;
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < upto) {
            const double2 p = e.pieces[turn][w][lane];
            if (w == W - 1) {
                const uint32_t at  = static_cast<uint32_t>(__cvta_generic_to_shared(&e.blocks[turn][rank][lane]));
                const uint32_t bar = static_cast<uint32_t>(__cvta_generic_to_shared(&e.arrived[turn]));
                const double2 all  = make_double2(a * p.x, fma(p.x, b, p.y));
                if (lane == 0)
                    mbar_expect_tx(bar, blocks * 512);
                for (int r = 0; r < blocks; ++r)
                    send(mapa(at, r), mapa(bar, r), all);
            } else {
                b = fma(p.x, b, p.y);
                a *= p.x;
            }
        }
    // a wait that has run out is reported by the kernel's end; until then the block goes on, for the others' sake
    if (!*(volatile int *)&e.gave_up)
        mbar_wait<kClusterWritten>(static_cast<uint32_t>(__cvta_generic_to_shared(&e.arrived[turn])), (tile >> 1) & 1, &e.gave_up);
    for (int r = 0; r < blocks; ++r) {
        const double2 p = e.blocks[turn][r][lane];
        before          = r == (int)rank ? state : before;
        state           = fma(p.x, state, p.y);
    }
    return fma(a, before, b);
}
template <int W> __device__ __forceinline__ void exchange_begin(Exchange<W> &e, int blocks) {
    if (blocks == 1)
        return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i)
            mbar_init(static_cast<uint32_t>(__cvta_generic_to_shared(&e.arrived[i])), 1);
        e.gave_up = 0;
        mbar_fence_init();
    }
    cluster_sync();
}
template <int W> __device__ __forceinline__ void exchange_end(Exchange<W> &e, int blocks, uint32_t *flags) {
    if (blocks == 1)
        return;
    cluster_sync(); // nothing is on its way to a block that has ended
    if (threadIdx.x == 0 && e.gave_up)
        atomicMax(&flags[FLAG_TIMEOUT], 1u + blockIdx.x);
}

struct Chain {
    int64_t first; // of its values, at step 0
    int64_t index; // of its state
    int64_t steps; // that belong to the sequence
    bool here;
};
__device__ __forceinline__ Chain chain_of(int64_t index, int64_t chains, int64_t steps, int64_t channels, const int64_t *__restrict__ lengths) {
    Chain c;
    c.here          = index < chains;
    c.index         = c.here ? index : 0;
    const int64_t b = c.index / channels;
    c.first         = b * steps * channels + (c.index - b * channels);
    c.steps         = c.here ? steps : 0;
    if (c.here && lengths) {
        const int64_t length = lengths[b];
        c.steps              = length < 0 ? 0 : (length < steps ? length : steps);
    }
    return c;
}

// W warps to a block, S steps to a lane; the blocks of a cluster have the same 32 chains.
template <int W, int S, int FIT>
__global__ void __launch_bounds__(W * 32, FIT) gated_scan_kernel(
    const float *__restrict__ gate, const float *__restrict__ value, const float *state0, const int64_t *__restrict__ lengths, int64_t chains,
    int64_t steps, int channels, int blocks, float *__restrict__ out, float *state_out, uint32_t *__restrict__ flags) {
    __shared__ Exchange<W> ex;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = blocks > 1 ? cluster_rank() : 0;
    exchange_begin(ex, blocks);
    griddep_wait();
    const Chain c      = chain_of((int64_t)(blockIdx.x / blocks) * 32 + lane, chains, steps, channels, lengths);
    double state       = c.here && state0 ? (double)state0[c.index] : 0.0;
    const int64_t tile = (int64_t)blocks * W * S;
    int64_t t0         = ((int64_t)rank * W + warp) * S;
    float g[S], v[S];
    // Steps that a chain does not have keep its state: a = 1, and nothing is added.
    auto fetch = [&](int64_t t) {
        const float *pg = gate + c.first + t * channels, *pv = value + c.first + t * channels;
        if (__all_sync(0xffffffffu, t + S <= c.steps)) {
#pragma unroll
            for (int i = 0; i < S; ++i)
                g[i] = __ldcs(pg + (int64_t)i * channels), v[i] = __ldcs(pv + (int64_t)i * channels);
        } else {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool in = t + i < c.steps;
                g[i]          = in ? __ldcs(pg + (int64_t)i * channels) : INFINITY;
                v[i]          = in ? __ldcs(pv + (int64_t)i * channels) : 0.0f;
            }
        }
    };
    fetch(t0);
    const int tiles = (int)((steps + tile - 1) / tile);
    for (int i = 0; i < tiles; ++i, t0 += tile) {
        float a[S], add[S];
        Piece mine;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            float rest;
            sigmoids(g[j], a[j], rest);
            add[j] = __fmul_rn(rest, v[j]);
            mine.step(a[j], rest, add[j]);
        }
        fetch(t0 + tile);
        float h = (float)exchange(ex, i, mine, state, warp, lane, blocks, rank);
        if (out) {
            float *to = out + c.first + t0 * channels;
            if (__all_sync(0xffffffffu, t0 + S <= c.steps)) {
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    h = __fmaf_rn(a[j], h, add[j]);
                    __stcs(to + (int64_t)j * channels, h);
                }
            } else {
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    h = __fmaf_rn(a[j], h, add[j]);
                    if (c.here && t0 + j < steps)
                        __stcs(to + (int64_t)j * channels, t0 + j < c.steps ? h : 0.0f);
                }
            }
        }
    }
    if (state_out && warp == 0 && rank == 0 && c.here)
        state_out[c.index] = (float)state;
    exchange_end(ex, blocks, flags);
}

// The same along the reversed axis: piece u of a tile ends u S steps before the tile's end.
template <int W, int S, int FIT>
__global__ void __launch_bounds__(W * 32, FIT) gated_scan_grad_kernel(
    const float *__restrict__ gate, const float *__restrict__ value, const float *state0, const int64_t *__restrict__ lengths,
    const float *__restrict__ out, const float *__restrict__ dout, const float *dstate, int64_t chains, int64_t steps, int channels, int blocks,
    float *__restrict__ dgate, float *__restrict__ dvalue, float *dstate0, uint32_t *__restrict__ flags) {
    __shared__ Exchange<W> ex;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = blocks > 1 ? cluster_rank() : 0;
    exchange_begin(ex, blocks);
    griddep_wait();
    const Chain c      = chain_of((int64_t)(blockIdx.x / blocks) * 32 + lane, chains, steps, channels, lengths);
    double state       = c.here && dstate ? (double)dstate[c.index] : 0.0; // c[t+1]
    const float first  = c.here && state0 ? state0[c.index] : 0.0f;
    const int64_t tile = (int64_t)blocks * W * S;
    int64_t t1         = steps - 1 - ((int64_t)rank * W + warp) * S; // the piece's last step
    float g[S], v[S], d[S], h[S];
    auto fetch = [&](int64_t t) {
        const int64_t at = c.first + t * channels;
        if (__all_sync(0xffffffffu, t < c.steps && t >= S)) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                g[i] = __ldcs(gate + at - (int64_t)i * channels), v[i] = __ldcs(value + at - (int64_t)i * channels);
                d[i] = __ldcs(dout + at - (int64_t)i * channels), h[i] = __ldcs(out + at - (int64_t)(i + 1) * channels);
            }
        } else {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool in = t - i >= 0 && t - i < c.steps;
                g[i]          = in ? __ldcs(gate + at - (int64_t)i * channels) : INFINITY;
                v[i]          = in ? __ldcs(value + at - (int64_t)i * channels) : 0.0f;
                d[i]          = in ? __ldcs(dout + at - (int64_t)i * channels) : 0.0f;
                h[i]          = in ? (t - i > 0 ? __ldcs(out + at - (int64_t)(i + 1) * channels) : first) : 0.0f;
            }
        }
    };
    fetch(t1);
    const int tiles = (int)((steps + tile - 1) / tile);
    for (int i = 0; i < tiles; ++i, t1 -= tile) {
        float a[S], rest[S], gap[S], dy[S];
        Piece mine;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            sigmoids(g[j], a[j], rest[j]);
            gap[j] = __fsub_rn(h[j], v[j]);
            dy[j]  = d[j];
            mine.step(a[j], rest[j], __fmul_rn(a[j], dy[j]));
        }
        fetch(t1 - tile);
        float carry = (float)exchange(ex, i, mine, state, warp, lane, blocks, rank);
        const int64_t at = c.first + t1 * channels;
        const bool whole = __all_sync(0xffffffffu, t1 < c.steps && t1 >= S - 1);
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const float x = __fadd_rn(dy[j], carry);
            carry         = __fmul_rn(a[j], x);
            const float dv = __fmul_rn(rest[j], x), dg = __fmul_rn(__fmul_rn(rest[j], carry), gap[j]);
            if (whole || (c.here && t1 - j >= 0)) {
                const bool in = whole || t1 - j < c.steps;
                if (dvalue)
                    __stcs(dvalue + at - (int64_t)j * channels, in ? dv : 0.0f);
                if (dgate)
                    __stcs(dgate + at - (int64_t)j * channels, in ? dg : 0.0f);
            }
        }
    }
    if (dstate0 && warp == 0 && rank == 0 && c.here)
        dstate0[c.index] = (float)state;
    exchange_end(ex, blocks, flags);
}

// A few steps, S at most: a thread goes through those of V chains, all of which are on their way together.
template <int V, int S>
__global__ void __launch_bounds__(128) gated_steps_kernel(
    const float *__restrict__ gate, const float *__restrict__ value, const float *state0, const int64_t *__restrict__ lengths, int64_t chains, int steps,
    int channels, float *__restrict__ out, float *state_out) {
    using Values = std::conditional_t<V == 4, float4, float>;
    griddep_wait();
    const Chain c = chain_of(((int64_t)blockIdx.x * 128 + threadIdx.x) * V, chains, steps, channels, lengths);
    if (!c.here)
        return;
    alignas(16) float g[S][V], v[S][V], h[V];
    auto load = [](const float *from, float (&to)[V]) { *reinterpret_cast<Values *>(to) = *reinterpret_cast<const Values *>(from); };
    auto store = [](float *to, const float (&from)[V]) { *reinterpret_cast<Values *>(to) = *reinterpret_cast<const Values *>(from); };
#pragma unroll
    for (int j = 0; j < S; ++j)
        if (j < c.steps) {
            load(gate + c.first + (int64_t)j * channels, g[j]);
            load(value + c.first + (int64_t)j * channels, v[j]);
        }
#pragma unroll
    for (int q = 0; q < V; ++q)
        h[q] = 0.0f;
    if (state0)
        load(state0 + c.index, h);
#pragma unroll
    for (int j = 0; j < S; ++j)
        if (j < steps) {
            alignas(16) float to[V];
#pragma unroll
            for (int q = 0; q < V; ++q) {
                to[q] = 0.0f;
                if (j < c.steps) {
                    float a, rest;
                    sigmoids(g[j][q], a, rest);
                    to[q] = h[q] = __fmaf_rn(a, h[q], __fmul_rn(rest, v[j][q]));
                }
            }
            if (out)
                store(out + c.first + (int64_t)j * channels, to);
        }
    if (state_out)
        store(state_out + c.index, h);
}

template <int V, int S>
__global__ void __launch_bounds__(128) gated_steps_grad_kernel(
    const float *__restrict__ gate, const float *__restrict__ value, const float *state0, const int64_t *__restrict__ lengths,
    const float *__restrict__ out, const float *__restrict__ dout, const float *dstate, int64_t chains, int steps, int channels,
    float *__restrict__ dgate, float *__restrict__ dvalue, float *dstate0) {
    using Values = std::conditional_t<V == 4, float4, float>;
    griddep_wait();
    const Chain c = chain_of(((int64_t)blockIdx.x * 128 + threadIdx.x) * V, chains, steps, channels, lengths);
    if (!c.here)
        return;
    alignas(16) float g[S][V], v[S][V], d[S][V], h[S][V], last[V]; // h: before the step
    auto load = [](const float *from, float (&to)[V]) { *reinterpret_cast<Values *>(to) = *reinterpret_cast<const Values *>(from); };
    auto store = [](float *to, const float (&from)[V]) { *reinterpret_cast<Values *>(to) = *reinterpret_cast<const Values *>(from); };
#pragma unroll
    for (int q = 0; q < V; ++q)
        last[q] = h[0][q] = 0.0f;
#pragma unroll
    for (int j = 0; j < S; ++j)
        if (j < c.steps) {
            load(gate + c.first + (int64_t)j * channels, g[j]);
            load(value + c.first + (int64_t)j * channels, v[j]);
            load(dout + c.first + (int64_t)j * channels, d[j]);
            if (j > 0)
                load(out + c.first + (int64_t)(j - 1) * channels, h[j]);
        }
    if (state0)
        load(state0 + c.index, h[0]);
    if (dstate)
        load(dstate + c.index, last);
    double carry[V];
#pragma unroll
    for (int q = 0; q < V; ++q)
        carry[q] = (double)last[q];
#pragma unroll
    for (int j = S - 1; j >= 0; --j)
        if (j < steps) {
            alignas(16) float dg[V], dv[V];
#pragma unroll
            for (int q = 0; q < V; ++q) {
                dg[q] = dv[q] = 0.0f;
                if (j < c.steps) {
                    float a, rest;
                    sigmoids(g[j][q], a, rest);
                    const double x = (double)d[j][q] + carry[q];
                    carry[q]       = (rest <= 0.5f ? 1.0 - (double)rest : (double)a) * x;
                    dv[q]          = __fmul_rn(rest, (float)x);
                    dg[q]          = __fmul_rn(__fmul_rn(rest, (float)carry[q]), __fsub_rn(h[j][q], v[j][q]));
                }
            }
            if (dvalue)
                store(dvalue + c.first + (int64_t)j * channels, dv);
            if (dgate)
                store(dgate + c.first + (int64_t)j * channels, dg);
        }
#pragma unroll
    for (int q = 0; q < V; ++q)
        last[q] = (float)carry[q];
    if (dstate0)
        store(dstate0 + c.index, last);
}

constexpr int kFewSteps = 16;

bool aligned16(std::initializer_list<const void *> all) { // null is
    for (const void *p : all)
        if (reinterpret_cast<uintptr_t>(p) & 15u)
            return false;
    return true;
}

ct_status check_scan(const char *name, int64_t batch, int64_t steps, int64_t channels) {
    if (batch < 0 || steps < 0 || channels < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (batch > 1 << 29 || steps > 1 << 29 || channels > 1 << 29)
        return fail(CT_ERR_TOO_LARGE, "%s: dimension too large", name);
    // a block has 32 chains, and a grid 2^31 - 1 blocks at most
    if (batch * channels > (int64_t)1 << 32)
        return fail(CT_ERR_TOO_LARGE, "%s: more than 2^32 states", name);
    return CT_OK;
}

// Blocks to a cluster: while the groups of 32 chains do not fill the machine, and a tile does not exceed the steps.
int scan_blocks(const DeviceState *st, int64_t groups, int64_t steps, int piece) {
    int blocks = 1;
    while (blocks < 8 && groups * blocks * 2 <= st->sm_count * 2 && steps > (int64_t)blocks * piece)
        blocks *= 2;
    return blocks;
}

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_gated_scan(
    const float *gate, const float *value, const float *state0, const int64_t *lengths, int64_t batch, int64_t steps, int64_t channels, float *out,
    float *state) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_scan("gated_scan", batch, steps, channels));
    const int64_t chains = batch * channels;
    if (chains == 0 || (!out && !state))
        return CT_OK;
    if (steps > 0 && (!gate || !value))
        return fail(CT_ERR_INVALID, "gated_scan: null pointer");
    ProfScope prof("gated_scan");
    constexpr int W = 8, S = 16;
    if (steps <= kFewSteps) {
        const bool four = channels % 4 == 0 && aligned16({gate, value, state0, out, state});
        auto launch     = [&](auto kernel, int v) -> ct_status {
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)((chains / v + 127) / 128)), dim3(128), 0, stream(), gate, value, state0, lengths, chains, (int)steps,
                                     (int)channels, out, state));
            CT_LAUNCH_CHECK("gated_steps");
            return CT_OK;
        };
        if (steps <= 1)
            return four ? launch(gated_steps_kernel<4, 1>, 4) : launch(gated_steps_kernel<1, 1>, 1);
        if (steps <= 4)
            return four ? launch(gated_steps_kernel<4, 4>, 4) : launch(gated_steps_kernel<1, 4>, 1);
        return launch(gated_steps_kernel<1, kFewSteps>, 1);
    }
    const int64_t groups = (chains + 31) / 32;
    const int blocks     = scan_blocks(st, groups, steps, W * S);
    CT_CUDA(launch_dependent_cluster(gated_scan_kernel<W, S, 2>, blocks, dim3((unsigned)(groups * blocks)), dim3(W * 32), 0, stream(), gate, value, state0,
                                     lengths, chains, steps, (int)channels, blocks, out, state, st->flags_dev));
    CT_LAUNCH_CHECK("gated_scan");
    return CT_OK;
}

ct_status ct_gated_scan_grad(
    const float *gate, const float *value, const float *state0, const int64_t *lengths, const float *out, const float *dout, const float *dstate,
    int64_t batch, int64_t steps, int64_t channels, float *dgate, float *dvalue, float *dstate0) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_scan("gated_scan_grad", batch, steps, channels));
    const int64_t chains = batch * channels;
    if (chains == 0 || (!dgate && !dvalue && !dstate0))
        return CT_OK;
    if (steps > 0 && (!gate || !value || !out || !dout))
        return fail(CT_ERR_INVALID, "gated_scan_grad: null pointer");
    ProfScope prof("gated_scan_grad");
    constexpr int W = 8, S = 8;
    if (steps <= kFewSteps) {
        const bool four = channels % 4 == 0 && aligned16({gate, value, state0, out, dout, dstate, dgate, dvalue, dstate0});
        auto launch     = [&](auto kernel, int v) -> ct_status {
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)((chains / v + 127) / 128)), dim3(128), 0, stream(), gate, value, state0, lengths, out, dout, dstate,
                                     chains, (int)steps, (int)channels, dgate, dvalue, dstate0));
            CT_LAUNCH_CHECK("gated_steps_grad");
            return CT_OK;
        };
        if (steps <= 1)
            return four ? launch(gated_steps_grad_kernel<4, 1>, 4) : launch(gated_steps_grad_kernel<1, 1>, 1);
        if (steps <= 4)
            return four ? launch(gated_steps_grad_kernel<4, 4>, 4) : launch(gated_steps_grad_kernel<1, 4>, 1);
        return launch(gated_steps_grad_kernel<1, kFewSteps>, 1);
    }
    const int64_t groups = (chains + 31) / 32;
    const int blocks     = scan_blocks(st, groups, steps, W * S);
    CT_CUDA(launch_dependent_cluster(gated_scan_grad_kernel<W, S, 2>, blocks, dim3((unsigned)(groups * blocks)), dim3(W * 32), 0, stream(), gate, value, state0,
                                     lengths, out, dout, dstate, chains, steps, (int)channels, blocks, dgate, dvalue, dstate0, st->flags_dev));
    CT_LAUNCH_CHECK("gated_scan_grad");
    return CT_OK;
}

} // extern "C"
