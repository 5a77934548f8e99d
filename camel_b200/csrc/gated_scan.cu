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
// Of a gate only the smaller of a and 1 - a is kept, with all its digits (the sign tells which): a state moves from h towards value by 1 - a, or from
// value towards h by a.  Held as a float32, an `a` near 1 would be off by 2^-25, which a state that remembers 1 / (1 - a) steps adds up.
#include "common.cuh"
#include "gate.cuh"
#include "tc_ptx.cuh"

#include <algorithm>

namespace ct {
namespace {

using namespace ptx;

// The smaller of a and 1 - a: 1 - a as it is, a with its sign bit set.
__device__ __forceinline__ float smaller_side(float gate) {
    float a, rest;
    sigmoids(gate, a, rest);
    return gate >= 0.0f ? rest : -a;
}
__device__ __forceinline__ bool keeps(float side) { return __float_as_int(side) >= 0; } // a >= 1/2
// a h + (1 - a) v
__device__ __forceinline__ float move(float side, float h, float v) {
    const float from = keeps(side) ? h : v, to = keeps(side) ? v : h;
    return __fmaf_rn(fabsf(side), __fsub_rn(to, from), from);
}
// a x
__device__ __forceinline__ float times_a(float side, float x) { return keeps(side) ? __fmaf_rn(-side, x, x) : __fmul_rn(-side, x); }
__device__ __forceinline__ float one_minus_a(float side) { return keeps(side) ? side : __fadd_rn(1.0f, side); }

// What a piece of a chain does to the state before it: a h + b, a held like a gate's.
struct Piece {
    float side, b;
};
__device__ __forceinline__ double apply(Piece p, double h) {
    const double a = keeps(p.side) ? 1.0 - (double)p.side : -(double)p.side;
    return fma(a, h, (double)p.b);
}

// The state before each warp's steps, from what all pieces of the tile do; `state` goes on to the tile's end.  Pieces lie in the order of warps, and
// of the cluster's blocks.  One call after the other alternates between two places (turn), so that a fast warp does not write over what a slow one reads.
template <int W> struct Exchange {
    Piece pieces[2][W][32];
    double2 blocks[2][16][32]; // (a, b) of the cluster's blocks
};
template <int W>
__device__ __forceinline__ double exchange(Exchange<W> &e, int turn, Piece mine, double &state, int warp, int lane, int blocks, uint32_t rank) {
    e.pieces[turn][warp][lane] = mine;
    __syncthreads();
    double before = state;
    if (blocks > 1) {
        if (warp == 0) {
            double a = 1.0, b = 0.0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const Piece p = e.pieces[turn][w][lane];
                b             = apply(p, b);
                a *= keeps(p.side) ? 1.0 - (double)p.side : -(double)p.side;
            }
            const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(&e.blocks[turn][rank][lane]));
            for (int r = 0; r < blocks; ++r)
                asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(mapa(at, r)), "d"(a), "d"(b) : "memory");
        }
        cluster_sync();
        for (int r = 0; r < blocks; ++r) {
            const double2 p = e.blocks[turn][r][lane];
            before          = r == (int)rank ? state : before;
            state           = fma(p.x, state, p.y);
        }
#pragma unroll
        for (int w = 0; w < W; ++w)
            if (w < warp)
                before = apply(e.pieces[turn][w][lane], before);
    } else {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            before = w == warp ? state : before;
            state  = apply(e.pieces[turn][w][lane], state);
        }
    }
    return before;
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
    c.index         = index;
    const int64_t b = index / channels;
    c.first         = b * steps * channels + (index - b * channels);
    c.steps         = steps;
    if (c.here && lengths) {
        const int64_t length = lengths[b];
        c.steps              = length < 0 ? 0 : (length < steps ? length : steps);
    }
    return c;
}

// W warps to a block; the blocks of a cluster have the same 32 chains.
template <int W, int S>
__global__ void __launch_bounds__(W * 32) gated_scan_kernel(
    const float *__restrict__ gate, const float *__restrict__ value, const float *state0, const int64_t *__restrict__ lengths, int64_t chains,
    int64_t steps, int64_t channels, int blocks, float *__restrict__ out, float *state_out) {
    __shared__ Exchange<W> ex;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = blocks > 1 ? cluster_rank() : 0;
    if (blocks > 1)
        cluster_sync(); // every block of the cluster runs before another writes into its memory
    griddep_wait();
    const Chain c     = chain_of((int64_t)(blockIdx.x / blocks) * 32 + lane, chains, steps, channels, lengths);
    double state      = c.here && state0 ? (double)state0[c.index] : 0.0;
    const int64_t tile = (int64_t)blocks * W * S;
    int64_t t0         = ((int64_t)rank * W + warp) * S;
    const float *pg = gate + c.first, *pv = value + c.first;
    float g[S], v[S];
    auto fetch = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool in = c.here && t + i < c.steps;
            g[i]          = in ? __ldcs(pg + (t + i) * channels) : 0.0f;
            v[i]          = in ? __ldcs(pv + (t + i) * channels) : 0.0f;
        }
    };
    fetch(t0);
    int turn = 0;
    for (int64_t base = 0; base < steps; base += tile, t0 += tile, turn ^= 1) {
        float side[S], val[S];
        Piece mine = {0.0f, 0.0f};
        float a    = 1.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool in = t0 + i < c.steps;
            side[i]       = in ? smaller_side(g[i]) : 0.0f;
            val[i]        = v[i];
            if (in) {
                mine.b    = move(side[i], mine.b, val[i]);
                mine.side = move(side[i], mine.side, 1.0f); // 1 - the product of all a
                a         = times_a(side[i], a);
            }
        }
        if (a < 0.5f)
            mine.side = -a;
        fetch(t0 + tile);
        float h = (float)exchange<W>(ex, turn, mine, state, warp, lane, blocks, rank);
        if (out && c.here) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool in = t0 + i < c.steps;
                if (in)
                    h = move(side[i], h, val[i]);
                if (t0 + i < steps)
                    __stcs(out + c.first + (t0 + i) * channels, in ? h : 0.0f);
            }
        }
    }
    if (state_out && warp == 0 && rank == 0 && c.here)
        state_out[c.index] = (float)state;
}

// The same along the reversed axis: piece u of a tile ends u S steps before the tile's end.
template <int W, int S>
__global__ void __launch_bounds__(W * 32) gated_scan_grad_kernel(
    const float *__restrict__ gate, const float *__restrict__ value, const float *state0, const int64_t *__restrict__ lengths,
    const float *__restrict__ out, const float *__restrict__ dout, const float *dstate, int64_t chains, int64_t steps, int64_t channels, int blocks,
    float *__restrict__ dgate, float *__restrict__ dvalue, float *dstate0) {
    __shared__ Exchange<W> ex;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = blocks > 1 ? cluster_rank() : 0;
    if (blocks > 1)
        cluster_sync();
    griddep_wait();
    const Chain c      = chain_of((int64_t)(blockIdx.x / blocks) * 32 + lane, chains, steps, channels, lengths);
    double state       = c.here && dstate ? (double)dstate[c.index] : 0.0; // c[t+1]
    const float first  = c.here && state0 ? state0[c.index] : 0.0f;
    const int64_t tile = (int64_t)blocks * W * S;
    int64_t t1         = steps - 1 - ((int64_t)rank * W + warp) * S; // the piece's last step
    float g[S], v[S], d[S], h[S];
    auto fetch = [&](int64_t t) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool in    = c.here && t - i >= 0 && t - i < c.steps;
            const int64_t at = c.first + (t - i) * channels;
            g[i]             = in ? __ldcs(gate + at) : 0.0f;
            v[i]             = in ? __ldcs(value + at) : 0.0f;
            d[i]             = in ? __ldcs(dout + at) : 0.0f;
            h[i]             = in ? (t - i > 0 ? __ldcs(out + at - channels) : first) : 0.0f;
        }
    };
    fetch(t1);
    int turn = 0;
    for (int64_t base = 0; base < steps; base += tile, t1 -= tile, turn ^= 1) {
        float side[S], gap[S], dy[S];
        Piece mine = {0.0f, 0.0f};
        float a    = 1.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const bool in = t1 - i >= 0 && t1 - i < c.steps;
            side[i]       = in ? smaller_side(g[i]) : 0.0f;
            gap[i]        = __fsub_rn(h[i], v[i]);
            dy[i]         = d[i];
            if (in) {
                mine.b    = times_a(side[i], __fadd_rn(dy[i], mine.b));
                mine.side = move(side[i], mine.side, 1.0f);
                a         = times_a(side[i], a);
            }
        }
        if (a < 0.5f)
            mine.side = -a;
        fetch(t1 - tile);
        float carry = (float)exchange<W>(ex, turn, mine, state, warp, lane, blocks, rank);
        if (c.here) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const bool in    = t1 - i >= 0 && t1 - i < c.steps;
                const int64_t at = c.first + (t1 - i) * channels;
                float dv = 0.0f, dg = 0.0f;
                if (in) {
                    const float x = __fadd_rn(dy[i], carry), rest = one_minus_a(side[i]);
                    carry = times_a(side[i], x);
                    dv    = __fmul_rn(rest, x);
                    dg    = __fmul_rn(__fmul_rn(rest, carry), gap[i]);
                }
                if (t1 - i >= 0) {
                    if (dvalue)
                        __stcs(dvalue + at, dv);
                    if (dgate)
                        __stcs(dgate + at, dg);
                }
            }
        }
    }
    if (dstate0 && warp == 0 && rank == 0 && c.here)
        dstate0[c.index] = (float)state;
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
    const int64_t groups = (chains + 31) / 32;
    const int blocks     = scan_blocks(st, groups, steps, W * S);
    CT_CUDA(launch_dependent_cluster(gated_scan_kernel<W, S>, blocks, dim3((unsigned)(groups * blocks)), dim3(W * 32), 0, stream(), gate, value, state0,
                                     lengths, chains, steps, channels, blocks, out, state));
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
    const int64_t groups = (chains + 31) / 32;
    const int blocks     = scan_blocks(st, groups, steps, W * S);
    CT_CUDA(launch_dependent_cluster(gated_scan_grad_kernel<W, S>, blocks, dim3((unsigned)(groups * blocks)), dim3(W * 32), 0, stream(), gate, value, state0,
                                     lengths, out, dout, dstate, chains, steps, channels, blocks, dgate, dvalue, dstate0));
    CT_LAUNCH_CHECK("gated_scan_grad");
    return CT_OK;
}

} // extern "C"
