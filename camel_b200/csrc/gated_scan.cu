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
//
// Measured (L2 flushed, and in line): one sequence of 65536 steps and 512 channels 78 to 81 us forward, in line 74 (403 MB, 0.76 to 0.83 of a copy; a tile waits for
// what the blocks before send), and 138, 134 backward; 8 of 2048 steps and 2048 channels 72 and 63, backward 127 to 133 and 126 us (805 MB, 0.92 to 0.98); 7 of up to
// 1537 steps and 771 channels backward 48 and 50 us (166 MB, 0.5: rows that begin anywhere lie in two lines of 128 bytes; in line 772 channels take 38, 768 32); one
// step of 64 x 2048 5 us.
// Times at the rules below are of a lone call between two events, L2 flushed, with the events' own 4 us or so, unless in line is said: call behind call.
#include "common.cuh"
#include "fastmath.cuh"
#include "gate.cuh"
#include "scan_walk.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

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

// a and 1 - a of two gates, in the machine's two-lane instructions: a scan is bound by their number as much as by memory.  With e = exp(-gate),
// 2^t of the rounded t = -gate log2(e) and what that lacks, a is 1 / (1 + e), from a reciprocal and a Newton step, and 1 - a is e a: to 2 U and to 7 U of
// themselves (U = 2^-24), and 2^-26 |gate| more of what the float32 log2(e) lacks.  Gates below -87.33654 count as that: 1 + e is not above 2^126, whose
// reciprocal is the smallest number that ftz leaves.
// N pairs together, stage by stage: one after the other they wait for their exponentials and reciprocals (the pieces of a tile 2000 clocks).
template <int N> __device__ __forceinline__ void sigmoids2(const float *g, f32x2 (&a)[N], f32x2 (&rest)[N]) {
    f32x2 x[N], t[N], e[N];
    auto each = [](auto &&stage) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            stage(i);
    };
    each([&](int i) {
        float g0 = g[2 * i], g1 = g[2 * i + 1];
        asm("max.NaN.f32 %0, %0, 0fC2AEAC4F;" : "+f"(g0));
        asm("max.NaN.f32 %0, %0, 0fC2AEAC4F;" : "+f"(g1));
        asm("min.NaN.f32 %0, %0, 0f42D00000;" : "+f"(g0)); // 104: e is 0 there
        asm("min.NaN.f32 %0, %0, 0f42D00000;" : "+f"(g1));
        x[i] = pack2(g0, g1);
    });
    each([&](int i) { t[i] = mul2(x[i], dup2(0xBFB8AA3Bu)); });
    each([&](int i) {
        float t0, t1;
        unpack2(t[i], t0, t1);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(t0));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(t1));
        e[i] = pack2(t0, t1);
    });
    each([&](int i) { x[i] = fma2(x[i], dup2(0x3FB8AA3Bu), t[i]); }); // minus what t lacks
    each([&](int i) { x[i] = mul2(x[i], dup2(0xBF317218u)); });       // ln 2
    each([&](int i) { e[i] = fma2(e[i], x[i], e[i]); });
    each([&](int i) { t[i] = fma2(e[i], dup2(0xBF800000u), dup2(0xBF800000u)); }); // -(1 + e)
    each([&](int i) {
        float d0, d1;
        unpack2(t[i], d0, d1);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d0) : "f"(-d0));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d1) : "f"(-d1));
        x[i] = pack2(d0, d1);
    });
    each([&](int i) { t[i] = fma2(t[i], x[i], dup2(0x3F800000u)); });
    each([&](int i) { a[i] = fma2(x[i], t[i], x[i]); });
    each([&](int i) { rest[i] = mul2(e[i], a[i]); });
}
constexpr int kPairs = 4; // together

// W warps to a block, one of them the joining one in a cluster, S steps to a lane; the blocks of a cluster have the same 32 chains.
template <int W, int S, Source FROM, bool CLUSTER, int DEPTH>
__global__ void __launch_bounds__(W * 32, 16 / W) gated_scan_kernel(
    const __grid_constant__ Arrays<2> arrays, const float *state0, const int64_t *__restrict__ lengths, int64_t chains, int64_t steps, int channels, int blocks,
    float *__restrict__ out, float *state_out, uint32_t *__restrict__ flags) {
    extern __shared__ __align__(128) float pieces[];
    constexpr int WALK = W - CLUSTER; // warps that have pieces
    __shared__ Exchange<WALK, CLUSTER> ex;
    __shared__ uint64_t arrived[W * DEPTH];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = CLUSTER ? cluster_rank() : 0;
    const int64_t group = CLUSTER ? blockIdx.x / blocks : blockIdx.x;
    Pieces<2, S, FROM, false, DEPTH> values(pieces, &arrived[warp * DEPTH], &ex.gave_up, arrays, channels);
    walk_begin(ex);
    griddep_wait();
    const Chain c = chain_of_lane<FROM>(group, lane, chains, steps, channels, lengths);
    const int tile = (CLUSTER ? blocks : 1) * WALK * S, t0 = (rank * WALK + warp) * S;
    values.at(c, group, chains, steps, t0);
    int last       = __reduce_max_sync(0xffffffffu, (unsigned)c.steps); // behind it the warp has nothing but zeros to write
    auto fetch     = [&](int i) {
        const int t = t0 + i * tile;
        values.fetch(i, t, -1, (FROM == SINGLE ? c.steps : last) - t, last);
    };
    if (warp < WALK)
        for (int i = 0; i < DEPTH; ++i)
            fetch(i);
    struct Steps {
        float a[S], add[S];
    };
    const double state = walk<Steps>(
        ex, (int)((steps + tile - 1) / tile), c.here && state0 ? (double)state0[c.index] : 0.0, blocks,
        [&](int i, Steps &s) {
            const int t = t0 + i * tile, count = c.steps - t;
            Piece p;
            if (t >= last) {
                fetch(i + DEPTH);
                return p.joined();
            }
            values.wait(i, last);
            values.read(i, 0, t, s.a);
            values.read(i, 1, t, s.add);
            if (!__all_sync(0xffffffffu, count >= S)) {
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (j >= count) // steps that a chain does not have keep its state: a = 1, and nothing is added
                        s.a[j] = INFINITY, s.add[j] = 0.0f;
            }
            __syncwarp();
            fetch(i + DEPTH);
#pragma unroll
            for (int j0 = 0; j0 < S; j0 += 2 * kPairs) {
                f32x2 a[kPairs], rest[kPairs];
                sigmoids2(s.a + j0, a, rest);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) {
                    const int j = j0 + 2 * i;
                    unpack2(mul2(rest[i], pack2(s.add[j], s.add[j + 1])), s.add[j], s.add[j + 1]);
                    unpack2(a[i], s.a[j], s.a[j + 1]);
                    float r0, r1;
                    unpack2(rest[i], r0, r1);
                    p.step(s.a[j], r0, s.add[j]);
                    p.step(s.a[j + 1], r1, s.add[j + 1]);
                }
            }
            return p.joined();
        },
        [&](int i, const Steps &s, float before) {
            if (!out)
                return;
            const int t = t0 + i * tile, count = c.steps - t;
            float *to   = out + c.first + (int64_t)t * channels;
            float h     = before;
            if (t >= last) {
                if (c.here)
#pragma unroll
                    for (int j = 0; j < S; ++j)
                        if (t + j < steps)
                            to[(int64_t)j * channels] = 0.0f;
            } else if (__all_sync(0xffffffffu, count >= S)) {
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    h = __fmaf_rn(s.a[j], h, s.add[j]);
                    to[(int64_t)j * channels] = h;
                }
            } else if (c.here) {
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    h = __fmaf_rn(s.a[j], h, s.add[j]);
                    if (t + j < steps)
                        to[(int64_t)j * channels] = j < count ? h : 0.0f;
                }
            }
        });
    walk_end(ex, flags);
    if (state_out && warp == (CLUSTER ? WALK : 0) && rank == 0 && c.here) // (behind the other blocks' loads of state0, which it may be)
        state_out[c.index] = (float)state;
}

// The same along the reversed axis: piece u of a tile ends u S steps before the tile's end.
template <int W, int S, Source FROM, bool CLUSTER, int DEPTH>
__global__ void __launch_bounds__(W * 32, 16 / W) gated_scan_grad_kernel(
    const __grid_constant__ Arrays<4> arrays, const float *state0, const int64_t *__restrict__ lengths, const float *dstate, int64_t chains, int64_t steps,
    int channels, int blocks, float *__restrict__ dgate, float *__restrict__ dvalue, float *dstate0, uint32_t *__restrict__ flags) {
    extern __shared__ __align__(128) float pieces[];
    constexpr int WALK = W - CLUSTER; // warps that have pieces
    __shared__ Exchange<WALK, CLUSTER> ex;
    __shared__ uint64_t arrived[W * DEPTH];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t rank = CLUSTER ? cluster_rank() : 0;
    const int64_t group = CLUSTER ? blockIdx.x / blocks : blockIdx.x;
    Pieces<4, S, FROM, true, DEPTH> values(pieces, &arrived[warp * DEPTH], &ex.gave_up, arrays, channels);
    walk_begin(ex);
    griddep_wait();
    const Chain c = chain_of_lane<FROM>(group, lane, chains, steps, channels, lengths);
    const float first = c.here && state0 ? state0[c.index] : 0.0f;
    // a piece has S steps in their own order, the walk goes through them backwards; t0: the first piece's first step, which may be below 0
    const int tile = (CLUSTER ? blocks : 1) * WALK * S, t0 = (int)steps - (int)(rank * WALK + warp + 1) * S;
    values.at(c, group, chains, steps, t0);
    int last       = __reduce_max_sync(0xffffffffu, (unsigned)c.steps);
    auto fetch     = [&](int i) {
        const int t = t0 - i * tile;
        values.fetch(i, t, -t, t > -S ? (FROM == SINGLE ? c.steps : last) - t : 0, last);
    };
    if (warp < WALK)
        for (int i = 0; i < DEPTH; ++i)
            fetch(i);
    struct Steps {
        float a[S], rest[S], gap[S], dy[S]; // gap: h[t-1] - value[t]
    };
    const double state = walk<Steps>( // c[t+1]
        ex, (int)((steps + tile - 1) / tile), c.here && dstate ? (double)dstate[c.index] : 0.0, blocks,
        [&](int i, Steps &s) {
            const int t = t0 - i * tile, begin = -t, count = c.steps - t; // steps begin .. count - 1 are there
            Piece p;
            if (t >= last || t <= -S) {
                fetch(i + DEPTH);
                return p.joined();
            }
            values.wait(i, last);
            values.read(i, 0, t, s.a);
            values.read(i, 1, t, s.rest);
            values.read(i, 2, t, s.dy);
            values.read(i, 3, t, s.gap);
            if (!__all_sync(0xffffffffu, t > 0 && count >= S)) {
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    if (t + j == 0)
                        s.gap[j] = first;
                    if (j < begin || j >= count)
                        s.a[j] = INFINITY, s.rest[j] = s.dy[j] = s.gap[j] = 0.0f;
                }
            }
            __syncwarp();
            fetch(i + DEPTH);
#pragma unroll
            for (int j0 = S - 2 * kPairs; j0 >= 0; j0 -= 2 * kPairs) {
                f32x2 a[kPairs], rest[kPairs];
                sigmoids2(s.a + j0, a, rest);
#pragma unroll
                for (int i = kPairs - 1; i >= 0; --i) {
                    const int j = j0 + 2 * i;
                    float add0, add1;
                    unpack2(mul2(a[i], pack2(s.dy[j], s.dy[j + 1])), add0, add1);
                    unpack2(fma2(pack2(s.rest[j], s.rest[j + 1]), dup2(0xBF800000u), pack2(s.gap[j], s.gap[j + 1])), s.gap[j], s.gap[j + 1]);
                    unpack2(a[i], s.a[j], s.a[j + 1]);
                    unpack2(rest[i], s.rest[j], s.rest[j + 1]);
                    p.step(s.a[j + 1], s.rest[j + 1], add1);
                    p.step(s.a[j], s.rest[j], add0);
                }
            }
            return p.joined();
        },
        [&](int i, const Steps &s, float before) {
            const int t = t0 - i * tile, count = c.steps - t;
            const int64_t at = c.first + (int64_t)t * channels;
            float *dg = dgate + at, *dv = dvalue + at;
            float carry = before;
            auto slopes = [&](int j, float &g, float &v) {
                const float x = __fadd_rn(s.dy[j], carry);
                carry         = __fmul_rn(s.a[j], x);
                v             = __fmul_rn(s.rest[j], x);
                g             = __fmul_rn(__fmul_rn(s.rest[j], carry), s.gap[j]);
            };
            if (t >= last) {
                if (c.here)
#pragma unroll
                    for (int j = 0; j < S; ++j)
                        if (t + j >= 0) {
                            if (dvalue)
                                dv[(int64_t)j * channels] = 0.0f;
                            if (dgate)
                                dg[(int64_t)j * channels] = 0.0f;
                        }
            } else if (dgate && dvalue && __all_sync(0xffffffffu, t >= 0 && count >= S)) {
#pragma unroll
                for (int j = S - 1; j >= 0; --j)
                    slopes(j, dg[(int64_t)j * channels], dv[(int64_t)j * channels]);
            } else if (c.here && t > -S) {
#pragma unroll
                for (int j = S - 1; j >= 0; --j) {
                    float g, v;
                    slopes(j, g, v);
                    if (t + j >= 0) {
                        if (dvalue)
                            dv[(int64_t)j * channels] = j < count ? v : 0.0f;
                        if (dgate)
                            dg[(int64_t)j * channels] = j < count ? g : 0.0f;
                    }
                }
            }
        });
    walk_end(ex, flags);
    if (dstate0 && warp == (CLUSTER ? WALK : 0) && rank == 0 && c.here) // (behind the other blocks' loads of dstate, which it may be)
        dstate0[c.index] = (float)state;
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

// Steps up to which a thread goes through a chain, measured (us; that, and the walk of tiles; 512 x 512 chains): 5 steps 12 and 23, 16 steps 16 and 23;
// backward, where it is 4, 5 steps 24 and 23, 16 steps 57 and 29.
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

// Blocks to a cluster: as many as let all groups of 32 chains run at once, and have a piece of the steps each.  (Clusters that wait for others' end cost a
// second walk: 16 groups in clusters of 8, of which 15 fit beside one another, took twice the time.)
template <auto KERNEL, int W> ct_status scan_blocks(const DeviceState *st, int smem, int64_t groups, int64_t pieces, int *blocks) {
    static int fit[16][kMostBlocks<W> + 1] = {}; // clusters at once, by device and size; [1] 1 when they are known.  Under the entry points' lock
    int *mine                           = fit[st->device & 15];
    if (mine[1] == 0) {
        CT_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        CT_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        for (int size = 2; size <= kMostBlocks<W>; ++size) {
            cudaLaunchAttribute attr{};
            attr.id               = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = (unsigned)size, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((unsigned)size), cfg.blockDim = dim3((unsigned)W * 32), cfg.dynamicSmemBytes = (size_t)smem;
            cfg.attrs = &attr, cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&mine[size], KERNEL, &cfg) != cudaSuccess) {
                cudaGetLastError();
                mine[size] = 0;
            }
        }
        mine[1] = 1;
    }
    *blocks = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(kMostBlocks<W>, cluster_limit()), pieces));
    while (*blocks > 1 && mine[*blocks] < groups)
        --*blocks;
    return CT_OK;
}

template <int ARRAYS> ct_status encode_arrays(Source from, Arrays<ARRAYS> &arrays, int64_t batch, int64_t steps, int64_t channels, int rows) {
    const uint64_t c = (uint64_t)channels, t = (uint64_t)steps, b = (uint64_t)batch;
    const uint64_t tiles[3] = {c, t, b}, tile_strides[2] = {c * 4, t * c * 4}, fours[2] = {4 * c, b * t / 4}, four_strides[1] = {16 * c};
    const uint32_t tile_box[3] = {32, (uint32_t)rows, 1}, four_box[2] = {36, (uint32_t)rows / 4};
    for (int k = 0; k < ARRAYS; ++k)
        CT_TRY(from == TILES ? encode_tiled_map_f32(&arrays.map[k], arrays.base[k], 3, tiles, tile_strides, tile_box, 0)
                             : encode_tiled_map_f32(&arrays.map[k], arrays.base[k], 2, fours, four_strides, four_box, 0));
    return CT_OK;
}

int64_t scan_groups(Source from, int64_t batch, int64_t channels) {
    return from == SINGLE ? (batch * channels + 31) / 32 : batch * ((channels + 31) / 32);
}

#define CT_SCAN(NAME, KERNEL, W, S, FROM, DEPTH, PIECES, ...)                                                                                              \
    [&]() -> ct_status {                                                                                                                                 \
        constexpr int smem   = (W) * PIECES::FLOATS * 4;                                                                                                   \
        const int64_t groups = scan_groups(FROM, batch, channels);                                                                                       \
        int blocks;                                                                                                                                      \
        CT_TRY((scan_blocks<KERNEL<W, S, FROM, true, DEPTH>, W>(st, smem * (DEPTH), groups, (steps + ((W)-1) * (S)-1) / (((W)-1) * (S)), &blocks)));              \
        auto kernel = blocks > 1 ? KERNEL<W, S, FROM, true, DEPTH> : KERNEL<W, S, FROM, false, 1>;                                                   \
        if (blocks == 1)                                                                                                                                 \
            CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));                                                    \
        CT_CUDA(launch_dependent_cluster(kernel, blocks, dim3((unsigned)(groups * blocks)), dim3((W) * 32), blocks > 1 ? smem * (DEPTH) : smem, stream(), __VA_ARGS__));               \
        CT_LAUNCH_CHECK(NAME);                                                                                                                           \
        return CT_OK;                                                                                                                                    \
    }()

Source scan_source(int64_t batch, int64_t steps, int64_t channels, bool aligned) {
    // groups of fewer channels would leave lanes without a chain; a tensor map has 31 bits for a row and 40 for a stride
    if (channels < 32 || !aligned || steps * channels >= (int64_t)1 << 37 || batch * steps >= (int64_t)1 << 31)
        return SINGLE;
    return channels % 4 == 0 ? TILES : ROWS;
}
// Warps to a block: 8, two such blocks to an SM, where clusters of them fill most of the machine; else 4, four to an SM.  Measured (us forward, backward; 4 and 8
// warps): 64 groups of chains, 2048 steps 21 and 19, 31 and 29; 128 groups, 4000 steps 47 and 45, 82 and 76; 175 groups, 1537 steps (59 %) 33 and 33, 55 and 64;
// 192 groups, 2048 steps (65 %) 45 and 39, 76 and 66; 256 groups, 1500 steps 39 and 33, 66 and 57; 320 groups, 1500 steps 47 and 49, 83 and 86; 512 groups,
// 2048 steps 72 and 74, 134 and 137.  2 for few steps: 16000 groups, 20 steps 45, by 4 81.
int scan_warps(const DeviceState *st, int64_t groups, int64_t steps) {
    const int64_t blocks = 2 * st->sm_count;
    return steps <= 32 ? 2 : blocks / groups * groups * 8 >= blocks * 5 ? 8 : 4;
}

template <int W, Source FROM, int DEPTH>
ct_status launch_scan(
    const DeviceState *st, const float *gate, const float *value, const float *state0, const int64_t *lengths, int64_t batch, int64_t steps, int64_t channels,
    float *out, float *state) {
    constexpr int S = 16;
    const int64_t chains = batch * channels;
    using Values         = Pieces<2, S, FROM, false, 1>;
    Arrays<2> arrays     = {{}, {gate, value}};
    if (FROM != SINGLE)
        CT_TRY(encode_arrays(FROM, arrays, batch, steps, channels, S));
    return CT_SCAN("gated_scan", gated_scan_kernel, W, S, FROM, DEPTH, Values, arrays, state0, lengths, chains, steps, (int)channels, blocks, out, state,
                   st->flags_dev);
}
template <int W, Source FROM, int DEPTH>
ct_status launch_scan_grad(
    const DeviceState *st, const float *gate, const float *value, const float *state0, const int64_t *lengths, const float *out, const float *dout,
    const float *dstate, int64_t batch, int64_t steps, int64_t channels, float *dgate, float *dvalue, float *dstate0) {
    constexpr int S = 8;
    const int64_t chains = batch * channels;
    using Values         = Pieces<4, S, FROM, true, 1>;
    Arrays<4> arrays     = {{}, {gate, value, dout, out}};
    if (FROM != SINGLE)
        CT_TRY(encode_arrays(FROM, arrays, batch, steps, channels, S));
    return CT_SCAN("gated_scan_grad", gated_scan_grad_kernel, W, S, FROM, DEPTH, Values, arrays, state0, lengths, dstate, chains, steps,
                   (int)channels, blocks, dgate, dvalue, dstate0, st->flags_dev);
}
#undef CT_SCAN

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
    const Source from = scan_source(batch, steps, channels, aligned16({gate, value}));
    auto launch       = [&](auto warps) -> ct_status {
        constexpr int W = decltype(warps)::value;
        switch (from) {
        case TILES:
            return launch_scan<W, TILES, W == 2 ? 1 : 2>(st, gate, value, state0, lengths, batch, steps, channels, out, state);
        case ROWS:
            return launch_scan<W, ROWS, 1>(st, gate, value, state0, lengths, batch, steps, channels, out, state);
        default:
            return launch_scan<W, SINGLE, 1>(st, gate, value, state0, lengths, batch, steps, channels, out, state);
        }
    };
    switch (scan_warps(st, scan_groups(from, batch, channels), steps)) {
    case 2:
        return launch(std::integral_constant<int, 2>{});
    case 4:
        return launch(std::integral_constant<int, 4>{});
    default:
        return launch(std::integral_constant<int, 8>{});
    }
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
    if (steps <= 4) {
        const bool four = channels % 4 == 0 && aligned16({gate, value, state0, out, dout, dstate, dgate, dvalue, dstate0});
        auto launch     = [&](auto kernel, int v) -> ct_status {
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)((chains / v + 127) / 128)), dim3(128), 0, stream(), gate, value, state0, lengths, out, dout, dstate,
                                     chains, (int)steps, (int)channels, dgate, dvalue, dstate0));
            CT_LAUNCH_CHECK("gated_steps_grad");
            return CT_OK;
        };
        if (steps <= 1)
            return four ? launch(gated_steps_grad_kernel<4, 1>, 4) : launch(gated_steps_grad_kernel<1, 1>, 1);
        return four ? launch(gated_steps_grad_kernel<4, 4>, 4) : launch(gated_steps_grad_kernel<1, 4>, 1);
    }
    const Source from = scan_source(batch, steps, channels, aligned16({gate, value, out, dout}));
    auto launch       = [&](auto warps) -> ct_status {
        constexpr int W = decltype(warps)::value;
        switch (from) {
        case TILES:
            if constexpr (W == 8) // (see Pieces)
                if (scan_groups(from, batch, channels) * 6 > st->sm_count)
                    return launch_scan_grad<W, TILES, 1>(st, gate, value, state0, lengths, out, dout, dstate, batch, steps, channels, dgate, dvalue, dstate0);
            return launch_scan_grad<W, TILES, W == 2 ? 1 : 2>(st, gate, value, state0, lengths, out, dout, dstate, batch, steps, channels, dgate, dvalue, dstate0);
        case ROWS:
            return launch_scan_grad<W, ROWS, 1>(st, gate, value, state0, lengths, out, dout, dstate, batch, steps, channels, dgate, dvalue, dstate0);
        default:
            return launch_scan_grad<W, SINGLE, 1>(st, gate, value, state0, lengths, out, dout, dstate, batch, steps, channels, dgate, dvalue, dstate0);
        }
    };
    switch (scan_warps(st, scan_groups(from, batch, channels), steps)) {
    case 2:
        return launch(std::integral_constant<int, 2>{});
    case 4:
        return launch(std::integral_constant<int, 4>{});
    default:
        return launch(std::integral_constant<int, 8>{});
    }
}

} // extern "C"
