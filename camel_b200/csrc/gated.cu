// Gated dense layer: out = gate(x . w_gate + b_gate) * (x . w_up + b_up), and its gradient.
//
// Forward: one product whose tiles have the same columns of both weight matrices (fused_product.cuh); a thread of the epilogue
// has both sums of an output and stores what the layer gives.  Up to 8 or 16 rows (takes_few_rows): few_rows.cu; up to 128: stream_product.cuh (takes_stream).
// Gradient: gated_slope_planes_kernel turns dout and what was kept into the planes of d = [dg | du], scaled by row; they are the left operand of
// dx = d . [w_gate | w_up]^T as they lie, and the right operand of dw = x'^T . d with their rows as k, x' being x with the rows' scales
// taken back.  So d is written once, 8 bytes for each of its values' pairs of terms, and read in place.
// Up to 16 rows: few_rows_grad.cuh.  The reduced precision runs the library's products one after the other.
#include "few_rows_grad.cuh"
#include "gate.cuh"
#include "stream_product.cuh"

#include <algorithm>
#include <type_traits>

namespace ct {
namespace {

// out = gate(g) * u
template <int GATE>
__global__ void __launch_bounds__(256) gated_product_kernel(const float *g, const float *u, int64_t count, float *out) {
    griddep_wait();
    griddep_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        out[i] = __fmul_rn(gate_value<GATE>(g[i]), u[i]);
}

// dg and du
template <int GATE>
__global__ void __launch_bounds__(256) gated_slopes_kernel(
    const float *__restrict__ g, const float *__restrict__ u, const float *__restrict__ dout, int64_t count, float *__restrict__ dg,
    float *__restrict__ du) {
    griddep_wait();
    griddep_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        float value, slope;
        gate_slope<GATE>(g[i], value, slope);
        dg[i] = __fmul_rn(__fmul_rn(dout[i], u[i]), slope);
        du[i] = __fmul_rn(dout[i], value);
    }
}

// ---- one product with the gate behind it ----

template <int GATE> struct GateEpilogue {
    static constexpr bool kTwin = true;
    struct Params {
        const float *b_gate, *b_up;
        float *out, *gate_pre, *up_pre;
        int vec;
    };
    template <int COLS>
    __device__ static __forceinline__ void store(
        const fused::Product &p, const Params &e, float (&acc)[COLS], int64_t row0, int lane, int64_t col0, int, int, uint8_t *stage) {
        const int64_t left = p.m - row0;
        const int rows     = left < 0 ? 0 : (left < 32 ? (int)left : 32);
        if (rows == 0)
            return;
        const float rs = lane < rows ? __ldg(p.row_scale + row0 + lane) : 0.0f;
#pragma unroll
        for (int g = 0; g < COLS / 32; ++g) {
            const int64_t col = col0 + g * 16;
            if (col >= p.n)
                break;
            const int cols = (int)(p.n - col < 16 ? p.n - col : 16);
            float *a = acc + g * 16, *b = acc + COLS / 2 + g * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 s = fused::scales4(p.col_scale, col + 4 * j), t = fused::scales4(p.col_scale, p.twin_offset + col + 4 * j);
                a[4 * j] = __fmul_rn(a[4 * j], fused::weight(rs, s.x)), a[4 * j + 1] = __fmul_rn(a[4 * j + 1], fused::weight(rs, s.y));
                a[4 * j + 2] = __fmul_rn(a[4 * j + 2], fused::weight(rs, s.z)), a[4 * j + 3] = __fmul_rn(a[4 * j + 3], fused::weight(rs, s.w));
                b[4 * j] = __fmul_rn(b[4 * j], fused::weight(rs, t.x)), b[4 * j + 1] = __fmul_rn(b[4 * j + 1], fused::weight(rs, t.y));
                b[4 * j + 2] = __fmul_rn(b[4 * j + 2], fused::weight(rs, t.z)), b[4 * j + 3] = __fmul_rn(b[4 * j + 3], fused::weight(rs, t.w));
            }
            if (e.b_gate)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    a[j] = __fadd_rn(a[j], j < cols ? __ldg(e.b_gate + col + j) : 0.0f);
            if (e.b_up)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    b[j] = __fadd_rn(b[j], j < cols ? __ldg(e.b_up + col + j) : 0.0f);
            const int64_t at = row0 * p.n + col;
            if (e.gate_pre)
                fused::store_block<false>(e.gate_pre + at, p.n, rows, 0, cols, e.vec != 0, stage, lane, [&](int j) { return a[j]; });
            if (e.up_pre)
                fused::store_block<false>(e.up_pre + at, p.n, rows, 0, cols, e.vec != 0, stage, lane, [&](int j) { return b[j]; });
            fused::store_block<false>(
                e.out + at, p.n, rows, 0, cols, e.vec != 0, stage, lane, [&](int j) { return __fmul_rn(gate_value<GATE>(a[j]), b[j]); });
        }
    }
};

// Streamed: a warp has a row of a tile's results at a time.
template <int GATE> struct GateStream {
    static constexpr bool kTwin = true;
    struct Params {
        const float *b_gate, *b_up;
        float *out, *gate_pre, *up_pre;
    };
    struct State {};
    __device__ static __forceinline__ void init(State &) {}
    template <int Q>
    __device__ static __forceinline__ void tile(const fused::Stream &p, const Params &e, State &, const float *z, int64_t c0, int cols, int t) {
        const int lane = t & 31, rows = p.m - 16 * Q < 16 ? p.m - 16 * Q : 16;
        for (int i = t >> 5; i < rows; i += fused::kStreamDrain) {
            const int r    = 16 * Q + i;
            const float rs = p.row_scale[r] * fused::kStreamUp;
#pragma unroll
            for (int c = lane; c < 64; c += 32)
                if (c < cols) {
                    float g = __fmul_rn(z[i * fused::kStreamPitch + c], rs), u = __fmul_rn(z[i * fused::kStreamPitch + 64 + c], rs);
                    const int64_t at = r * p.n + c0 + c;
                    if (e.b_gate)
                        g = __fadd_rn(g, __ldg(e.b_gate + c0 + c));
                    if (e.b_up)
                        u = __fadd_rn(u, __ldg(e.b_up + c0 + c));
                    if (e.gate_pre)
                        e.gate_pre[at] = g;
                    if (e.up_pre)
                        e.up_pre[at] = u;
                    e.out[at] = __fmul_rn(gate_value<GATE>(g), u);
                }
        }
    }
    __device__ static __forceinline__ void finish(const fused::Stream &, const Params &, State &, float *, int) {}
};

ct_status gated_stream(
    DeviceState *st, const float *x, const float *w_gate, const float *b_gate, const float *w_up, const float *b_up, int64_t m, int64_t k, int64_t n,
    int gate, float *out, float *gate_pre, float *up_pre) {
    using namespace fused;
    const int64_t lk = padded(k);
    Parts parts;
    const size_t xp = parts.planes(m, lk), xi = parts.take((size_t)m * 4);
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    const Planes px     = planes_at(s, xp, m, lk, lk);
    const Split operand = {x, nullptr, m, k, false, nullptr, px, s.as<float>(xi)};
    CT_TRY(split(st, &operand, 1));
    Stream p{};
    p.w = w_gate, p.w2 = w_up, p.k = k, p.n = p.ld = n, p.row_scale = s.as<float>(xi);
    return with_gate(gate, [&](auto G) -> ct_status {
        using E = GateStream<G.value>;
        const typename E::Params e{b_gate, b_up, out, gate_pre, up_pre};
        return launch_stream<E>(st, px, p, e, "dense_gated", [&](typename E::Params f, int64_t r) {
            f.out += r * n, f.gate_pre = f.gate_pre ? f.gate_pre + r * n : nullptr, f.up_pre = f.up_pre ? f.up_pre + r * n : nullptr;
            return f;
        });
    });
}

bool whole(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

ct_status gated_fused(
    DeviceState *st, const float *x, const float *w_gate, const float *b_gate, const float *w_up, const float *b_up, int64_t m, int64_t k, int64_t n,
    int gate, float *out, float *gate_pre, float *up_pre) {
    using namespace fused;
    const int64_t lk = padded(k), ln = padded(n);
    Parts parts;
    const size_t xp = parts.planes(m, lk), xi = parts.take((size_t)m * 4), wp = parts.planes(k, 2 * ln), wi = parts.take((size_t)scales(2 * ln) * 4);
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    const Planes px = planes_at(s, xp, m, lk, lk), pw = planes_at(s, wp, k, 2 * ln, 2 * ln);
    const Split operands[2] = {{w_gate, w_up, k, n, true, nullptr, pw, s.as<float>(wi)}, {x, nullptr, m, k, false, nullptr, px, s.as<float>(xi)}};
    CT_TRY(split(st, operands, 2));
    Product p{};
    p.m = m, p.n = n, p.twin_offset = (int)ln, p.row_scale = s.as<float>(xi), p.col_scale = s.as<float>(wi);
    return with_gate(gate, [&](auto G) -> ct_status {
        using E = GateEpilogue<G.value>;
        typename E::Params e{b_gate, b_up, out, gate_pre, up_pre, (n & 3) == 0 && whole(out) && whole(gate_pre) && whole(up_pre) ? 1 : 0};
        return takes_pairs(st, m, 2 * n) ? launch<E, 256, 2, false, true>(st, px, pw, p, e, 1, "dense_gated")
                                                    : launch<E, 128, 1, false, true>(st, px, pw, p, e, 1, "dense_gated");
    });
}

// ---- the gradient's left operand ----

// d = [dg | du] of a row, its largest magnitude, and its planes: TPR threads to a row, which hold V groups of four columns of both; longer
// rows are computed twice.  inverse[row] is zero for a row of zeros: such a row must not widen the range of x' (gated_grad_fused), where only
// what is no number is left of it.
// BIAS: a thread also sums its columns over the rows that it has, in float32, into partial[which of the grid's rows at a time][2][n] - of the
// values themselves, since what the planes hold of a value depends on the rest of its row.  By a kernel that computes the slopes again
// 1537 x 2050 took 17 us more.
template <int GATE, int TPR, int V, bool BIAS>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) gated_slope_planes_kernel(
    const float *__restrict__ g, const float *__restrict__ u, const float *__restrict__ dout, int64_t rows, int64_t n, int vec, const fused::Planes to,
    float *__restrict__ inverse, double *__restrict__ partial) {
    __shared__ uint32_t words[2][32];
    griddep_wait();
    griddep_launch_dependents();
    constexpr int RPB = (TPR < 256 ? 256 : TPR) / TPR;
    const int t = threadIdx.x % TPR;
    const int64_t row0 = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR, ld = to.ld / 2;
    auto load = [&](const float *src, int64_t row, int64_t c) {
        src += row * n + c;
        if (vec && c + 3 < n)
            return __ldcs(reinterpret_cast<const float4 *>(src));
        float4 q;
        q.x = c < n ? src[0] : 0.0f, q.y = c + 1 < n ? src[1] : 0.0f;
        q.z = c + 2 < n ? src[2] : 0.0f, q.w = c + 3 < n ? src[3] : 0.0f;
        return q;
    };
    auto slopes = [&](int64_t row, int64_t c, float4 &dg, float4 &du) {
        const float4 a = load(g, row, c), b = load(u, row, c), d = load(dout, row, c);
        auto one = [](float a, float b, float d, float &dg, float &du) {
            float value, slope;
            gate_slope<GATE>(a, value, slope);
            dg = __fmul_rn(__fmul_rn(d, b), slope), du = __fmul_rn(d, value);
        };
        one(a.x, b.x, d.x, dg.x, du.x), one(a.y, b.y, d.y, dg.y, du.y), one(a.z, b.z, d.z, dg.z, du.z), one(a.w, b.w, d.w, dg.w, du.w);
    };
    auto bits = [](const float4 &q) {
        return max(max(fused::finite_bits(q.x), fused::finite_bits(q.y)), max(fused::finite_bits(q.z), fused::finite_bits(q.w)));
    };
    const bool fits = ld <= TPR * V * 4;
    float sum_g[BIAS ? 4 * V : 1] = {}, sum_u[BIAS ? 4 * V : 1] = {};
    int turn = 0;
    for (int64_t row = row0; row < rows; row += (int64_t)gridDim.x * RPB, turn ^= 1) { // whole warps, or the whole block
        float4 dg[V], du[V];
        uint32_t mx = 0;
        if (fits) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t c = (int64_t)(j * TPR + t) * 4;
                dg[j] = du[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c < n)
                    slopes(row, c, dg[j], du[j]);
                mx = max(mx, max(bits(dg[j]), bits(du[j])));
                if (BIAS) {
                    sum_g[4 * j] = __fadd_rn(sum_g[4 * j], dg[j].x), sum_g[4 * j + 1] = __fadd_rn(sum_g[4 * j + 1], dg[j].y);
                    sum_g[4 * j + 2] = __fadd_rn(sum_g[4 * j + 2], dg[j].z), sum_g[4 * j + 3] = __fadd_rn(sum_g[4 * j + 3], dg[j].w);
                    sum_u[4 * j] = __fadd_rn(sum_u[4 * j], du[j].x), sum_u[4 * j + 1] = __fadd_rn(sum_u[4 * j + 1], du[j].y);
                    sum_u[4 * j + 2] = __fadd_rn(sum_u[4 * j + 2], du[j].z), sum_u[4 * j + 3] = __fadd_rn(sum_u[4 * j + 3], du[j].w);
                }
            }
        } else {
            for (int64_t c = t * 4; c < n; c += TPR * 4) {
                slopes(row, c, dg[0], du[0]);
                mx = max(mx, max(bits(dg[0]), bits(du[0])));
            }
        }
        mx = __reduce_max_sync(0xffffffffu, mx);
        if (TPR > 32) {
            if ((threadIdx.x & 31) == 0)
                words[turn][threadIdx.x >> 5] = mx;
            __syncthreads();
            mx = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < TPR / 32 ? words[turn][threadIdx.x & 31] : 0u);
        }
        const float s = fused::line_scale(mx);
        auto put      = [&](int64_t c, const float4 &q) {
            __half2 hi[2], lo[2];
            fused::split2(q.x * s, q.y * s, hi[0], lo[0]);
            fused::split2(q.z * s, q.w * s, hi[1], lo[1]);
            *reinterpret_cast<uint2 *>(to.hi + row * to.ld + c) = *reinterpret_cast<uint2 *>(hi);
            *reinterpret_cast<uint2 *>(to.lo + row * to.ld + c) = *reinterpret_cast<uint2 *>(lo);
        };
        if (fits) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t c = (int64_t)(j * TPR + t) * 4;
                if (c < ld)
                    put(c, dg[j]), put(ld + c, du[j]);
            }
        } else {
            for (int64_t c = t * 4; c < ld; c += TPR * 4) {
                dg[0] = du[0] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c < n)
                    slopes(row, c, dg[0], du[0]);
                put(c, dg[0]), put(ld + c, du[0]);
            }
        }
        if (t == 0)
            inverse[row] = mx ? fused::line_inverse(mx) : 0.0f;
    }
    if (BIAS) {
        double *mine = partial + row0 * 2 * n; // row0 counts the rows that the grid has at a time
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t c = (int64_t)(j * TPR + t) * 4 + q;
                if (c < n)
                    mine[c] = (double)sum_g[4 * j + q], mine[n + c] = (double)sum_u[4 * j + q];
            }
    }
}

// The columns' sums of dg and du where rows are too long for the kernel above to keep theirs (kSlopesFit).  A lane has four columns, a warp
// every eighth row of the block's; partial[block][2][n] are added up by join_columns.
template <int GATE>
__global__ void __launch_bounds__(256) gated_bias_kernel(
    const float *__restrict__ g, const float *__restrict__ u, const float *__restrict__ dout, int64_t rows, int64_t n, int vec, int64_t rows_each,
    double *__restrict__ partial, float *__restrict__ db_gate, float *__restrict__ db_up) {
    __shared__ float sums[8][2][128];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c  = (int64_t)blockIdx.x * 128 + lane * 4;
    const int64_t r0 = (int64_t)blockIdx.y * rows_each, r1 = min(rows, r0 + rows_each);
    float sg[4] = {}, su[4] = {};
    auto load = [&](const float *src, int64_t r) {
        src += r * n + c;
        if (vec && c + 3 < n)
            return *reinterpret_cast<const float4 *>(src);
        float4 q;
        q.x = c < n ? src[0] : 0.0f, q.y = c + 1 < n ? src[1] : 0.0f;
        q.z = c + 2 < n ? src[2] : 0.0f, q.w = c + 3 < n ? src[3] : 0.0f;
        return q;
    };
    if (c < n)
#pragma unroll 4
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            const float4 a = load(g, r), b = load(u, r), d = load(dout, r);
            auto one = [&](float a, float b, float d, int q) {
                float value, slope;
                gate_slope<GATE>(a, value, slope);
                sg[q] = __fmaf_rn(__fmul_rn(d, b), slope, sg[q]);
                su[q] = __fmaf_rn(d, value, su[q]);
            };
            one(a.x, b.x, d.x, 0), one(a.y, b.y, d.y, 1), one(a.z, b.z, d.z, 2), one(a.w, b.w, d.w, 3);
        }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        sums[warp][0][lane * 4 + q] = sg[q], sums[warp][1][lane * 4 + q] = su[q];
    __syncthreads();
    const int which = threadIdx.x >> 7, at = threadIdx.x & 127;
    const int64_t mine = (int64_t)blockIdx.x * 128 + at;
    if (mine < n) {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < 8; ++w)
            all += (double)sums[w][which][at];
        float *to = which ? db_up : db_gate;
        if (partial)
            partial[((int64_t)blockIdx.y * 2 + which) * n + mine] = all;
        else if (to)
            to[mine] = (float)all;
    }
}

ct_status gated_bias(
    DeviceState *st, const float *g, const float *u, const float *dout, int64_t m, int64_t n, int gate, int vec, float *db_gate, float *db_up) {
    const int64_t strips = (n + 127) / 128;
    const int64_t slices = fused::row_slices(st, m, strips);
    const int64_t each = (m + slices - 1) / slices, parts = (m + each - 1) / each;
    Scratch partial; // of one part there is nothing to add up
    if (parts > 1)
        CT_TRY(partial.get((size_t)(parts * 2 * n) * 8));
    CT_TRY(with_gate(gate, [&](auto G) -> ct_status {
        CT_CUDA(launch_dependent(gated_bias_kernel<G.value>, dim3((unsigned)strips, (unsigned)parts), dim3(256), 0, stream(), g, u, dout, m, n, vec, each,
                                 parts > 1 ? partial.as<double>() : nullptr, db_gate, db_up));
        CT_LAUNCH_CHECK("gated_bias");
        return CT_OK;
    }));
    if (parts == 1)
        return CT_OK;
    return fused::join_columns(partial.as<const double>(), parts, n, 2 * n, db_gate, db_up);
}

constexpr int64_t kSlopesFit = 512 * 4 * 4; // columns

template <int GATE, int TPR, int V>
ct_status launch_slopes_of(
    const DeviceState *st, const float *g, const float *u, const float *dout, int64_t m, int64_t n, int vec, const fused::Planes &to, float *inverse,
    float *db_gate, float *db_up) {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    int64_t blocks    = (m + RPB - 1) / RPB;
    if (!db_gate && !db_up) {
        CT_CUDA(launch_dependent(gated_slope_planes_kernel<GATE, TPR, V, false>, dim3((unsigned)blocks), dim3(TPR * RPB), 0, stream(), g, u, dout, m, n, vec,
                                 to, inverse, (double *)nullptr));
        CT_LAUNCH_CHECK("gated_slopes");
        return CT_OK;
    }
    blocks = blocks_for(blocks, (int64_t)st->sm_count * (TPR <= 256 ? 4 : 2), 256); // rows of a thread's sums
    Scratch partial;
    CT_TRY(partial.get((size_t)(blocks * RPB * 2 * n) * 8));
    CT_CUDA(launch_dependent(gated_slope_planes_kernel<GATE, TPR, V, true>, dim3((unsigned)blocks), dim3(TPR * RPB), 0, stream(), g, u, dout, m, n, vec, to,
                             inverse, partial.as<double>()));
    CT_LAUNCH_CHECK("gated_slopes");
    return fused::join_columns(partial.as<const double>(), blocks * RPB, n, 2 * n, db_gate, db_up);
}
template <int GATE>
ct_status launch_slopes(
    const DeviceState *st, const float *g, const float *u, const float *dout, int64_t m, int64_t n, int vec, const fused::Planes &to, float *inverse,
    float *db_gate, float *db_up) {
    // As gated gradients (us): 128 columns with biases a warp to a row 131, 256 threads 211 (60000 rows x 64), 55 and 48 (4096 rows x 8), without 38 and 42;
    // 256 columns 197 and 251, 67 and 53, 42 and 46; then of 4096 rows x 8 with biases, 1000 columns 256 threads 68, 512 73; 2048 100 and 98; 4096
    // 201 and 175; 6144 columns 3 float4 to a thread 262, 4 265; 40 rows take 17 to 26 in each form
    if (n <= 128)
        return launch_slopes_of<GATE, 32, 1>(st, g, u, dout, m, n, vec, to, inverse, db_gate, db_up);
    if (n <= 256)
        return launch_slopes_of<GATE, 32, 2>(st, g, u, dout, m, n, vec, to, inverse, db_gate, db_up);
    if (n <= 1024)
        return launch_slopes_of<GATE, 256, 1>(st, g, u, dout, m, n, vec, to, inverse, db_gate, db_up);
    if (n <= 2048)
        return launch_slopes_of<GATE, 256, 2>(st, g, u, dout, m, n, vec, to, inverse, db_gate, db_up);
    if (n <= 4096)
        return launch_slopes_of<GATE, 512, 2>(st, g, u, dout, m, n, vec, to, inverse, db_gate, db_up);
    if (n <= 6144)
        return launch_slopes_of<GATE, 512, 3>(st, g, u, dout, m, n, vec, to, inverse, db_gate, db_up);
    return launch_slopes_of<GATE, 512, 4>(st, g, u, dout, m, n, vec, to, inverse, n <= kSlopesFit ? db_gate : nullptr, n <= kSlopesFit ? db_up : nullptr);
}

ct_status gated_grad_fused(
    DeviceState *st, const float *x, const float *w_gate, const float *w_up, const float *gate_pre, const float *up_pre, const float *dout, int64_t m,
    int64_t k, int64_t n, int gate, float *dx, float *dw_gate, float *dw_up, float *db_gate, float *db_up) {
    using namespace fused;
    const int64_t lk = padded(k), ln = padded(n);
    const bool weights = (dw_gate || dw_up) && k > 0, back = dx && k > 0;
    Parts parts;
    const size_t dp = parts.planes(m, 2 * ln), di = parts.take((size_t)m * 4);
    const size_t wp = back ? parts.planes(k, 2 * ln) : 0, wi = back ? parts.take((size_t)scales(k) * 4) : 0;
    const size_t xp = weights ? parts.planes(m, lk) : 0, xi = weights ? parts.take((size_t)scales(lk) * 4) : 0;
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    const Planes pd = planes_at(s, dp, m, 2 * ln, 2 * ln);
    const int vec   = (n & 3) == 0 && whole(gate_pre) && whole(up_pre) && whole(dout) ? 1 : 0;
    CT_TRY(with_gate(gate, [&](auto G) { return launch_slopes<G.value>(st, gate_pre, up_pre, dout, m, n, vec, pd, s.as<float>(di), db_gate, db_up); }));
    if (n > kSlopesFit && (db_gate || db_up))
        CT_TRY(gated_bias(st, gate_pre, up_pre, dout, m, n, gate, vec, db_gate, db_up));
    const Planes pw = planes_at(s, wp, k, 2 * ln, 2 * ln), px = planes_at(s, xp, m, lk, lk);
    Split operands[2];
    int count = 0;
    if (back)
        operands[count++] = {w_gate, w_up, k, n, false, nullptr, pw, s.as<float>(wi)};
    if (weights)
        operands[count++] = {x, nullptr, m, k, true, s.as<float>(di), px, s.as<float>(xi)};
    CT_TRY(split(st, operands, count));
    Wanted wanted[2];
    count = 0;
    if (back) {
        Result r{dx};
        r.cols = r.stride = k;
        wanted[count++] = {pd, pw, false, m, k, s.as<float>(di), s.as<float>(wi), r};
    }
    if (weights) {
        Result r{dw_gate ? dw_gate : dw_up};
        r.cols = r.stride = n;
        if (dw_gate && dw_up)
            r.out2 = dw_up, r.second = ln;
        const Planes right = dw_gate && dw_up ? pd : columns_of(pd, dw_gate ? 0 : ln, n);
        wanted[count++]    = {px, right, true, k, dw_gate && dw_up ? 2 * ln : n, s.as<float>(xi), nullptr, r};
    }
    return count ? products(st, wanted, count) : CT_OK;
}

// Few rows: dg or du of what was kept.
template <int GATE> struct FewGateSlopes {
    static constexpr int kMatrices = 2;
    const float *g, *u, *dout;
    int64_t n;
    __device__ __forceinline__ bool has(int) const { return true; }
    __device__ __forceinline__ float at(int which, int r, int64_t c) const {
        const int64_t i = r * n + c;
        float value, slope;
        gate_slope<GATE>(g[i], value, slope);
        return which ? __fmul_rn(dout[i], value) : __fmul_rn(__fmul_rn(dout[i], u[i]), slope);
    }
};

unsigned grid_of(const DeviceState *st, int64_t count) {
    return (unsigned)std::min<int64_t>((count + 255) / 256, (int64_t)st->sm_count * 16);
}

ct_status check_gated(const char *name, int64_t m, int64_t k, int64_t n, int gate) {
    if (m < 0 || k < 0 || n < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (!valid_gate(gate))
        return fail(CT_ERR_INVALID, "%s: unknown gate", name);
    if (m > fused::kMostSize || k > fused::kMostSize || n > fused::kMostSize)
        return fail(CT_ERR_TOO_LARGE, "%s: dimension too large", name);
    return CT_OK;
}

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_dense_gated(
    const float *x, const float *w_gate, const float *b_gate, const float *w_up, const float *b_up, int64_t m, int64_t k, int64_t n, ct_gate gate,
    float *out, float *gate_pre, float *up_pre) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_gated("dense_gated", m, k, n, gate));
    if (m == 0 || n == 0)
        return CT_OK;
    if (!out || (k > 0 && (!x || !w_gate || !w_up)))
        return fail(CT_ERR_INVALID, "dense_gated: null pointer");
    ProfScope prof("dense_gated");
    if (ct_get_precision() == CT_PREC_3XTF32 && k > 0) {
        if (fused::takes_few_rows(m, 2 * n))
            return fused::few_rows(st, x, w_gate, b_gate, w_up, b_up, m, k, n, gate, out, gate_pre, up_pre);
        if (fused::takes_stream(m, k, 2 * n))
            return gated_stream(st, x, w_gate, b_gate, w_up, b_up, m, k, n, gate, out, gate_pre, up_pre);
        return gated_fused(st, x, w_gate, b_gate, w_up, b_up, m, k, n, gate, out, gate_pre, up_pre);
    }
    const int64_t count = m * n;
    Scratch scratch;
    float *g = gate_pre, *u = up_pre;
    if (!g || !u) {
        CT_TRY(scratch.get((size_t)count * 8));
        g = g ? g : scratch.as<float>();
        u = u ? u : scratch.as<float>((size_t)count * 4);
    }
    CT_TRY(ct_dense(x, w_gate, b_gate, m, k, n, CT_ACT_NONE, g, nullptr));
    CT_TRY(ct_dense(x, w_up, b_up, m, k, n, CT_ACT_NONE, u, nullptr));
    return with_gate(gate, [&](auto G) -> ct_status {
        CT_CUDA(launch_dependent(gated_product_kernel<G.value>, dim3(grid_of(st, count)), dim3(256), 0, stream(), (const float *)g, (const float *)u, count,
                                 out));
        CT_LAUNCH_CHECK("gated_product");
        return CT_OK;
    });
}

ct_status ct_dense_gated_grad(
    const float *x, const float *w_gate, const float *w_up, const float *gate_pre, const float *up_pre, const float *dout, int64_t m, int64_t k,
    int64_t n, ct_gate gate, float *dx, float *dw_gate, float *dw_up, float *db_gate, float *db_up) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_gated("dense_gated_grad", m, k, n, gate));
    if (m > 0 && n > 0 && (!gate_pre || !up_pre || !dout))
        return fail(CT_ERR_INVALID, "dense_gated_grad: null pointer");
    if (m > 0 && n > 0 && k > 0 && ((dx && (!w_gate || !w_up)) || ((dw_gate || dw_up) && !x)))
        return fail(CT_ERR_INVALID, "dense_gated_grad: null pointer");
    ProfScope prof("dense_gated_grad");
    if (m == 0 || n == 0) { // sums of nothing
        auto clear = [&](float *p, int64_t count) {
            return p && count > 0 ? cudaMemsetAsync(p, 0, (size_t)count * 4, stream()) : cudaSuccess;
        };
        CT_CUDA(clear(dx, m * k));
        CT_CUDA(clear(dw_gate, k * n));
        CT_CUDA(clear(dw_up, k * n));
        CT_CUDA(clear(db_gate, n));
        CT_CUDA(clear(db_up, n));
        return CT_OK;
    }
    if (ct_get_precision() == CT_PREC_3XTF32 && m <= fused::kFewRows && k > 0 && (dx || dw_gate || dw_up || db_gate || db_up)) {
        fused::FewGrad p{};
        p.x = x, p.w[0] = w_gate, p.w[1] = w_up, p.dw[0] = dw_gate, p.dw[1] = dw_up, p.db[0] = db_gate, p.db[1] = db_up;
        p.dx = dx, p.k = k, p.n = n, p.m = (int)m;
        return with_gate(gate, [&](auto G) { return fused::few_rows_grad(st, p, FewGateSlopes<G.value>{gate_pre, up_pre, dout, n}); });
    }
    if (ct_get_precision() == CT_PREC_3XTF32)
        return gated_grad_fused(st, x, w_gate, w_up, gate_pre, up_pre, dout, m, k, n, gate, dx, dw_gate, dw_up, db_gate, db_up);
    const int64_t count = m * n;
    Scratch slopes;
    CT_TRY(slopes.get((size_t)count * 8));
    float *dg = slopes.as<float>(), *du = dg + count;
    CT_TRY(with_gate(gate, [&](auto G) -> ct_status {
        CT_CUDA(launch_dependent(gated_slopes_kernel<G.value>, dim3(grid_of(st, count)), dim3(256), 0, stream(), gate_pre, up_pre, dout, count, dg, du));
        CT_LAUNCH_CHECK("gated_slopes");
        return CT_OK;
    }));
    if (k > 0 && dw_gate)
        CT_TRY(ct_matmul_tn(x, dg, k, m, n, dw_gate));
    if (k > 0 && dw_up)
        CT_TRY(ct_matmul_tn(x, du, k, m, n, dw_up));
    if (db_gate)
        CT_TRY(ct_sum_axis(CT_F32, dg, m, n, 0, db_gate));
    if (db_up)
        CT_TRY(ct_sum_axis(CT_F32, du, m, n, 0, db_up));
    if (k > 0 && dx) {
        Scratch turned;
        CT_TRY(turned.get((size_t)(k * n + m * k) * 4));
        float *wt = turned.as<float>(), *part = wt + k * n;
        CT_TRY(ct_transpose(CT_F32, w_gate, k, n, wt));
        CT_TRY(ct_matmul(CT_F32, dg, CT_F32, wt, m, n, k, part));
        CT_TRY(ct_transpose(CT_F32, w_up, k, n, wt));
        CT_TRY(ct_matmul(CT_F32, du, CT_F32, wt, m, n, k, dx));
        CT_TRY(ct_binary(CT_ADD, CT_F32, part, CT_F32, dx, (uint64_t)(m * k), dx));
    }
    return CT_OK;
}

} // extern "C"
