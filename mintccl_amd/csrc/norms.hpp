// What stands before and after a block of a model: the norm of its input, and its output taken into the residual stream.
//
//   N(x) = (x - m) q w + b      rms: m = 0, q = 1 / sqrt(mean x^2 + eps)      layer: m = mean x, q = 1 / sqrt(mean (x - m)^2 + eps)
//   u = N_after(y), or y        r = carry s + scale a(g) u                     h = N_before(r as it is stored)
//
// s the stream, y the block's output, g a gate by channel, by row or for every number, a none or an activation; r the new stream, h the next
// block's input.  Without y only h = N_before(s) is made.  The gradients, with xh = (x - m) q and d' = w d:
//
//   N^T d = q (d' - xh mean(d' xh) [- mean d'])     d_w = sum over rows of d xh     d_b = sum over rows of d
//   D = d_r + N_before^T d_h     d_s = carry D     G = scale D     d_y = N_after^T(a(g) G)     d_g = a'(g) G u, summed over what g is shared by
//
// With a gate by channel the sums over rows of G xh and of G give all three: d_w = a(g) sum G xh, d_b = a(g) sum G and
// d_g = a'(g) (w sum G xh + b sum G).  Statistics and sums are in 32 bits and have a fixed order.
#pragma once
#include "activations.hpp"

#include <algorithm>

namespace mint {

constexpr int V = 8;                            // consecutive numbers of a lane

struct NormArgs {
    const void *weight, *bias;                  // 0: ones, zeros
    int kind, dtype;
    float eps;
};
struct JoinArgs {
    const void *stream, *y, *gate;
    void *new_stream, *next;
    int64_t stream_stride, y_stride, gate_row, new_stride, next_stride;
    NormArgs after, before;
    float scale, carry;
    uint32_t rows, width;
    int gate_dtype, gate_by, gate_form;
};

// N numbers of a vector whose type is known only here (the branch is the same for all)
template <int N>
__device__ __forceinline__ void load_any(const void* p, int dtype, int64_t at, int64_t left, float (&v)[N]) {
    if (dtype == MINT_F32) load_elements<DT_F32, N>(static_cast<const float*>(p) + at, left, v);
    else if (dtype == MINT_BF16) load_elements<DT_BF16, N>(static_cast<const __bf16*>(p) + at, left, v);
    else load_elements<DT_F16, N>(static_cast<const _Float16*>(p) + at, left, v);
}
__device__ __forceinline__ float load_one(const void* p, int dtype, int64_t at) {
    if (dtype == MINT_F32) return *as_global(static_cast<const float*>(p) + at);
    if (dtype == MINT_BF16) return (float)*as_global(static_cast<const __bf16*>(p) + at);
    return (float)*as_global(static_cast<const _Float16*>(p) + at);
}
__device__ __forceinline__ void store_one(void* p, int dtype, int64_t at, float v) {
    if (dtype == MINT_F32) *as_global(static_cast<float*>(p) + at) = v;
    else if (dtype == MINT_BF16) *as_global(static_cast<__bf16*>(p) + at) = (__bf16)v;
    else *as_global(static_cast<_Float16*>(p) + at) = (_Float16)v;
}
template <int N>
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t at, int64_t left, const float (&v)[N]) {
    if (dtype == MINT_F32) store_elements<DT_F32, N>(static_cast<float*>(p) + at, left, v);
    else if (dtype == MINT_BF16) store_elements<DT_BF16, N>(static_cast<__bf16*>(p) + at, left, v);
    else store_elements<DT_F16, N>(static_cast<_Float16*>(p) + at, left, v);
}

// Sums over the WAVES wavefronts that have a row, K at a time, in their order.  Two halves of `slots` in turn: whoever writes one again
// has met all others behind their reads of it.
template <int WAVES, int K>
struct RowSums {
    float (*slots)[WAVES][K];
    uint32_t half = 0;
    template <int N>
    __device__ __forceinline__ void operator()(float (&v)[N]) {
        static_assert(N <= K, "they have room");
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
        if constexpr (WAVES > 1) {
            if (lane_id() == 0) {
#pragma unroll
                for (int k = 0; k < N; ++k) slots[half][wave_in_block()][k] = v[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int k = 0; k < N; ++k) v[k] += slots[half][w][k];
            half ^= 1u;
        }
    }
};

// Of a row in registers: C times V numbers of a lane, LANES lanes side by side.  What lies behind the row's end is zero, and stays.
template <int LANES, int C>
struct RowOf {
    uint32_t width, lane;
    __device__ __forceinline__ uint32_t at(int c) const { return ((uint32_t)c * LANES + lane) * V; }
    __device__ __forceinline__ int64_t left(int c) const { return (int64_t)width - at(c); }
    // takes the mean off, but not off what is not there
    __device__ __forceinline__ void centre(float (&x)[C][V], float mean) const {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) x[c][i] = i < left(c) ? x[c][i] - mean : 0.0f;
    }
    static __device__ __forceinline__ float sum(const float (&x)[C][V]) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) s += x[c][i];
        return s;
    }
    static __device__ __forceinline__ float dot(const float (&x)[C][V], const float (&y)[C][V]) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) s = fmaf(x[c][i], y[c][i], s);
        return s;
    }
};
// x becomes (x - m) q; q comes back
template <int LANES, int C, typename Sums>
__device__ __forceinline__ float normalise(const RowOf<LANES, C>& row, const NormArgs& n, float (&x)[C][V], Sums& sums) {
    const float share = 1.0f / (float)row.width;
    if (n.kind == MINT_NORM_LAYER) {
        float mean[1] = {row.sum(x)};
        sums(mean);
        row.centre(x, mean[0] * share);
    }
    float square[1] = {row.dot(x, x)};
    sums(square);
    const float q = 1.0f / sqrtf(fmaf(square[0], share, n.eps));
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) x[c][i] *= q;
    return q;
}
// the weight's (or bias's) numbers of chunk c
__device__ __forceinline__ void weight_of(const NormArgs& n, uint32_t at, int64_t left, float (&w)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 1.0f;
    if (n.weight) load_any(n.weight, n.dtype, at, left, w);
}
__device__ __forceinline__ void bias_of(const NormArgs& n, uint32_t at, int64_t left, float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = 0.0f;
    if (n.bias) load_any(n.bias, n.dtype, at, left, b);
}
// a row's gate for chunk c, as it was given (ones where there is none)
__device__ __forceinline__ void gate_of(const JoinArgs& a, uint64_t row, uint32_t at, int64_t left, float (&g)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = 1.0f;
    if (!a.gate) return;
    if (a.gate_form != MINT_GATE_ROW) {
        load_any(a.gate, a.gate_dtype, (int64_t)row * a.gate_row + at, left, g);
    } else {
        const float one = load_one(a.gate, a.gate_dtype, (int64_t)row * a.gate_row);
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = one;
    }
}

// S: the stream's type, T: that of y and of h.
template <int S, int T, int LANES, int C>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) join_kernel(JoinArgs a) {
    using TS = typename Elem<S>::type;
    using TT = typename Elem<T>::type;
    constexpr int WAVES = LANES / 64, ROWS = LANES < 256 ? 256 / LANES : 1;
    static_assert(WAVES == 1 || ROWS == 1, "wavefronts that meet have the same row");
    __shared__ float slots[2][WAVES][1];
    const uint64_t r = (uint64_t)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / LANES : 0u);
    if (r >= a.rows) return;
    const RowOf<LANES, C> row = {a.width, threadIdx.x % LANES};
    RowSums<WAVES, 1> sums = {slots};
    float s[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) load_elements<S, V>(static_cast<const TS*>(a.stream) + (int64_t)r * a.stream_stride + row.at(c), row.left(c), s[c]);
    if (a.y) {
        float y[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c) load_elements<T, V>(static_cast<const TT*>(a.y) + (int64_t)r * a.y_stride + row.at(c), row.left(c), y[c]);
        if (a.after.kind) normalise(row, a.after, y, sums);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (row.left(c) <= 0) continue;
            float w[V], b[V], g[V];
            weight_of(a.after, row.at(c), row.left(c), w);
            bias_of(a.after, row.at(c), row.left(c), b);
            gate_of(a, r, row.at(c), row.left(c), g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = fmaf(y[c][i], w[i], b[i]) * (a.gate ? gate_value(a.gate_by, g[i]) : 1.0f);
                // (as it is stored: what the next norm is of)
                s[c][i] = i < row.left(c) ? Elem<S>::load(Elem<S>::round(fmaf(a.scale, u, a.carry * s[c][i]))) : 0.0f;
            }
            store_elements<S, V>(static_cast<TS*>(a.new_stream) + (int64_t)r * a.new_stride + row.at(c), row.left(c), s[c]);
        }
    }
    if (!a.next) return;
    normalise(row, a.before, s, sums);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (row.left(c) <= 0) continue;
        float w[V], b[V];
        weight_of(a.before, row.at(c), row.left(c), w);
        bias_of(a.before, row.at(c), row.left(c), b);
#pragma unroll
        for (int i = 0; i < V; ++i) s[c][i] = fmaf(s[c][i], w[i], b[i]);
        store_elements<T, V>(static_cast<TT*>(a.next) + (int64_t)r * a.next_stride + row.at(c), row.left(c), s[c]);
    }
}

struct JoinGradArgs {
    JoinArgs f;                                 // stream: the new one; y, gate, norms
    const void *d_stream, *d_next;              // either may be 0
    void *to_stream, *to_y, *to_gate;
    int64_t d_stream_stride, d_next_stride, to_stream_stride, to_y_stride, to_gate_stride;
    float* sums;                                // (groups, SUMS, width): each group's sums over its rows
    uint32_t groups;
};
// Which of a group's sums over rows are where: before's weight, [its bias,] [after's weight, [its bias]].
template <bool BLOCK, bool BIAS>
constexpr int kSums = (BLOCK ? 2 : 1) * (BIAS ? 2 : 1);

// A group of LANES lanes has every groups-th row and keeps its sums over them in registers.
template <int S, int T, int LANES, int C, bool BLOCK, bool BIAS>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) join_grad_kernel(JoinGradArgs a) {
    using TS = typename Elem<S>::type;
    using TT = typename Elem<T>::type;
    constexpr int WAVES = LANES / 64, GROUPS = LANES < 256 ? 256 / LANES : 1, SUMS = kSums<BLOCK, BIAS>;
    __shared__ float slots[2][WAVES][3];
    const uint32_t group = blockIdx.x * GROUPS + (GROUPS > 1 ? threadIdx.x / LANES : 0u);
    if (group >= a.groups) return;
    const JoinArgs& f = a.f;
    const RowOf<LANES, C> row = {f.width, threadIdx.x % LANES};
    RowSums<WAVES, 3> sums = {slots};
    const float share = 1.0f / (float)f.width;
    const bool by_row = f.gate && f.gate_form == MINT_GATE_ROW, by_channel = f.gate && f.gate_form == MINT_GATE_CHANNEL;
    float total[SUMS][C][V];
#pragma unroll
    for (int k = 0; k < SUMS; ++k)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) total[k][c][i] = 0.0f;
    for (uint64_t r = group; r < f.rows; r += a.groups) {
        float x[C][V], d[C][V], y[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (a.d_next) {
                load_elements<S, V>(static_cast<const TS*>(f.stream) + (int64_t)r * f.stream_stride + row.at(c), row.left(c), x[c]);
                load_elements<T, V>(static_cast<const TT*>(a.d_next) + (int64_t)r * a.d_next_stride + row.at(c), row.left(c), d[c]);
            }
            if (BLOCK) load_elements<T, V>(static_cast<const TT*>(f.y) + (int64_t)r * f.y_stride + row.at(c), row.left(c), y[c]);
        }
        float q = 0.0f, mean[2] = {0.0f, 0.0f};
        if (a.d_next) {
            q = normalise(row, f.before, x, sums);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float w[V];
                weight_of(f.before, row.at(c), row.left(c), w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    total[0][c][i] = fmaf(d[c][i], x[c][i], total[0][c][i]);
                    if (BIAS) total[1][c][i] += d[c][i];
                    d[c][i] *= w[i];
                }
            }
            mean[0] = row.dot(d, x);
            mean[1] = row.sum(d);
            sums(mean);
            mean[0] *= share;
            mean[1] = f.before.kind == MINT_NORM_LAYER ? mean[1] * share : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float more[V];
#pragma unroll
            for (int i = 0; i < V; ++i) more[i] = 0.0f;
            if (a.d_stream)
                load_elements<S, V>(static_cast<const TS*>(a.d_stream) + (int64_t)r * a.d_stream_stride + row.at(c), row.left(c), more);
            float to[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float part = a.d_next && i < row.left(c) ? q * (d[c][i] - fmaf(x[c][i], mean[0], mean[1])) : 0.0f;
                d[c][i] = more[i] + part;
                to[i] = f.carry * d[c][i];
            }
            if (a.to_stream && row.left(c) > 0)
                store_elements<S, V>(static_cast<TS*>(a.to_stream) + (int64_t)r * a.to_stream_stride + row.at(c), row.left(c), to);
        }
        if constexpr (BLOCK) {
            constexpr int A = BIAS ? 2 : 1;                  // after's sums
            float yq = 1.0f;
            if (f.after.kind) yq = normalise(row, f.after, y, sums);
            float of_row[3] = {0.0f, 0.0f, 0.0f};            // of d' yh, of d', of G u (a gate by row)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float w[V], b[V], g[V], dg[V];
                weight_of(f.after, row.at(c), row.left(c), w);
                bias_of(f.after, row.at(c), row.left(c), b);
                gate_of(f, r, row.at(c), row.left(c), g);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float grad = f.scale * d[c][i], u = fmaf(y[c][i], w[i], b[i]), open = f.gate ? gate_value(f.gate_by, g[i]) : 1.0f;
                    of_row[2] = fmaf(grad, u, of_row[2]);
                    dg[i] = grad * u * (f.gate ? gate_slope(f.gate_by, g[i]) : 0.0f);
                    const float inner = grad * open, sum = by_channel ? grad : inner;
                    total[A][c][i] = fmaf(sum, y[c][i], total[A][c][i]);
                    if (BIAS) total[A + 1][c][i] += sum;
                    d[c][i] = inner * w[i];
                    of_row[0] = fmaf(d[c][i], y[c][i], of_row[0]);
                    of_row[1] += d[c][i];
                }
                if (a.to_gate && !by_row && !by_channel && row.left(c) > 0)
                    store_any(a.to_gate, f.gate_dtype, (int64_t)r * a.to_gate_stride + row.at(c), row.left(c), dg);
            }
            float m0 = 0.0f, m1 = 0.0f;
            if (f.after.kind || by_row) {
                sums(of_row);
                if (f.after.kind) m0 = of_row[0] * share;
                if (f.after.kind == MINT_NORM_LAYER) m1 = of_row[1] * share;
                if (by_row && a.to_gate && row.lane == 0)
                    store_one(a.to_gate, f.gate_dtype, (int64_t)r * a.to_gate_stride,
                              of_row[2] * gate_slope(f.gate_by, load_one(f.gate, f.gate_dtype, (int64_t)r * f.gate_row)));
            }
            if (a.to_y) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (row.left(c) <= 0) continue;
                    float to[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) to[i] = yq * (d[c][i] - fmaf(y[c][i], m0, m1));
                    store_elements<T, V>(static_cast<TT*>(a.to_y) + (int64_t)r * a.to_y_stride + row.at(c), row.left(c), to);
                }
            }
        }
    }
    if (a.sums) {
#pragma unroll
        for (int k = 0; k < SUMS; ++k)
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (row.left(c) > 0) store_elements<DT_F32, V>(a.sums + ((uint64_t)group * SUMS + k) * f.width + row.at(c), row.left(c), total[k][c]);
    }
}

// ---- rows too long for registers: they are read again for every step -------------
// A thread block has a row at a time; a thread reads back what it has written itself.
constexpr int kLongThreads = 1024;
using LongSums = RowSums<kLongThreads / 64, 3>;
template <typename F>
__device__ __forceinline__ void over_row(uint32_t width, const F& f) {
    for (uint64_t at = threadIdx.x * V; at < width; at += kLongThreads * V) f((uint32_t)at, (int64_t)width - (int64_t)at);
}
// m and q of a row whose numbers `load` brings
template <typename F>
__device__ __forceinline__ void long_stats(uint32_t width, const NormArgs& n, LongSums& sums, const F& load, float& m, float& q) {
    m = 0.0f;
    if (n.kind == MINT_NORM_LAYER) {
        float sum[1] = {0.0f};
        over_row(width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
            float x[V];
            load(at, left, x);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0] += x[i];
        });
        sums(sum);
        m = sum[0] / (float)width;
    }
    float square[1] = {0.0f};
    over_row(width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
        float x[V];
        load(at, left, x);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float c = i < left ? x[i] - m : 0.0f;
            square[0] = fmaf(c, c, square[0]);
        }
    });
    sums(square);
    q = 1.0f / sqrtf(square[0] / (float)width + n.eps);
}

template <int S, int T>
__global__ void __launch_bounds__(kLongThreads) join_long_kernel(JoinArgs a) {
    using TS = typename Elem<S>::type;
    using TT = typename Elem<T>::type;
    __shared__ float slots[2][kLongThreads / 64][3];
    LongSums sums = {slots};
    const uint64_t r = blockIdx.x;
    const TS* stream = static_cast<const TS*>(a.stream) + (int64_t)r * a.stream_stride;
    if (a.y) {
        const TT* const from = static_cast<const TT*>(a.y) + (int64_t)r * a.y_stride;
        TS* const to = static_cast<TS*>(a.new_stream) + (int64_t)r * a.new_stride;
        float m = 0.0f, q = 1.0f;
        if (a.after.kind)
            long_stats(a.width, a.after, sums, [&](uint32_t at, int64_t left, float (&x)[V]) MINT_INLINE_LAMBDA { load_elements<T, V>(from + at, left, x); }, m, q);
        over_row(a.width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
            float s[V], y[V], w[V], b[V], g[V];
            load_elements<S, V>(stream + at, left, s);
            load_elements<T, V>(from + at, left, y);
            weight_of(a.after, at, left, w);
            bias_of(a.after, at, left, b);
            gate_of(a, r, at, left, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = fmaf((y[i] - m) * q, w[i], b[i]) * (a.gate ? gate_value(a.gate_by, g[i]) : 1.0f);
                s[i] = fmaf(a.scale, u, a.carry * s[i]);
            }
            store_elements<S, V>(to + at, left, s);
        });
        stream = to;
    }
    if (!a.next) return;
    float m, q;
    const auto load = [&](uint32_t at, int64_t left, float (&x)[V]) MINT_INLINE_LAMBDA { load_elements<S, V>(stream + at, left, x); };
    long_stats(a.width, a.before, sums, load, m, q);
    over_row(a.width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
        float s[V], w[V], b[V];
        load(at, left, s);
        weight_of(a.before, at, left, w);
        bias_of(a.before, at, left, b);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = fmaf((s[i] - m) * q, w[i], b[i]);
        store_elements<T, V>(static_cast<TT*>(a.next) + (int64_t)r * a.next_stride + at, left, s);
    });
}

// A thread block's sums over its rows are kept in its part of the workspace.
template <int S, int T, bool BLOCK, bool BIAS>
__global__ void __launch_bounds__(kLongThreads) join_grad_long_kernel(JoinGradArgs a) {
    using TS = typename Elem<S>::type;
    using TT = typename Elem<T>::type;
    constexpr int SUMS = kSums<BLOCK, BIAS>, A = BIAS ? 2 : 1;
    __shared__ float slots[2][kLongThreads / 64][3];
    LongSums sums = {slots};
    const JoinArgs& f = a.f;
    const bool by_row = f.gate && f.gate_form == MINT_GATE_ROW, by_channel = f.gate && f.gate_form == MINT_GATE_CHANNEL;
    const auto add = [&](int k, uint32_t at, int64_t left, const float (&v)[V], bool first) MINT_INLINE_LAMBDA {
        if (!a.sums) return;
        float* const to = a.sums + ((uint64_t)blockIdx.x * SUMS + k) * f.width + at;
        float t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = 0.0f;
        if (!first) load_elements<DT_F32, V>(to, left, t);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] += v[i];
        store_elements<DT_F32, V>(to, left, t);
    };
    for (uint64_t r = blockIdx.x; r < f.rows; r += a.groups) {
        const bool first = r == blockIdx.x;
        const auto load_x = [&](uint32_t at, int64_t left, float (&v)[V]) MINT_INLINE_LAMBDA {
            load_elements<S, V>(static_cast<const TS*>(f.stream) + (int64_t)r * f.stream_stride + at, left, v);
        };
        const auto load_y = [&](uint32_t at, int64_t left, float (&v)[V]) MINT_INLINE_LAMBDA {
            load_elements<T, V>(static_cast<const TT*>(f.y) + (int64_t)r * f.y_stride + at, left, v);
        };
        const auto load_d = [&](uint32_t at, int64_t left, float (&v)[V]) MINT_INLINE_LAMBDA {
            load_elements<T, V>(static_cast<const TT*>(a.d_next) + (int64_t)r * a.d_next_stride + at, left, v);
        };
        float m = 0.0f, q = 0.0f, mean[2] = {0.0f, 0.0f};
        if (a.d_next) {
            long_stats(f.width, f.before, sums, load_x, m, q);
            over_row(f.width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
                float x[V], d[V], w[V], dx[V];
                load_x(at, left, x);
                load_d(at, left, d);
                weight_of(f.before, at, left, w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[i] = (x[i] - m) * q;
                    dx[i] = d[i] * x[i];
                    mean[0] = fmaf(d[i] * w[i], x[i], mean[0]);
                    mean[1] = fmaf(d[i], w[i], mean[1]);
                }
                add(0, at, left, dx, first);
                if (BIAS) add(1, at, left, d, first);
            });
            sums(mean);
            mean[0] /= (float)f.width;
            mean[1] = f.before.kind == MINT_NORM_LAYER ? mean[1] / (float)f.width : 0.0f;
        } else if (first) {
            const float none[V] = {};
            over_row(f.width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
                add(0, at, left, none, true);
                if (BIAS) add(1, at, left, none, true);
            });
        }
        // D, as often as it is wanted
        const auto load_whole = [&](uint32_t at, int64_t left, float (&v)[V]) MINT_INLINE_LAMBDA {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = 0.0f;
            if (a.d_stream) load_elements<S, V>(static_cast<const TS*>(a.d_stream) + (int64_t)r * a.d_stream_stride + at, left, v);
            if (a.d_next) {
                float x[V], d[V], w[V];
                load_x(at, left, x);
                load_d(at, left, d);
                weight_of(f.before, at, left, w);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] += i < left ? q * (d[i] * w[i] - fmaf((x[i] - m) * q, mean[0], mean[1])) : 0.0f;
            }
        };
        float ym = 0.0f, yq = 1.0f, of_row[3] = {0.0f, 0.0f, 0.0f};
        // what the gate and the norm make of G, and y normalised
        const auto inner_of = [&](uint32_t at, int64_t left, const float (&whole)[V], float (&y)[V], float (&inner)[V], float (&w)[V], float (&dg)[V],
                                  float (&gu)[V]) MINT_INLINE_LAMBDA {
            float b[V], g[V];
            load_y(at, left, y);
            weight_of(f.after, at, left, w);
            bias_of(f.after, at, left, b);
            gate_of(f, r, at, left, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                y[i] = i < left ? (y[i] - ym) * yq : 0.0f;
                const float grad = f.scale * whole[i];
                gu[i] = grad * fmaf(y[i], w[i], b[i]);
                dg[i] = gu[i] * (f.gate ? gate_slope(f.gate_by, g[i]) : 0.0f);
                inner[i] = grad * (f.gate ? gate_value(f.gate_by, g[i]) : 1.0f);
            }
        };
        if (BLOCK && f.after.kind) long_stats(f.width, f.after, sums, load_y, ym, yq);
        over_row(f.width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
            float whole[V], to[V];
            load_whole(at, left, whole);
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = f.carry * whole[i];
            if (BLOCK) {
                float y[V], inner[V], w[V], dg[V], gu[V], of_w[V], of_b[V];
                inner_of(at, left, whole, y, inner, w, dg, gu);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    of_row[0] = fmaf(inner[i] * w[i], y[i], of_row[0]);
                    of_row[1] = fmaf(inner[i], w[i], of_row[1]);
                    of_row[2] += gu[i];
                    of_b[i] = by_channel ? f.scale * whole[i] : inner[i];
                    of_w[i] = of_b[i] * y[i];
                }
                add(A, at, left, of_w, first);
                if (BIAS) add(A + 1, at, left, of_b, first);
                if (a.to_gate && !by_row && !by_channel) store_any(a.to_gate, f.gate_dtype, (int64_t)r * a.to_gate_stride + at, left, dg);
            }
            // (the gradient of the stream may not be written where what it is made from lies: it is made again below)
            if (!BLOCK && a.to_stream) store_elements<S, V>(static_cast<TS*>(a.to_stream) + (int64_t)r * a.to_stream_stride + at, left, to);
        });
        if (BLOCK) {
            sums(of_row);
            const float m0 = f.after.kind ? of_row[0] / (float)f.width : 0.0f;
            const float m1 = f.after.kind == MINT_NORM_LAYER ? of_row[1] / (float)f.width : 0.0f;
            if (by_row && a.to_gate && threadIdx.x == 0)
                store_one(a.to_gate, f.gate_dtype, (int64_t)r * a.to_gate_stride,
                          of_row[2] * gate_slope(f.gate_by, load_one(f.gate, f.gate_dtype, (int64_t)r * f.gate_row)));
            over_row(f.width, [&](uint32_t at, int64_t left) MINT_INLINE_LAMBDA {
                float whole[V], y[V], inner[V], w[V], dg[V], gu[V], to[V];
                load_whole(at, left, whole);
                inner_of(at, left, whole, y, inner, w, dg, gu);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    to[i] = yq * (inner[i] * w[i] - fmaf(y[i], m0, m1));
                    whole[i] *= f.carry;
                }
                if (a.to_y) store_elements<T, V>(static_cast<TT*>(a.to_y) + (int64_t)r * a.to_y_stride + at, left, to);
                if (a.to_stream) store_elements<S, V>(static_cast<TS*>(a.to_stream) + (int64_t)r * a.to_stream_stride + at, left, whole);
            });
        }
    }
}

// ---- the launches --------------------------------------------------------------------
// Lanes and numbers of a lane: 64 lanes (four rows to a thread block) up to 512 numbers, then thread blocks of 256 to 1024.
constexpr uint32_t kLongest = 1024 * V * 2;
template <int S, int T>
int go_join(const JoinArgs& a, hipStream_t s) {
#define MINT_JOIN(LANES, C) return Launch<&join_kernel<S, T, LANES, C>>::go((uint32_t)ceil_div(a.rows, LANES < 256 ? 256 / LANES : 1), LANES < 256 ? 256 : LANES, 0, s, a)
    if (a.width <= 64 * V) MINT_JOIN(64, 1);
    if (a.width <= 128 * V) MINT_JOIN(64, 2);
    if (a.width <= 256 * V) MINT_JOIN(256, 1);
    if (a.width <= 512 * V) MINT_JOIN(256, 2);
    if (a.width <= 1024 * V) MINT_JOIN(512, 2);
    if (a.width <= kLongest) MINT_JOIN(1024, 2);
#undef MINT_JOIN
    return Launch<&join_long_kernel<S, T>>::go((uint32_t)a.rows, kLongThreads, 0, s, a);
}
template <int S, int T, bool BLOCK, bool BIAS>
int go_join_grad(const JoinGradArgs& a, hipStream_t s) {
#define MINT_JOIN(LANES, C) \
    return Launch<&join_grad_kernel<S, T, LANES, C, BLOCK, BIAS>>::go((uint32_t)ceil_div(a.groups, LANES < 256 ? 256 / LANES : 1), LANES < 256 ? 256 : LANES, 0, s, a)
    if (a.f.width <= 64 * V) MINT_JOIN(64, 1);
    if (a.f.width <= 128 * V) MINT_JOIN(64, 2);
    if (a.f.width <= 256 * V) MINT_JOIN(256, 1);
    if (a.f.width <= 512 * V) MINT_JOIN(256, 2);
    if (a.f.width <= 1024 * V) MINT_JOIN(512, 2);
#undef MINT_JOIN
    return Launch<&join_grad_long_kernel<S, T, BLOCK, BIAS>>::go(a.groups, kLongThreads, 0, s, a);
}
template <int S, int T>
int go_join_grad(const JoinGradArgs& a, bool bias, hipStream_t s) {
    if (a.f.y) return bias ? go_join_grad<S, T, true, true>(a, s) : go_join_grad<S, T, true, false>(a, s);
    return bias ? go_join_grad<S, T, false, true>(a, s) : go_join_grad<S, T, false, false>(a, s);
}

// A launcher for each pair of types that go together (norms_family.hip): the stream is of the block's type, or in 32 bits.
#define MINT_NORM_FAMILY(X) X(f16, DT_F16, DT_F16) X(bf16, DT_BF16, DT_BF16) X(f32, DT_F32, DT_F32) X(f32_f16, DT_F32, DT_F16) X(f32_bf16, DT_F32, DT_BF16)
#define MINT_DECLARE(name, S, T)                               \
    int launch_join_##name(const JoinArgs& a, hipStream_t s);  \
    int launch_join_grad_##name(const JoinGradArgs& a, bool bias, hipStream_t s);
MINT_NORM_FAMILY(MINT_DECLARE)
#undef MINT_DECLARE

}  // namespace mint
