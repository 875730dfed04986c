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

// Of a row in registers: V numbers of a lane, LANES lanes side by side.  What lies behind the row's end is zero, and stays.  WHOLE: a lane has all of its
// numbers or none (ends inside a lane's numbers cost registers, which the kernels that hold most of them do not have).
template <int LANES, bool WHOLE>
struct RowOf {
    static constexpr bool whole = WHOLE;
    uint32_t width, at;
    int64_t left;
    __device__ __forceinline__ RowOf(uint32_t w, uint32_t lane)
        : width(w), at(lane * V), left(WHOLE ? (lane * V < w ? V : 0) : (int64_t)w - lane * V) {}
    // takes the mean off, but not off what is not there
    __device__ __forceinline__ void centre(float (&x)[V], float mean) const {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = i < left ? x[i] - mean : 0.0f;
    }
    static __device__ __forceinline__ float sum(const float (&x)[V]) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) s += x[i];
        return s;
    }
    static __device__ __forceinline__ float dot(const float (&x)[V], const float (&y)[V]) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) s = fmaf(x[i], y[i], s);
        return s;
    }
};
// x becomes (x - m) q; q comes back
template <int LANES, bool WHOLE, typename Sums>
__device__ __forceinline__ float normalise(const RowOf<LANES, WHOLE>& row, const NormArgs& n, float (&x)[V], Sums& sums) {
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
    for (int i = 0; i < V; ++i) x[i] *= q;
    return q;
}
// a lane's numbers of the weight, of the bias
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
// a lane's numbers of a row's gate, as it was given (ones where there is none)
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

// V numbers as they are in memory, zeros behind the `left` first: what is on its way while the row before is worked on.  At a row's end the lane reads the row's
// last V numbers and moves its own to the front when they are wanted: one by one they would have to be there at once, for what is put together of
// them, and the other lanes' rows with them (8000 x 2501 f16, rms: 70 us, so 56; 2504 numbers 39).
template <int DT>
struct Raw {
    using T = typename Elem<DT>::type;
    static constexpr int WORDS = V * (int)sizeof(T) / 4;
    typedef uint32_t words __attribute__((ext_vector_type(WORDS), aligned(sizeof(T))));
    typedef T numbers __attribute__((ext_vector_type(V)));
    uint32_t v[WORDS];           // (words: numbers of 16 bits would take a register each)
    // (where the row is, the same for all, apart from the lane's place in it: the address takes one register)
    template <typename Row>
    __device__ __forceinline__ void load(const void* p, int64_t row, const Row& of) {
        const T* const first = static_cast<const T*>(p) + row;
        if (of.whole ? of.left > 0 : of.width >= V) {
            const words w = *(MINT_GLOBAL const words*)as_global(first + (of.whole ? of.at : min(of.at, of.width - V)));
#pragma unroll
            for (int i = 0; i < WORDS; ++i) v[i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) v[i] = 0u;
            if (of.whole) return;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < of.left) {
                    if constexpr (sizeof(T) == 4) v[i] = *(MINT_GLOBAL const uint32_t*)as_global(first + i);
                    else v[i / 2] |= (uint32_t)*(MINT_GLOBAL const uint16_t*)as_global(first + i) << (i % 2 * 16);
                }
        }
    }
    // `of` as it was for load()
    template <typename Row>
    __device__ __forceinline__ void place(const Row& of) {
        if (of.whole || of.left >= V || of.width < V) return;
        const uint32_t skip = of.left > 0 ? (uint32_t)(V - of.left) : V;         // numbers in front that are another lane's
        if constexpr (sizeof(T) == 2) {
            if (skip & 1u) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) v[i] = __builtin_amdgcn_alignbit(i + 1 < WORDS ? v[i + 1] : 0u, v[i], 16);
            }
        }
#pragma unroll
        for (int step = 1; step <= WORDS; step *= 2)
            if (skip & (uint32_t)(step * V / WORDS)) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i) v[i] = i + step < WORDS ? v[i + step] : 0u;
            }
    }
    template <typename Row>
    __device__ __forceinline__ void get(const Row& of, float (&x)[V]) {
        place(of);
        typedef uint32_t whole __attribute__((ext_vector_type(WORDS)));
        whole w;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = v[i];
        const numbers n = __builtin_bit_cast(numbers, w);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = Elem<DT>::load(n[i]);
    }
};
// a lane's numbers of a row's gate, as it was given, for rows in registers
template <typename Row>
__device__ __forceinline__ void gate_of(const JoinArgs& a, uint64_t r, const Row& of, float (&g)[V]) {
    const auto all = [&](auto raw) MINT_INLINE_LAMBDA {
        raw.load(a.gate, (int64_t)r * a.gate_row, of);
        raw.get(of, g);
    };
    if (!a.gate || a.gate_form == MINT_GATE_ROW) gate_of(a, r, of.at, of.left, g);
    else if (a.gate_dtype == MINT_F32) all(Raw<DT_F32>());
    else if (a.gate_dtype == MINT_BF16) all(Raw<DT_BF16>());
    else all(Raw<DT_F16>());
}
constexpr int threads_of(int lanes) { return lanes == 64 ? 256 : lanes; }         // four rows to a thread block, or one
constexpr int rows_of(int lanes) { return lanes == 64 ? 4 : 1; }

// S: the stream's type, T: that of y and of h.  LANES lanes have every groups-th row, of which the next one is on its way while one is worked on;
// the weights stay in registers.  Bound by memory: 16384 x 4096 bf16 with a gate by channel 98 us
// (5.5 TB/s; rows one by one, the weights read again for each, 134), 8192 x 8192 with the stream in 32 bits and a gate by row 136 (5.9; the gate evaluated for each of a lane's
// numbers 166).  Widths between those that fill their lanes, and narrow ones, leave lanes without work: 16384 x 2560 without a block 31 us for 168 MB, 10^6 x 128 235 for 512.
template <int S, int T, int LANES, bool WHOLE>
__global__ void __launch_bounds__(threads_of(LANES)) join_kernel(JoinArgs a) {
    using TS = typename Elem<S>::type;
    using TT = typename Elem<T>::type;
    constexpr int WAVES = LANES / 64, ROWS = rows_of(LANES);
    __shared__ float slots[2][WAVES][1];
    const uint32_t groups = gridDim.x * ROWS, first = blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / LANES : 0u);
    if (first >= a.rows) return;
    const RowOf<LANES, WHOLE> row(a.width, threadIdx.x % LANES);
    const uint32_t at = row.at;
    const int64_t left = row.left;
    RowSums<WAVES, 1> sums = {slots};
    // u's weight and bias with the scale and a gate by channel in them.  (An infinite gate is of the whole u: of the weight and of the bias it would make
    // infinities whose sum is NaN.  Then the gates are read for every row, as those of every number are.)
    bool one_by_one = a.gate && a.gate_form != MINT_GATE_CHANNEL;
    float wa[V], ba[V], wb[V], bb[V], open[V];
    weight_of(a.after, at, left, wa);
    bias_of(a.after, at, left, ba);
    weight_of(a.before, at, left, wb);
    bias_of(a.before, at, left, bb);
    if (!one_by_one) {
        bool infinite = false;
        gate_of(a, 0, row, open);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            open[i] = a.scale * (a.gate ? gate_value(a.gate_by, open[i]) : 1.0f);
            infinite |= fabsf(open[i]) == INFINITY;
        }
        one_by_one = a.gate && __ballot(infinite) != 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float all = one_by_one ? a.scale : open[i];
        wa[i] *= all;
        ba[i] *= all;
    }
    Raw<S> next_s;
    Raw<T> next_y;
    const auto ask = [&](uint32_t r) MINT_INLINE_LAMBDA {
        next_s.load(a.stream, (int64_t)r * a.stream_stride, row);
        if (a.y) next_y.load(a.y, (int64_t)r * a.y_stride, row);
    };
    ask(first);
    for (uint64_t r = first; r < a.rows; r += groups) {
        float s[V], y[V];
        next_s.get(row, s);
        if (a.y) next_y.get(row, y);
        if (r + groups < a.rows) ask((uint32_t)(r + groups));
        if (a.y) {
            if (a.after.kind) normalise(row, a.after, y, sums);
            if (one_by_one && a.gate_form == MINT_GATE_ROW) {
                const float one = gate_value(a.gate_by, load_one(a.gate, a.gate_dtype, (int64_t)r * a.gate_row));
#pragma unroll
                for (int i = 0; i < V; ++i) open[i] = one;
            } else if (one_by_one) {
                gate_of(a, r, row, open);
#pragma unroll
                for (int i = 0; i < V; ++i) open[i] = gate_value(a.gate_by, open[i]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = fmaf(y[i], wa[i], ba[i]);
                const float sum = one_by_one ? fmaf(open[i], u, a.carry * s[i]) : fmaf(a.carry, s[i], u);
                // (as it is stored: what the next norm is of)
                s[i] = i < left ? Elem<S>::load(Elem<S>::round(sum)) : 0.0f;
            }
            if (left > 0) store_elements<S, V>(static_cast<TS*>(a.new_stream) + (int64_t)r * a.new_stride + at, left, s);
        }
        if (!a.next) continue;
        normalise(row, a.before, s, sums);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = fmaf(s[i], wb[i], bb[i]);
        if (left > 0) store_elements<T, V>(static_cast<TT*>(a.next) + (int64_t)r * a.next_stride + at, left, s);
    }
}

struct JoinGradArgs {
    JoinArgs f;                                 // stream: the new one; y, gate, norms
    const void *d_stream, *d_next;              // either may be 0
    void *to_stream, *to_y, *to_gate;
    int64_t d_stream_stride, d_next_stride, to_stream_stride, to_y_stride, to_gate_stride;
    float* sums;                                // (groups, SUMS, width): each thread block's sums over its rows
    uint32_t groups;                            // thread blocks
};
// Which of a group's sums over rows are where: before's weight, [its bias,] [after's weight, [its bias]].
template <bool BLOCK, bool BIAS>
constexpr int kSums = (BLOCK ? 2 : 1) * (BIAS ? 2 : 1);

// LANES lanes have every groups-th row; the weights stay in registers, and up to 4096 numbers so do the sums over their rows, while the next row is on its
// way (AHEAD); a thread block of 1024 has the sums in LDS.
// Bound by memory, and by three meetings for a row: 16384 x 4096 bf16 with a gate by channel 177 us, 4.6 TB/s
// (twice eight numbers to a lane, half as many wavefronts, nothing held or ahead: 397), 8192 x 8192 with the stream in 32 bits and a gate by row 295, 4.2.
template <int S, int T, int LANES, bool WHOLE, bool BLOCK, bool BIAS, int GATE>      // GATE: 0 (none, or by channel), MINT_GATE_ROW, MINT_GATE_ALL
__global__ void __launch_bounds__(threads_of(LANES)) join_grad_kernel(JoinGradArgs a) {
    using TS = typename Elem<S>::type;
    using TT = typename Elem<T>::type;
    constexpr int WAVES = LANES / 64, ROWS = rows_of(LANES), SUMS = kSums<BLOCK, BIAS>;
    constexpr bool AHEAD = LANES < 1024;
    __shared__ float slots[2][WAVES][3];
    __shared__ __attribute__((aligned(16))) float joined[!AHEAD ? SUMS * LANES * V : ROWS > 1 ? (ROWS - 1) * SUMS * LANES * V : 1];
    const uint32_t groups = gridDim.x * ROWS, nth = ROWS > 1 ? threadIdx.x / LANES : 0u;
    const JoinArgs& f = a.f;
    const uint32_t lane = threadIdx.x % LANES;
    const RowOf<LANES, WHOLE> row(f.width, lane);
    const uint32_t at = row.at;
    const int64_t left = row.left;
    RowSums<WAVES, 3> sums = {slots};
    const float share = 1.0f / (float)f.width;
    constexpr bool by_row = GATE == MINT_GATE_ROW;
    float total[AHEAD ? SUMS : 1][V], wb[V], wa[V], ba[V];
    // a lane's eight of sum k in LDS: four, and four behind all lanes' first ones
    const auto in_lds = [&](int k, int half) MINT_INLINE_LAMBDA { return reinterpret_cast<f32x4*>(joined + ((k * 2 + half) * LANES + lane) * 4); };
    const auto add = [&](int k, const float (&v)[V]) MINT_INLINE_LAMBDA {
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < V; ++i) total[k][i] += v[i];
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) *in_lds(k, half) += f32x4{v[half * 4], v[half * 4 + 1], v[half * 4 + 2], v[half * 4 + 3]};
        }
    };
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < V; ++i) total[k][i] = 0.0f;
        } else {
            *in_lds(k, 0) = *in_lds(k, 1) = f32x4{0, 0, 0, 0};
        }
    }
    constexpr bool HOLD = AHEAD || GATE == 0;
    if (HOLD) weight_of(f.before, at, left, wb);
    if (BLOCK && HOLD) {
        weight_of(f.after, at, left, wa);
        bias_of(f.after, at, left, ba);
        if (GATE == 0 && f.gate) {           // (of a gate by channel the sums are without it: column_sums_kernel)
            float g[V];
            gate_of(f, 0, row, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                wa[i] *= gate_value(f.gate_by, g[i]);
                __builtin_amdgcn_sched_barrier(0);           // (one behind the other: all at once take registers that there are not)
            }
        }
    }
    Raw<S> next_x, next_d;
    Raw<T> next_h, next_y;
    const auto ask = [&](uint32_t r) MINT_INLINE_LAMBDA {
        if (a.d_next) {
            next_x.load(f.stream, (int64_t)r * f.stream_stride, row);
            next_h.load(a.d_next, (int64_t)r * a.d_next_stride, row);
        }
        if (a.d_stream) next_d.load(a.d_stream, (int64_t)r * a.d_stream_stride, row);
        if (BLOCK) next_y.load(f.y, (int64_t)r * f.y_stride, row);
    };
    const uint32_t first = blockIdx.x * ROWS + nth;
    if (AHEAD && first < f.rows) ask(first);
    for (uint64_t r = first; r < f.rows; r += groups) {
        if constexpr (!AHEAD) {
            compiler_fence();                                // (or what does not change is read ahead of all rows, into registers that there are not)
            ask((uint32_t)r);
        }
        float row_open = 1.0f, row_slope = 0.0f, g[V];
        if (AHEAD && GATE == MINT_GATE_ALL) gate_of(f, r, row, g);
        if (by_row) {
            const float one = load_one(f.gate, f.gate_dtype, (int64_t)r * f.gate_row);
            row_open = gate_value(f.gate_by, one);
            row_slope = gate_slope(f.gate_by, one);
            __builtin_amdgcn_sched_barrier(0);
        }
        float x[V], h[V], d[V], y[V];
#pragma unroll
        for (int i = 0; i < V; ++i) d[i] = 0.0f;
        if (a.d_next) {
            next_x.get(row, x);
            next_h.get(row, h);
        }
        if (a.d_stream) next_d.get(row, d);
        if (BLOCK && AHEAD) next_y.get(row, y);
        if (AHEAD && r + groups < f.rows) ask((uint32_t)(r + groups));
        if (a.d_next) {
            const float q = normalise(row, f.before, x, sums);
            if (!HOLD) weight_of(f.before, at, left, wb);
            float mean[2], part[V];
#pragma unroll
            for (int i = 0; i < V; ++i) part[i] = h[i] * x[i];
            add(0, part);
            if (BIAS) add(1, h);
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] *= wb[i];
            mean[0] = row.dot(h, x);
            mean[1] = row.sum(h);
            sums(mean);
            mean[0] *= share;
            mean[1] = f.before.kind == MINT_NORM_LAYER ? mean[1] * share : 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] += i < left ? q * (h[i] - fmaf(x[i], mean[0], mean[1])) : 0.0f;
        }
        if (a.to_stream && left > 0) {
            float to[V];
#pragma unroll
            for (int i = 0; i < V; ++i) to[i] = f.carry * d[i];
            store_elements<S, V>(static_cast<TS*>(a.to_stream) + (int64_t)r * a.to_stream_stride + at, left, to);
        }
        if constexpr (BLOCK) {
            constexpr int A = BIAS ? 2 : 1;                  // after's sums
            float yq = 1.0f;
            if (!AHEAD) {
                __builtin_amdgcn_sched_barrier(0);
                next_y.get(row, y);
            }
            if (f.after.kind) yq = normalise(row, f.after, y, sums);
            __builtin_amdgcn_sched_barrier(0);               // (what follows would begin further above, in registers that there are not)
            if (!HOLD) {
                weight_of(f.after, at, left, wa);
                bias_of(f.after, at, left, ba);
            }
            float of_row[3] = {0.0f, 0.0f, 0.0f};            // of d' yh, of d', of G b; d' without a gate by row
            if constexpr (GATE == MINT_GATE_ALL) {
                float dg[V];
                if (!AHEAD) gate_of(f, r, row, g);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float grad = f.scale * d[i];
                    dg[i] = grad * fmaf(y[i], wa[i], ba[i]) * gate_slope(f.gate_by, g[i]);
                    d[i] = grad * gate_value(f.gate_by, g[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (a.to_gate && left > 0) store_any(a.to_gate, f.gate_dtype, (int64_t)r * a.to_gate_stride + at, left, dg);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) d[i] *= f.scale;
            }
            __builtin_amdgcn_sched_barrier(0);
            float part[V];
#pragma unroll
            for (int i = 0; i < V; ++i) part[i] = row_open * d[i] * y[i];
            add(A, part);
            if (BIAS) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    part[i] = row_open * d[i];
                    if (by_row) of_row[2] = fmaf(d[i], ba[i], of_row[2]);
                }
                add(A + 1, part);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                d[i] *= wa[i];
                of_row[0] = fmaf(d[i], y[i], of_row[0]);
                of_row[1] += d[i];
            }
            float m0 = 0.0f, m1 = 0.0f;
            if (f.after.kind || by_row) {
                sums(of_row);
                if (f.after.kind) m0 = of_row[0] * share;
                if (f.after.kind == MINT_NORM_LAYER) m1 = of_row[1] * share;
            }
            if (a.to_y && left > 0) {
                float to[V];
#pragma unroll
                for (int i = 0; i < V; ++i) to[i] = yq * row_open * (d[i] - fmaf(y[i], m0, m1));
                store_elements<T, V>(static_cast<TT*>(a.to_y) + (int64_t)r * a.to_y_stride + at, left, to);
            }
            if (by_row && a.to_gate && lane == 0)
                store_one(a.to_gate, f.gate_dtype, (int64_t)r * a.to_gate_stride, (of_row[0] + of_row[2]) * row_slope);
        }
    }
    if (!a.sums) return;
    if constexpr (ROWS > 1) {                                // a thread block's sums are one group's
        if (nth) {
#pragma unroll
            for (int k = 0; k < SUMS; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) joined[(((nth - 1) * SUMS + k) * V + i) * LANES + lane] = total[k][i];
        }
        __syncthreads();
        if (nth) return;
#pragma unroll
        for (int n = 0; n < ROWS - 1; ++n)
#pragma unroll
            for (int k = 0; k < SUMS; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) total[k][i] += joined[((n * SUMS + k) * V + i) * LANES + lane];
    }
    if (left > 0) {
        if constexpr (!AHEAD) {
#pragma unroll
            for (int k = 0; k < SUMS; ++k) {
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = (*in_lds(k, i / 4))[i % 4];
                store_elements<DT_F32, V>(a.sums + ((uint64_t)blockIdx.x * SUMS + k) * f.width + at, left, v);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < (AHEAD ? SUMS : 1); ++k) store_elements<DT_F32, V>(a.sums + ((uint64_t)blockIdx.x * SUMS + k) * f.width + at, left, total[k]);
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

// A thread block's sums over its rows are kept in its part of the workspace.  Each of the steps (two statistics, their sums, the results) reads x, d, y and the gate
// again: 8192 x 9000 bf16, both norms, 725 us (1.2 TB/s of what has to pass), 4096 x 16384 514 (1.6), 8192 x 5001, whose ends are inside a lane's numbers, 564 (0.9; 8192 x 5000 in
// registers 165), 8192 x 8192 with the stream in 32 bits, biases and a gate by row 775 (1.6; without biases 295).
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
// Lanes of a row: 64 (four rows to a thread block) up to 512 numbers, then a thread block of 128 to 1024.
constexpr uint32_t kLongest = 1024 * V;
constexpr uint32_t kMostLong = 1u << 18;         // longer ones of a launch, which has fewer than 2^32 threads
inline uint32_t threads_for(uint64_t width) {
    return width <= 64 * V ? 256 : width <= 128 * V ? 128 : width <= 256 * V ? 256 : width <= 512 * V ? 512 : 1024;
}
// Thread blocks: as many as are at work together; of a number that does not depend on the device, so that a sum over rows has the same order everywhere.
inline uint32_t blocks_of(uint64_t rows, uint64_t width, uint32_t threads) {
    return (uint32_t)std::min<uint64_t>(ceil_div(rows, width <= 64 * V ? 4 : 1), 256 * threads / threads_for(width));
}
inline uint32_t blocks_of(uint64_t rows, uint64_t width) { return blocks_of(rows, width, 1024); }      // ... of the gradients
template <int S, int T, bool WHOLE>
int go_join_rows(const JoinArgs& a, hipStream_t s) {
#define MINT_JOIN(LANES) return Launch<&join_kernel<S, T, LANES, WHOLE>>::go(blocks_of(a.rows, a.width, 2048), threads_of(LANES), 0, s, a)
    if (a.width <= 64 * V) MINT_JOIN(64);
    if (a.width <= 128 * V) MINT_JOIN(128);
    if (a.width <= 256 * V) MINT_JOIN(256);
    if (a.width <= 512 * V) MINT_JOIN(512);
    MINT_JOIN(1024);
#undef MINT_JOIN
}
template <int S, int T>
int go_join(const JoinArgs& a, hipStream_t s) {
    if (a.width > kLongest) {
        const auto on = [](const void* p, int64_t rows, int64_t stride, size_t size) { return p ? static_cast<const uint8_t*>(p) + rows * stride * (int64_t)size : nullptr; };
        const size_t of_s = sizeof(typename Elem<S>::type), of_t = sizeof(typename Elem<T>::type), of_gate = a.gate_dtype == MINT_F32 ? 4 : 2;
        for (uint32_t first = 0; first < a.rows; first += kMostLong) {
            JoinArgs part = a;
            part.rows = std::min(a.rows - first, kMostLong);
            part.stream = on(a.stream, first, a.stream_stride, of_s);
            part.new_stream = const_cast<uint8_t*>(on(a.new_stream, first, a.new_stride, of_s));
            part.y = on(a.y, first, a.y_stride, of_t);
            part.next = const_cast<uint8_t*>(on(a.next, first, a.next_stride, of_t));
            part.gate = on(a.gate, first, a.gate_row, of_gate);              // (by channel its rows are 0 apart)
            if (const int err = Launch<&join_long_kernel<S, T>>::go(part.rows, kLongThreads, 0, s, part)) return err;
        }
        return MINT_OK;
    }
    return a.width % V == 0 ? go_join_rows<S, T, true>(a, s) : go_join_rows<S, T, false>(a, s);
}
template <int S, int T, bool WHOLE, bool BLOCK, bool BIAS, int GATE>
int go_join_grad_rows(const JoinGradArgs& a, hipStream_t s) {
#define MINT_JOIN(LANES) return Launch<&join_grad_kernel<S, T, LANES, WHOLE, BLOCK, BIAS, GATE>>::go(a.groups, threads_of(LANES), 0, s, a)
    if (a.f.width <= 64 * V) MINT_JOIN(64);
    if (a.f.width <= 128 * V) MINT_JOIN(128);
    if (a.f.width <= 256 * V) MINT_JOIN(256);
    if (a.f.width <= 512 * V) MINT_JOIN(512);
    // (the registers of a thread block of 1024 do not do for every combination)
    if constexpr (WHOLE && (GATE != MINT_GATE_ROW || S != DT_F32 || (!BIAS && T != DT_F32))) MINT_JOIN(1024);
    else return Launch<&join_grad_long_kernel<S, T, BLOCK, BIAS>>::go(a.groups, kLongThreads, 0, s, a);
#undef MINT_JOIN
}
template <int S, int T, bool BLOCK, bool BIAS>
int go_join_grad(const JoinGradArgs& a, hipStream_t s) {
    if (a.f.width > kLongest) return Launch<&join_grad_long_kernel<S, T, BLOCK, BIAS>>::go(a.groups, kLongThreads, 0, s, a);
    const bool whole = a.f.width % V == 0;
    if constexpr (BLOCK) {
        if (a.f.gate && a.f.gate_form == MINT_GATE_ALL)
            return whole ? go_join_grad_rows<S, T, true, true, BIAS, MINT_GATE_ALL>(a, s) : go_join_grad_rows<S, T, false, true, BIAS, MINT_GATE_ALL>(a, s);
        if (a.f.gate && a.f.gate_form == MINT_GATE_ROW)
            return whole ? go_join_grad_rows<S, T, true, true, BIAS, MINT_GATE_ROW>(a, s) : go_join_grad_rows<S, T, false, true, BIAS, MINT_GATE_ROW>(a, s);
    }
    return whole ? go_join_grad_rows<S, T, true, BLOCK, BIAS, 0>(a, s) : go_join_grad_rows<S, T, false, BLOCK, BIAS, 0>(a, s);
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
