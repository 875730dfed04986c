// A token's rows from its experts, added up with their weights, and the gradients of both:
//
//   out_t = sum_j w_tj rows[slot_tj]        d_rows[slot_tj] = w_tj d_t        d_w_tj = < d_t, rows[slot_tj] >
//
// Sums in 32 bits, in the order of j; a slot of -1 (or beyond the rows) adds nothing.  Without weights all are 1.
// Every row is read once and every result written once: bound by memory (16384 tokens of 4 rows of 4096 numbers of 16 bits:
// 132 us forward, 5.1 TB/s, and 218 back, 5.5 TB/s).
#include "operators.hpp"

namespace mint {
namespace {

struct CombineArgs {
    const void* rows;
    const int32_t* slots;
    const float* weights;
    void* out;
    int64_t row_stride, out_stride;
    uint32_t n_rows, tokens, topk, width, chunks;     // chunks of 64 lanes' elements to a row
};
constexpr int kCombineV = 8, kCombineWaves = 4;

// A wavefront has 512 elements of a token's row.
template <int DT>
__global__ void __launch_bounds__(64 * kCombineWaves) combine_kernel(CombineArgs a) {
    using T = typename Elem<DT>::type;
    constexpr int V = kCombineV;
    const uint64_t unit = (uint64_t)blockIdx.x * kCombineWaves + __builtin_amdgcn_readfirstlane(wave_in_block());
    const uint32_t token = (uint32_t)(unit / a.chunks), at = ((uint32_t)(unit % a.chunks) * 64u + lane_id()) * V;
    if (token >= a.tokens || at >= a.width) return;
    const int64_t left = (int64_t)a.width - at;
    const int32_t* const slots = a.slots + (uint64_t)token * a.topk;
    const float* const weights = a.weights ? a.weights + (uint64_t)token * a.topk : nullptr;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    for (uint32_t j0 = 0; j0 < a.topk; j0 += 4) {
        float v[4][V], w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t j = j0 + u;
            const int32_t slot = j < a.topk ? slots[j] : -1;
            const bool there = (uint32_t)slot < a.n_rows;
            w[u] = there ? weights ? weights[j] : 1.0f : 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] = 0.0f;
            if (there) load_elements<DT, V>(static_cast<const T*>(a.rows) + slot * a.row_stride + at, left, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = fmaf(w[u], v[u][i], sum[i]);
    }
    store_elements<DT, V>(static_cast<T*>(a.out) + token * a.out_stride + at, left, sum);
}

struct CombineGradArgs {
    const void *d_out, *rows;
    const int32_t *slots, *ends;      // ends: the number of rows that some token has
    const float* weights;
    void* d_rows;
    float* d_weights;
    int64_t d_stride, row_stride, d_row_stride;
    uint32_t n_rows, tokens, topk, width;
};
// A thread block has a token; those behind the tokens' clear the rows that are no token's.  (A slot that is one of those counts as none:
// no row is written by two.)
constexpr uint32_t kClearing = 128;
template <int DT>
__global__ void __launch_bounds__(64 * kCombineWaves) combine_grad_kernel(CombineGradArgs a) {
    using T = typename Elem<DT>::type;
    constexpr int V = kCombineV;
    __shared__ float part[kCombineWaves][4];
    const uint32_t step = 64 * kCombineWaves * V, used = a.n_rows ? min((uint32_t)max(*a.ends, 0), a.n_rows) : 0u;
    if (blockIdx.x >= a.tokens) {
        const float none[V] = {};
        for (uint64_t row = (uint64_t)used + (blockIdx.x - a.tokens); row < a.n_rows; row += kClearing)
            for (uint32_t at = threadIdx.x * V; at < a.width; at += step)
                store_elements<DT, V>(static_cast<T*>(a.d_rows) + row * a.d_row_stride + at, (int64_t)a.width - at, none);
        return;
    }
    const uint32_t token = blockIdx.x;
    const int32_t* const slots = a.slots + (uint64_t)token * a.topk;
    for (uint32_t j0 = 0; j0 < a.topk; j0 += 4) {
        float dot[4] = {}, w[4];
        int32_t slot[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            slot[u] = j0 + u < a.topk ? slots[j0 + u] : -1;
            if ((uint32_t)slot[u] >= used) slot[u] = -1;
            w[u] = slot[u] < 0 ? 0.0f : a.weights ? a.weights[(uint64_t)token * a.topk + j0 + u] : 1.0f;
        }
        for (uint32_t at = threadIdx.x * V; at < a.width; at += step) {
            const int64_t left = (int64_t)a.width - at;
            float d[V], v[4][V];
            load_elements<DT, V>(static_cast<const T*>(a.d_out) + token * a.d_stride + at, left, d);
            if (a.d_weights)
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (slot[u] >= 0) load_elements<DT, V>(static_cast<const T*>(a.rows) + slot[u] * a.row_stride + at, left, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (slot[u] >= 0) {
                    if (a.d_weights)
#pragma unroll
                        for (int i = 0; i < V; ++i) dot[u] = fmaf(d[i], v[u][i], dot[u]);
                    float scaled[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) scaled[i] = w[u] * d[i];
                    store_elements<DT, V>(static_cast<T*>(a.d_rows) + slot[u] * a.d_row_stride + at, left, scaled);
                }
        }
        if (a.d_weights) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float sum = wave_sum(dot[u]);
                if (lane_id() == 0) part[wave_in_block()][u] = sum;
            }
            __syncthreads();
            if (threadIdx.x < 4 && j0 + threadIdx.x < a.topk) {
                float sum = 0.0f;
                for (int i = 0; i < kCombineWaves; ++i) sum += part[i][threadIdx.x];
                a.d_weights[(uint64_t)token * a.topk + j0 + threadIdx.x] = sum;
            }
            __syncthreads();
        }
    }
}

bool known(int dtype) { return dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32; }

}  // namespace
}  // namespace mint

using namespace mint;

extern "C" int mint_combine(const void* rows, int64_t row_stride, uint64_t n_rows, const void* slots, const void* weights,
                            uint64_t tokens, uint32_t topk, uint32_t width, void* out, int64_t out_stride, int dtype, void* stream) {
    if (!known(dtype) || topk < 1) return MINT_ERR_ARG;
    if (tokens > 0x7FFFFFFFull / topk || n_rows > 0x7FFFFFFFull || width > 0x7FFFFFFFu - 4096u) return MINT_ERR_TOO_LARGE;
    if (tokens == 0 || width == 0) return MINT_OK;
    if (!slots || !out || (n_rows && !rows)) return MINT_ERR_ARG;
    const uint32_t chunks = (uint32_t)ceil_div(width, 64 * kCombineV);
    const uint64_t blocks = ceil_div(tokens * chunks, kCombineWaves);
    if (blocks > 0x7FFFFFFFull / (64 * kCombineWaves)) return MINT_ERR_TOO_LARGE;
    const CombineArgs a = {rows, static_cast<const int32_t*>(slots), static_cast<const float*>(weights), out, row_stride, out_stride,
                           (uint32_t)n_rows, (uint32_t)tokens, topk, width, chunks};
    const auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case MINT_F16: return Launch<&combine_kernel<DT_F16>>::go((uint32_t)blocks, 64 * kCombineWaves, 0, s, a);
        case MINT_BF16: return Launch<&combine_kernel<DT_BF16>>::go((uint32_t)blocks, 64 * kCombineWaves, 0, s, a);
        default: return Launch<&combine_kernel<DT_F32>>::go((uint32_t)blocks, 64 * kCombineWaves, 0, s, a);
    }
}

extern "C" int mint_combine_grad(const void* d_out, int64_t d_stride, const void* rows, int64_t row_stride, uint64_t n_rows,
                                 const void* slots, const void* weights, const void* rows_used, uint64_t tokens, uint32_t topk,
                                 uint32_t width, void* d_rows, int64_t d_row_stride, void* d_weights, int dtype, void* stream) {
    if (!known(dtype) || topk < 1) return MINT_ERR_ARG;
    if (tokens > 0x7FFFFFFFull / topk || n_rows > 0x7FFFFFFFull || width > 0x7FFFFFFFu - 8192u) return MINT_ERR_TOO_LARGE;
    if (tokens + kClearing > 0x7FFFFFFFull / (64 * kCombineWaves)) return MINT_ERR_TOO_LARGE;
    if (tokens + n_rows == 0) return MINT_OK;
    if ((tokens && (!slots || !d_out)) || (n_rows && (!d_rows || !rows_used || (d_weights && !rows)))) return MINT_ERR_ARG;
    const CombineGradArgs a = {d_out, rows, static_cast<const int32_t*>(slots), static_cast<const int32_t*>(rows_used),
                               static_cast<const float*>(weights), d_rows, static_cast<float*>(d_weights), d_stride, row_stride, d_row_stride,
                               (uint32_t)n_rows, (uint32_t)tokens, topk, width};
    const auto s = static_cast<hipStream_t>(stream);
    const uint32_t blocks = (uint32_t)(tokens + (n_rows ? kClearing : 0));
    switch (dtype) {
        case MINT_F16: return Launch<&combine_grad_kernel<DT_F16>>::go(blocks, 64 * kCombineWaves, 0, s, a);
        case MINT_BF16: return Launch<&combine_grad_kernel<DT_BF16>>::go(blocks, 64 * kCombineWaves, 0, s, a);
        default: return Launch<&combine_grad_kernel<DT_F32>>::go(blocks, 64 * kCombineWaves, 0, s, a);
    }
}
