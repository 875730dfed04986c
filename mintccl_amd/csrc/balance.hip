// The loss that keeps experts in balance, with their counts, and its gradient.
//
//   p_te = softmax(x_t)_e, or sigmoid(x_te) / sum_i sigmoid(x_ti)          shares of a token's scores
//   c_se: how many choices of sequence s name expert e     n_s: its tokens that have an expert left     S: sequences that have such a token
//   f_se = E c_se / (k n_s)     P_se = sum over tokens of p_te / n_s
//   loss = 1 / S sum_s sum_e f_se P_se + z / N sum_t lse(x_t)^2            N = sum n_s
//
// The choice has no gradient, so with a_se = f_se / (S n_s) and <p, a> over a token's experts:
//
//   softmax   d x_te = p_te (a_se - <p, a>)         sigmoid   d x_te = p_te (1 - sigmoid(x_te)) (a_se - <p, a>)
//   z         d x_te += 2 z / N lse_t softmax(x_t)_e
//
// A logit of -inf masks its expert (p 0, gradient 0); a token with no expert left, or in no sequence, counts nowhere and has a gradient of
// zeros.  Tokens go by in tiles that do not reach over sequences; a tile's sums are left in memory and added up in the tiles' order, so
// the bits repeat.
#include "activations.hpp"

#include <algorithm>
#include <cfloat>

namespace mint {
namespace {

constexpr uint32_t kMostExperts = 1024;
constexpr int kWaves = 4;                       // wavefronts of a thread block

struct BalanceArgs {
    const void* logits;
    const int32_t *chosen, *offsets;            // offsets 0: one sequence of all tokens
    int64_t row_stride;
    uint32_t tokens, experts, topk, sequences, tile, tiles;      // tokens of a tile; tiles at most
    uint32_t sigmoid;
    float z;
    // what a tile leaves: shares' sums (tiles, experts), counts (tiles, experts), {squares' sum, tokens} (tiles, 2)
    float *shares, *square;
    uint32_t *counts;
    // ... a sequence: {term of the loss, squares' sum} by block of experts (sequences, blocks), then its tokens (sequences)
    uint64_t* terms;
    uint32_t* arrived;
    int32_t *out_counts, *out_tokens;
    float *out_shares, *out_loss;
};

// Where tile `t` of `tile` tokens is.  With offsets the tokens before the first sequence and those behind the last one count as a sequence each: v = 0, 1 ... S,
// S + 1 begin at tokens b_v, and v has the tiles from b_v / tile + v on, whole numbers, which is room enough for it, and is found by a search.  (Tiles that
// a sequence has room for and does not need are nobody's.)  Offsets are device data: whatever they say, tokens and tiles stay inside.
struct Span {
    uint32_t sequence, begin, end;              // tokens [begin, end)
    bool found, outside;                        // outside: tokens of no sequence
};
__device__ __forceinline__ uint32_t begin_of(const BalanceArgs& a, uint32_t v) {
    return v == 0 ? 0u : v > a.sequences + 1 ? a.tokens : min((uint32_t)max(a.offsets[v - 1], 0), a.tokens);
}
// the last v of `n` of which the first ones, v = 0 among them, are `below`: 64 of them at a time
template <typename F>
__device__ __forceinline__ uint32_t last_below(uint32_t n, const F& below) {
    const uint32_t lane = lane_id();
    uint32_t v = 0;
    for (uint32_t step = 0; step != 1;) {
        step = (n + 63) / 64;
        const uint32_t at = min(lane * step, n - 1);
        const uint64_t found = __ballot(lane * step < n && below(v + at));
        const uint32_t skip = (found ? (uint32_t)__popcll(found) - 1u : 0u) * step;
        v += skip;
        n = min(step, n - skip);
    }
    return v;
}
__device__ __forceinline__ Span find_span(const BalanceArgs& a, uint32_t t) {
    if (!a.offsets) return {0, min(t * a.tile, a.tokens), min(t * a.tile + a.tile, a.tokens), t * a.tile < a.tokens, false};
    const uint32_t v = last_below(a.sequences + 2, [&](uint32_t u) MINT_INLINE_LAMBDA { return begin_of(a, u) / a.tile + u <= t; });
    const uint32_t begin = begin_of(a, v), end = max(begin, begin_of(a, v + 1)), nth = t - (begin / a.tile + v);
    const bool found = nth < (end - begin + a.tile - 1) / a.tile, outside = v == 0 || v > a.sequences;
    const uint32_t from = found ? begin + nth * a.tile : 0u;
    return {v - 1, from, found ? min(from + a.tile, end) : 0u, found, outside};
}
// the tiles of sequence s
__device__ __forceinline__ void tiles_of_sequence(const BalanceArgs& a, uint32_t s, uint32_t& first, uint32_t& end) {
    first = 0;
    end = a.tiles;
    if (!a.offsets) return;
    const uint32_t begin = begin_of(a, s + 1), tokens = max(begin, begin_of(a, s + 2)) - begin;
    first = min(begin / a.tile + s + 1, a.tiles);
    end = min(first + (tokens + a.tile - 1) / a.tile, a.tiles);
}

// Of U tokens' logits (V consecutive ones of a lane), side by side so that their steps across lanes overlap: the shares, and what the gradient needs.
template <int V, int U>
struct Tokens {
    float p[U][V];               // scores divided by their sum; zeros where the token counts nowhere
    float rest[U][V];            // sigmoids: 1 - score
    float soft[U][V];            // sigmoids, where z is not 0: the softmax
    float lse[U];                // where z is not 0: the log of the exponentials' sum
    bool there[U];
    uint32_t vanished = 0;       // sigmoids: a bit for each token whose all may have left the range; it has no shares
    // `in` of the U there are tokens, whose logits have been moved down by `up`
    __device__ __forceinline__ Tokens(const float (&x)[U][V], const float (&up)[U], const bool (&in)[U], uint32_t first, uint32_t experts, bool use_sigmoid,
                                      bool wants_lse) {
        float top[U], sum[U], scores[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            bool any = false;
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool counts = first + i < experts && x[u][i] != -INFINITY;
                any |= counts;                                // (a NaN is a number that is there, and makes the token's shares NaN)
                m = counts ? fmaxf(m, x[u][i]) : m;
            }
            there[u] = in[u] && __ballot(any) != 0;
            top[u] = m;
        }
        if (!use_sigmoid || wants_lse) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                top[u] = wave_max(top[u]);
                top[u] = top[u] == -INFINITY ? 0.0f : top[u];
                sum[u] = 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float e = first + i < experts && x[u][i] != -INFINITY ? exponential(x[u][i] - top[u]) : 0.0f;
                    soft[u][i] = e;
                    sum[u] += e;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                sum[u] = wave_sum(sum[u]);
                lse[u] = there[u] && wants_lse ? top[u] + logf(sum[u]) + up[u] : 0.0f;
                const float r = there[u] ? 1.0f / sum[u] : 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) soft[u][i] *= r;
            }
        }
        if (use_sigmoid) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                scores[u] = 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const bool counts = first + i < experts && x[u][i] != -INFINITY;
                    const float e = fminf(exponential(-x[u][i]), FLT_MAX), s = reciprocal(1.0f + e);
                    p[u][i] = counts ? x[u][i] != x[u][i] ? x[u][i] : s : 0.0f;
                    rest[u][i] = e * s;
                    scores[u] += p[u][i];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                scores[u] = wave_sum(scores[u]);
                const bool far = there[u] && scores[u] < 0x1p-60f;
                vanished |= far ? 1u << u : 0u;
                const float r = there[u] && !far ? 1.0f / scores[u] : 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) p[u][i] *= r;
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) p[u][i] = soft[u][i];
        }
    }
};
// Sigmoids far below 1 are e^x to the last bit: where all of a token's are, their quotients are those of its logits moved to -20 and less.  By how much comes
// back.  (Seldom: such tokens are done behind the others, one by one.)
template <int V>
__device__ __forceinline__ float move_up(float (&x)[V], uint32_t first, uint32_t experts) {
    float top = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < V; ++i) top = first + i < experts ? fmaxf(top, x[i]) : top;
    const float up = wave_max(top) + 20.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] -= up;
    return up;
}
constexpr int tokens_at_once(int v) { return v <= 4 ? 4 : v <= 8 ? 2 : 1; }

struct Sums {
    float share, squares;
    uint32_t count, tokens;
};
// an expert's counts and shares of a sequence, and its term of the loss
__device__ __forceinline__ float store_expert(const BalanceArgs& a, uint32_t s, uint32_t e, const Sums& v) {
    const float some = (float)max(v.tokens, 1u), share = v.share / some;
    a.out_counts[(uint64_t)s * a.experts + e] = (int32_t)v.count;
    a.out_shares[(uint64_t)s * a.experts + e] = share;
    return (float)v.count * (float)a.experts / ((float)a.topk * some) * share;
}
__device__ __forceinline__ float loss_of(const BalanceArgs& a, float terms, float squares, uint32_t sequences, uint32_t tokens) {
    return terms / (float)max(sequences, 1u) + (a.z != 0.0f ? a.z * (squares / (float)max(tokens, 1u)) : 0.0f);
}

// A wavefront has every kWaves-th token of the tile, a lane V consecutive experts.  ALONE: the tile has all tokens, and the results are made here.
// Bound by its vector instructions and their steps across lanes: 65536 tokens of 256 experts, sigmoids: 19.6 us, of which the 67 MB are 12 (one token at a
// time, the library's exponential: 37).
template <int DT, int V, bool ALONE>
__global__ void __launch_bounds__(64 * kWaves) balance_tiles_kernel(BalanceArgs a) {
    using T = typename Elem<DT>::type;
    constexpr int U = tokens_at_once(V);
    __shared__ float shares[kWaves][64 * V];
    __shared__ uint32_t counts[kMostExperts], there[kWaves];
    __shared__ float square[kWaves];
    const Span span = find_span(a, blockIdx.x);
    if (!ALONE && blockIdx.x == 0 && threadIdx.x == 0) *a.arrived = 0u;
    if (!ALONE && (!span.found || span.outside)) {           // (nobody's: but offsets that descend may have it read)
        for (uint32_t e = threadIdx.x; e < a.experts; e += 64 * kWaves) {
            a.shares[(uint64_t)blockIdx.x * a.experts + e] = 0.0f;
            a.counts[(uint64_t)blockIdx.x * a.experts + e] = 0u;
        }
        if (threadIdx.x < 2) a.square[blockIdx.x * 2 + threadIdx.x] = 0.0f;
        return;
    }
    for (uint32_t e = threadIdx.x; e < a.experts; e += 64 * kWaves) counts[e] = 0u;
    __syncthreads();
    const uint32_t lane = lane_id(), wave = wave_in_block(), first = lane * V;
    // choices: whole numbers, whose sum has no order
    for (uint64_t i = (uint64_t)span.begin * a.topk + threadIdx.x; i < (uint64_t)span.end * a.topk; i += 64 * kWaves) {
        const uint32_t e = (uint32_t)a.chosen[i];
        if (e < a.experts) atomicAdd(counts + e, 1u);
    }
    float sum[V], squares = 0.0f;
    uint32_t n = 0, vanished = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    for (uint32_t t0 = span.begin + wave; t0 < span.end; t0 += kWaves * U) {
        float x[U][V];
        const float up[U] = {};
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t t = t0 + u * kWaves;
            in[u] = t < span.end;
            load_elements<DT, V>(static_cast<const T*>(a.logits) + (int64_t)(in[u] ? t : t0) * a.row_stride + first, (int64_t)a.experts - first, x[u]);
        }
        const Tokens<V, U> tokens(x, up, in, first, a.experts, a.sigmoid, a.z != 0.0f);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] += in[u] ? tokens.p[u][i] : 0.0f;
            if (a.z != 0.0f) squares = fmaf(tokens.lse[u], tokens.lse[u], squares);
            n += tokens.there[u];
        }
        vanished |= tokens.vanished;
    }
    for (uint32_t t = vanished ? span.begin + wave : span.end; t < span.end; t += kWaves) {
        float x[1][V], up[1] = {};
        const bool in[1] = {true};
        load_elements<DT, V>(static_cast<const T*>(a.logits) + (int64_t)t * a.row_stride + first, (int64_t)a.experts - first, x[0]);
        if (!Tokens<V, 1>(x, up, in, first, a.experts, true, false).vanished) continue;
        up[0] = move_up(x[0], first, a.experts);
        const Tokens<V, 1> token(x, up, in, first, a.experts, true, false);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += token.p[0][i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) shares[wave][first + i] = sum[i];
    if (lane == 0) {
        square[wave] = squares;
        there[wave] = n;
    }
    __syncthreads();
    Sums all = {0.0f, 0.0f, 0u, 0u};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        all.squares += square[w];
        all.tokens += there[w];
    }
    float terms = 0.0f;
    for (uint32_t e = threadIdx.x; e < a.experts; e += 64 * kWaves) {
        all.share = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all.share += shares[w][e];
        all.count = counts[e];
        if (ALONE) {
            terms += store_expert(a, 0, e, all);
        } else {
            a.shares[(uint64_t)blockIdx.x * a.experts + e] = all.share;
            a.counts[(uint64_t)blockIdx.x * a.experts + e] = all.count;
        }
    }
    if (ALONE) {
        terms = wave_sum(terms);
        __syncthreads();                                     // (the squares have been read)
        if (lane == 0) square[wave] = terms;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (ALONE) {
            terms = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) terms += square[w];
            a.out_tokens[0] = (int32_t)all.tokens;
            *a.out_loss = loss_of(a, terms, all.squares, 1u, all.tokens);
        } else {
            a.square[blockIdx.x * 2] = all.squares;
            a.square[blockIdx.x * 2 + 1] = __uint_as_float(all.tokens);
        }
    }
}

// A thread block has 16 experts of a sequence, 16 lanes every kSlots-th tile's sums of them.  The last block that is done adds the sequences' terms
// up, in their order.  1024 tiles of 256 experts: 11 us, the wait for two rounds of loads and
// the last block's turn (64 experts to a thread block, a quarter of the lanes: 27).
constexpr uint32_t kSlots = 64, kOfBlock = 16;
__global__ void __launch_bounds__(kSlots * kOfBlock) balance_join_kernel(BalanceArgs a) {
    __shared__ Sums part[kSlots][kOfBlock];
    __shared__ bool last;
    const uint32_t blocks = (a.experts + kOfBlock - 1) / kOfBlock, s = blockIdx.x / blocks, block = blockIdx.x % blocks;
    const uint32_t lane = threadIdx.x % kOfBlock, slot = threadIdx.x / kOfBlock, e = block * kOfBlock + lane, from = min(e, a.experts - 1);
    uint32_t first, end;
    tiles_of_sequence(a, s, first, end);
    Sums sum = {0.0f, 0.0f, 0u, 0u};
    for (uint32_t t0 = first + slot; t0 < end; t0 += kSlots * 8) {
        Sums v[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) {
            const uint64_t t = min(t0 + u * kSlots, end - 1);
            v[u] = {a.shares[t * a.experts + from], a.square[t * 2], a.counts[t * a.experts + from], __float_as_uint(a.square[t * 2 + 1])};
        }
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u)
            if (t0 + u * kSlots < end) sum = {sum.share + v[u].share, sum.squares + v[u].squares, sum.count + v[u].count, sum.tokens + v[u].tokens};
    }
    part[slot][lane] = sum;
    // 64 slots, eight at a time
    for (uint32_t step = 8; step <= 64; step *= 8) {
        __syncthreads();
        const uint32_t each = kSlots / step;                 // 8, then 1
        if (slot < each) {
            sum = part[slot * step][lane];
#pragma unroll
            for (uint32_t u = 1; u < 8; ++u) {
                const Sums v = part[slot * step + u * (step / 8)][lane];
                sum = {sum.share + v.share, sum.squares + v.squares, sum.count + v.count, sum.tokens + v.tokens};
            }
            part[slot * step][lane] = sum;
        }
    }
    const uint32_t wave = wave_in_block();
    if (wave == 0) {
        // (the first 16 lanes have the block's experts)
        const bool mine = slot == 0 && e < a.experts;
        const float term = wave_sum(mine ? store_expert(a, s, e, sum) : 0.0f);
        if (lane_id() == 0) {
            if (block == 0) a.out_tokens[s] = (int32_t)sum.tokens;
            // (read by another block of this launch: past the caches that are not shared)
            st64_agent(a.terms + blockIdx.x, (uint64_t)__float_as_uint(sum.squares) << 32 | __float_as_uint(term));
            if (block == 0) st64_agent(a.terms + gridDim.x + s, sum.tokens);
            wait_stores_visible();
            last = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    compiler_fence();
    // (threads have sequences in turn, lanes add theirs up, then wavefronts: a fixed order too)
    Sums all = {0.0f, 0.0f, 0u, 0u};
    for (uint32_t i = threadIdx.x; i < a.sequences; i += kSlots * kOfBlock) {
        const uint32_t k = (uint32_t)ld64_agent(a.terms + gridDim.x + i);
        all.count += k != 0;
        all.tokens += k;
        float of_one = 0.0f;
        for (uint32_t b = 0; b < blocks; ++b) of_one += __uint_as_float((uint32_t)ld64_agent(a.terms + (uint64_t)i * blocks + b));
        all.share += of_one;
        all.squares += __uint_as_float((uint32_t)(ld64_agent(a.terms + (uint64_t)i * blocks) >> 32));
    }
    all.share = wave_sum(all.share);
    all.squares = wave_sum(all.squares);
    all.count = (uint32_t)__builtin_amdgcn_readlane((int)sum_below(all.count), 63);
    all.tokens = (uint32_t)__builtin_amdgcn_readlane((int)sum_below(all.tokens), 63);
    if (lane_id() == 0) part[wave][0] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kSlots * kOfBlock / 64; ++w)
            all = {all.share + part[w][0].share, all.squares + part[w][0].squares, all.count + part[w][0].count, all.tokens + part[w][0].tokens};
        *a.out_loss = loss_of(a, all.share, all.squares, all.count, all.tokens);
    }
}

struct BalanceGradArgs {
    BalanceArgs f;
    const float* d_loss;
    const int32_t *counts, *there;              // (sequences, experts), (sequences)
    const void* add;                            // a gradient that is added, or 0
    void* d_logits;
    int64_t add_stride, d_stride;
};
// Tiles lie side by side here, whatever the offsets say, and a token belongs to the last of the sequences that begin at it or before it: so every row is written once, by
// one thread block, also where the offsets descend; and there are no more thread blocks where there are more sequences, whose tokens each of them adds up, eight loads
// of a thread at a time (66000 tokens of 20 experts in 65535 sequences 39 us; a thread block for each of them 1180).  65536 tokens of 256 experts,
// sigmoids: 30 us for 134 MB (4.5 TB/s; one token at a time, the library's exponential: 56).
template <int DT, int V>
__global__ void __launch_bounds__(64 * kWaves) balance_grad_kernel(BalanceGradArgs a) {
    using T = typename Elem<DT>::type;
    constexpr int U = tokens_at_once(V);
    const BalanceArgs& f = a.f;
    const uint32_t lane = lane_id(), first = lane * V;
    const int64_t left = (int64_t)f.experts - first;
    __shared__ uint32_t some_of[kWaves], every_of[kWaves];
    // 64 sequences' beginnings, from `window` on, one to a lane
    uint32_t window = 0, begins = f.offsets ? begin_of(f, lane) : 0u;
    // sequences that have a token, and all tokens
    uint32_t some = 0, every = 0;
    for (uint32_t s0 = threadIdx.x; s0 < f.sequences; s0 += 64 * kWaves * 8) {
        uint32_t n[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) n[k] = (uint32_t)max(a.there[min(s0 + k * 64 * kWaves, f.sequences - 1)], 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            n[k] = s0 + k * 64 * kWaves < f.sequences ? n[k] : 0u;
            some += n[k] != 0;
            every += n[k];
        }
    }
    some = sum_below(some);
    every = sum_below(every);
    if (lane == 63) {
        some_of[wave_in_block()] = some;
        every_of[wave_in_block()] = every;
    }
    __syncthreads();
    some = every = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        some += some_of[w];
        every += every_of[w];
    }
    some = max(some, 1u);
    every = max(every, 1u);
    const float d = *a.d_loss, by_z = f.z != 0.0f ? 2.0f * f.z * d / (float)every : 0.0f;
    const uint32_t begin = blockIdx.x * f.tile, end = min(begin + f.tile, f.tokens);
    // a token's sequence, 1 and on (0, and behind the last one: none), and where the next one begins
    const auto sequence_of = [&](uint32_t t, uint32_t& next) MINT_INLINE_LAMBDA {
        next = f.tokens;
        if (!f.offsets) return 1u;
        // the last lane whose beginning is not behind `t`
        uint64_t before = __ballot(begins <= t);
        if (!(before & 1ull) || before >> 63) {               // (there may be more in front of them, or behind)
            window = last_below(f.sequences + 2, [&](uint32_t u) MINT_INLINE_LAMBDA { return begin_of(f, u) <= t; });
            begins = begin_of(f, window + lane);
            before = __ballot(begins <= t);
        }
        const uint32_t nth = 63u - (uint32_t)__clzll(before | 1ull);
        // (behind the search lane 63's is behind `t` too, unless the offsets descend)
        next = nth == 63 ? t : (uint32_t)__builtin_amdgcn_readlane((int)begins, (int)nth + 1);
        return window + nth;
    };
    const auto load_logits = [&](uint32_t t0, auto& x, auto& in) MINT_INLINE_LAMBDA {
        constexpr int N = sizeof(in) / sizeof(in[0]);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint32_t t = t0 + u * kWaves;
            in[u] = t < end;
            const T* const row = static_cast<const T*>(f.logits) + (int64_t)(in[u] ? t : t0) * f.row_stride;
            // (one to a lane: the last one in the place of those behind it, since loads that some lanes have not are waited for one by one)
            if constexpr (V == 1) x[u][0] = Elem<DT>::load(*as_global(row + min(first, f.experts - 1)));
            else load_elements<DT, V>(row + first, left, x[u]);
        }
        if constexpr (V <= 2) __builtin_amdgcn_sched_barrier(0);      // (all of them, before the first is waited for)
    };
    // (clamped where it is one to a lane, as there)
    const auto count_of = [&](uint64_t sequence, int i) MINT_INLINE_LAMBDA {
        const int32_t* const row = a.counts + sequence * f.experts;
        return V == 1 ? (float)row[min(first, f.experts - 1)] : first + i < f.experts ? (float)row[first + i] : 0.0f;
    };
    // what the loss's gradient is by an expert's mean share
    const auto load_of = [&](float count, float n) MINT_INLINE_LAMBDA { return d * (float)f.experts / ((float)f.topk * n) / ((float)some * n) * count; };
    // N tokens, of one sequence (W 1) or each of its own; those that are not `inside` count nowhere.  Whose sigmoids have vanished are left out, and come back,
    // unless their logits have been `moved`.
    const auto gradients = [&](uint32_t t0, const auto& x, const auto& up, bool moved, const auto& in, const auto& inside, const auto& often) MINT_INLINE_LAMBDA {
        constexpr int N = sizeof(in) / sizeof(in[0]), W = sizeof(often) / sizeof(often[0]);
        float mean[N];
        const Tokens<V, N> tokens(x, up, inside, first, f.experts, f.sigmoid, f.z != 0.0f);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            mean[u] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) mean[u] = fmaf(tokens.p[u][i], often[u % W][i], mean[u]);
        }
#pragma unroll
        for (int u = 0; u < N; ++u) mean[u] = wave_sum(mean[u]);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint32_t t = t0 + u * kWaves;
            if (!in[u] || left <= 0 || (!moved && tokens.vanished >> u & 1u)) continue;
            float more[V];
#pragma unroll
            for (int i = 0; i < V; ++i) more[i] = 0.0f;
            if (a.add) load_elements<DT, V>(static_cast<const T*>(a.add) + (int64_t)t * a.add_stride + first, left, more);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float dx = tokens.p[u][i] * (often[u % W][i] - mean[u]);
                if (f.sigmoid) dx *= tokens.rest[u][i];
                if (f.z != 0.0f) dx = fmaf(by_z * tokens.lse[u], tokens.soft[u][i], dx);
                more[i] += x[u][i] == -INFINITY || !tokens.there[u] ? 0.0f : dx;
            }
            store_elements<DT, V>(static_cast<T*>(a.d_logits) + (int64_t)t * a.d_stride + first, left, more);
        }
        return tokens.vanished;
    };
    uint32_t next, vanished = 0;
    const uint32_t v = sequence_of(begin, next);
    if (next < end) {
        // Tokens of several sequences: each has its own load, all of them on their way with the logits.  (Two at a time: four take registers that
        // the tokens below then have not either, 2^20 of 128 experts 283 us for 261.)
        constexpr int N = U < 2 ? U : 2;
        for (uint32_t t0 = begin + wave_in_block(); t0 < end; t0 += kWaves * N) {
            float x[N][V], often[N][V], n[N];
            const float up[N] = {};
            bool in[N], inside[N];
            load_logits(t0, x, in);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const uint32_t of = sequence_of(in[u] ? t0 + u * kWaves : t0, next);
                const uint64_t at = min(max(of, 1u), f.sequences) - 1;
                inside[u] = in[u] && of != 0 && of <= f.sequences;
                n[u] = (float)max(a.there[at], 1);
#pragma unroll
                for (int i = 0; i < V; ++i) often[u][i] = count_of(at, i);
            }
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) often[u][i] = load_of(often[u][i], n[u]);
            vanished |= gradients(t0, x, up, false, in, inside, often);
        }
    } else if (v == 0 || v > f.sequences) {                   // tokens of no sequence
        for (uint32_t t = begin + wave_in_block(); t < end; t += kWaves) {
            float none[V] = {};
            if (a.add) load_elements<DT, V>(static_cast<const T*>(a.add) + (int64_t)t * a.add_stride + first, left, none);
            if (left > 0) store_elements<DT, V>(static_cast<T*>(a.d_logits) + (int64_t)t * a.d_stride + first, left, none);
        }
    } else {
        const float n = (float)max(a.there[v - 1], 1);
        float often[1][V];
#pragma unroll
        for (int i = 0; i < V; ++i) often[0][i] = load_of(count_of(v - 1, i), n);
        const float up[U] = {};
        for (uint32_t t0 = begin + wave_in_block(); t0 < end; t0 += kWaves * U) {
            float x[U][V];
            bool in[U];
            load_logits(t0, x, in);
            vanished |= gradients(t0, x, up, false, in, in, often);
        }
    }
    for (uint32_t t = vanished ? begin + wave_in_block() : end; t < end; t += kWaves) {
        float x[1][V], often[1][V], up[1] = {};
        bool in[1];
        const uint32_t of = sequence_of(t, next);
        if (of == 0 || of > f.sequences) continue;
        load_logits(t, x, in);
        if (!Tokens<V, 1>(x, up, in, first, f.experts, true, false).vanished) continue;
        const float n = (float)max(a.there[of - 1], 1);
#pragma unroll
        for (int i = 0; i < V; ++i) often[0][i] = load_of(count_of(of - 1, i), n);
        up[0] = move_up(x[0], first, f.experts);
        gradients(t, x, up, true, in, in, often);
    }
}

uint32_t values_per_lane(uint32_t experts) {
    uint32_t v = 1;
    while (v * 64 < experts) v *= 2;
    return v;
}
template <int DT, int V>
int go_tiles(const BalanceArgs& a, hipStream_t s) {
    if (!a.shares) return Launch<&balance_tiles_kernel<DT, V, true>>::go(1, 64 * kWaves, 0, s, a);
    return Launch<&balance_tiles_kernel<DT, V, false>>::go(a.tiles, 64 * kWaves, 0, s, a);
}
template <int DT, int V>
int go_grad(const BalanceGradArgs& a, hipStream_t s) {
    return Launch<&balance_grad_kernel<DT, V>>::go((uint32_t)ceil_div(a.f.tokens, a.f.tile), 64 * kWaves, 0, s, a);
}
#define MINT_BY_VALUES(GO, DT)                     \
    switch (values_per_lane(op->experts)) {        \
        case 1: return GO<DT, 1>(a, s);            \
        case 2: return GO<DT, 2>(a, s);            \
        case 4: return GO<DT, 4>(a, s);            \
        case 8: return GO<DT, 8>(a, s);            \
        default: return GO<DT, 16>(a, s);          \
    }
#define MINT_BY_TYPES(GO)                                  \
    switch (op->dtype) {                                   \
        case MINT_F16: MINT_BY_VALUES(GO, DT_F16)          \
        case MINT_BF16: MINT_BY_VALUES(GO, DT_BF16)        \
        default: MINT_BY_VALUES(GO, DT_F32)                \
    }

bool known(int dtype) { return dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32; }
uint32_t sequences_of(const mint_balance_op& op) { return op.offsets ? (uint32_t)op.sequences : 1u; }
// Tokens of a tile: so that there are about as many tiles as fill the device.
uint32_t tile_of(uint64_t tokens) { return (uint32_t)std::min<uint64_t>(256, std::max<uint64_t>(16, ceil_div(tokens, 1024))); }
// So few that one thread block takes less than two launches.
bool alone(const mint_balance_op& op) { return !op.offsets && op.tokens <= 64; }
constexpr uint64_t kMostSequences = 0xFFFF;      // (with 64 thread blocks each of 1024 threads: a launch has fewer than 2^32)
// tiles, those that are nobody's among them
uint64_t tiles_of(const mint_balance_op& op) {
    const uint64_t tile = tile_of(op.tokens);
    return op.offsets ? op.tokens / tile + op.sequences + 2 : ceil_div(op.tokens, tile);
}
int balance_checks(const mint_balance_op* op) {
    if (!op || !known(op->dtype) || (op->score != MINT_SCORE_SOFTMAX && op->score != MINT_SCORE_SIGMOID)) return MINT_ERR_ARG;
    if (op->experts < 1 || op->experts > kMostExperts || op->topk < 1 || op->topk > kMostExperts) return MINT_ERR_ARG;
    if (op->tokens > 0x7FFFFFFFull / op->topk || (op->offsets && op->sequences > kMostSequences)) return MINT_ERR_TOO_LARGE;
    if (op->offsets && op->sequences == 0) return MINT_ERR_ARG;
    if (op->tokens && (!op->logits || !op->chosen)) return MINT_ERR_ARG;
    return MINT_OK;
}
BalanceArgs balance_args(const mint_balance_op& op) {
    BalanceArgs a = {};
    a.logits = reinterpret_cast<const void*>(op.logits);
    a.chosen = reinterpret_cast<const int32_t*>(op.chosen);
    a.offsets = reinterpret_cast<const int32_t*>(op.offsets);
    a.row_stride = op.row_stride;
    a.tokens = (uint32_t)op.tokens;
    a.experts = op.experts;
    a.topk = op.topk;
    a.sequences = sequences_of(op);
    a.tile = tile_of(op.tokens);
    a.tiles = (uint32_t)tiles_of(op);
    a.sigmoid = op.score == MINT_SCORE_SIGMOID;
    a.z = op.z;
    return a;
}
// shares, counts, squares of the tiles; terms and tokens of the sequences; the count of blocks that are done
struct BalanceRoom {
    uint64_t terms, shares, counts, square, arrived, bytes;
    explicit BalanceRoom(const mint_balance_op& op) {
        const uint64_t tiles = tiles_of(op), s = sequences_of(op), blocks = ceil_div(op.experts, kOfBlock);
        terms = 0;
        shares = terms + s * (blocks + 1) * 8;
        counts = shares + tiles * op.experts * 4;
        square = counts + tiles * op.experts * 4;
        arrived = square + tiles * 8;
        bytes = alone(op) ? 0 : arrived + 4;
    }
};

}  // namespace
}  // namespace mint

using namespace mint;

extern "C" size_t mint_balance_workspace(const mint_balance_op* op) { return balance_checks(op) == MINT_OK ? BalanceRoom(*op).bytes : 0; }

extern "C" int mint_balance(const mint_balance_op* op, uint64_t loss, uint64_t counts, uint64_t shares, uint64_t there, void* workspace,
                            size_t workspace_bytes, void* stream) {
    if (const int err = balance_checks(op)) return err;
    if (!loss || !counts || !shares || !there) return MINT_ERR_ARG;
    const BalanceRoom room(*op);
    if (room.bytes && (!workspace || workspace_bytes < room.bytes)) return MINT_ERR_STAGING;
    if (room.bytes && !aligned_to(workspace, 8)) return MINT_ERR_ALIGN;
    BalanceArgs a = balance_args(*op);
    a.out_counts = reinterpret_cast<int32_t*>(counts);
    a.out_tokens = reinterpret_cast<int32_t*>(there);
    a.out_shares = reinterpret_cast<float*>(shares);
    a.out_loss = reinterpret_cast<float*>(loss);
    const auto s = static_cast<hipStream_t>(stream);
    const auto tiles = [&]() -> int { MINT_BY_TYPES(go_tiles) };
    if (alone(*op)) {
        a.tile = 64;
        return tiles();
    }
    auto* const at = static_cast<uint8_t*>(workspace);
    a.terms = reinterpret_cast<uint64_t*>(at + room.terms);
    a.shares = reinterpret_cast<float*>(at + room.shares);
    a.counts = reinterpret_cast<uint32_t*>(at + room.counts);
    a.square = reinterpret_cast<float*>(at + room.square);
    a.arrived = reinterpret_cast<uint32_t*>(at + room.arrived);
    const uint64_t blocks = a.sequences * ceil_div(a.experts, kOfBlock);
    const int err = tiles();
    if (err != MINT_OK) return err;
    return Launch<&balance_join_kernel>::go((uint32_t)blocks, kSlots * kOfBlock, 0, s, a);
}

extern "C" int mint_balance_grad(const mint_balance_op* op, uint64_t d_loss, uint64_t counts, uint64_t there, uint64_t add, int64_t add_stride,
                                 uint64_t d_logits, int64_t d_stride, void* stream) {
    if (const int err = balance_checks(op)) return err;
    if (op->tokens == 0) return MINT_OK;
    if (!d_loss || !counts || !there || !d_logits) return MINT_ERR_ARG;
    const BalanceGradArgs a = {balance_args(*op), reinterpret_cast<const float*>(d_loss), reinterpret_cast<const int32_t*>(counts),
                               reinterpret_cast<const int32_t*>(there), reinterpret_cast<const void*>(add), reinterpret_cast<void*>(d_logits), add_stride, d_stride};
    const auto s = static_cast<hipStream_t>(stream);
    MINT_BY_TYPES(go_grad)
}
