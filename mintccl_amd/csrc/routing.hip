// Routing of tokens to experts: the choice and its weights, their gradient, and the
// assignment of the chosen pairs to places in the experts' order.
//
//   s_i = exp(x_i) / sum_e exp(x_e)   or   1 / (1 + exp(-x_i))           scores of a token's logits x
//   key_i = x_i + b_i   or   s_i + b_i                                    what the choice goes by
//   chosen: the k largest keys, lowest expert first among equals, in the `kept` groups whose one or
//   two largest keys have the largest sum
//   w_j = scale * s_j [ / sum over the chosen ]
//
// A logit of -inf masks its expert; a token with fewer experts than k left has -1 and a weight of 0 in
// their places.  A NaN ranks above every number and makes the weights NaN that the formula says: the choice
// itself always names experts that exist.
#include "operators.hpp"

#include <algorithm>
#include <cfloat>

namespace mint {
namespace {

constexpr int kRouteWaves = 4;                  // tokens of a thread block, a wavefront for each

// Order-preserving unsigned numbers: 0 = not there (masked, or taken), every NaN the largest.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);        // (-0 is 0: they are equal)
    const uint32_t key = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
    return v != v ? 0xFFFFFFFFu : v == -INFINITY ? 0u : key;
}
__device__ __forceinline__ float number_of(uint32_t key) {
    return key == 0u ? -INFINITY : __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// The key of a group whose two largest keys are these (the second may be missing): of two that are there the sum is too, also where it is
// beyond 32 bits' range, as that of two masks of the type's lowest number.
__device__ __forceinline__ uint32_t sum_of_two(uint32_t best, uint32_t second) {
    if (second == 0u) return best;
    const float sum = number_of(best) + number_of(second);
    return order_of(sum == -INFINITY ? -FLT_MAX : sum);
}
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

struct RouteArgs {
    const void* logits;
    const float* bias;
    float* weights;
    int32_t* chosen;
    int64_t row_stride;
    uint32_t tokens, experts, topk, groups, kept, group_top;
    float scale;
    uint32_t sigmoid, renormalise;
};

// What LANES lanes have together: 16 (a row, whose lanes the additions' cross-lane operands reach in four steps) or all 64.
template <int LANES>
struct Lanes;
template <>
struct Lanes<64> {
    static __device__ __forceinline__ uint32_t max_of(uint32_t v) { return wave_max(v); }
    static __device__ __forceinline__ float max_of(float v) { return wave_max(v); }
    static __device__ __forceinline__ float sum_of(float v) { return wave_sum(v); }
    static __device__ __forceinline__ uint32_t first(bool p) { return __builtin_ctzll(__ballot(p)); }
};
template <>
struct Lanes<16> {
    template <typename F>
    static __device__ __forceinline__ float fold(float v, const F& join) {
        v = join(v, __uint_as_float(dpp<0xB1, 0xf>(__float_as_uint(v), 0u)));
        v = join(v, __uint_as_float(dpp<0x4E, 0xf>(__float_as_uint(v), 0u)));
        v = join(v, __uint_as_float(dpp<0x141, 0xf>(__float_as_uint(v), 0u)));
        return join(v, __uint_as_float(dpp<0x140, 0xf>(__float_as_uint(v), 0u)));
    }
    static __device__ __forceinline__ uint32_t max_of(uint32_t v) { return row_max(v); }
    static __device__ __forceinline__ float max_of(float v) { return fold(v, [](float a, float b) { return fmaxf(a, b); }); }
    static __device__ __forceinline__ float sum_of(float v) { return fold(v, [](float a, float b) { return a + b; }); }
    // the first of the row's lanes where p holds (one of them does)
    static __device__ __forceinline__ uint32_t first(bool p) {
        const uint32_t row = lane_id() & 48u;
        return row + (uint32_t)__builtin_ctz((uint32_t)(__ballot(p) >> row) | 0x10000u);
    }
};
// a group's two largest keys joined with those of the lanes that CTRL reaches
template <int CTRL>
__device__ __forceinline__ void join_best(uint32_t& best, uint32_t& second) {
    const uint32_t b = dpp<CTRL, 0xf>(best, 0u), s = dpp<CTRL, 0xf>(second, 0u);
    second = max(min(best, b), max(second, s));
    best = max(best, b);
}

// LANES lanes have a token, a lane V consecutive experts of it, so that among equal keys the lowest lane has the lowest expert.
// Bound by its vector instructions: a choice is the largest of the lanes' largest keys, taken k times, about 120 instructions each, and
// a lane's scores are 39 each, one behind the other (16 sigmoids 620).  With 16 lanes
// the steps between lanes are for four tokens at once: 65536 tokens, 256 experts in 8 groups, 8 chosen: 44 us (with 64 lanes
// and groups looked at one by one 104), of which the 71 MB that it reads and writes are 15.
template <int DT, int V, int LANES>
__global__ void __launch_bounds__(64 * kRouteWaves) route_kernel(RouteArgs a) {
    using T = typename Elem<DT>::type;
    using L = Lanes<LANES>;
    constexpr uint32_t TOKENS = 64 * kRouteWaves / LANES;
    __shared__ int32_t picked[TOKENS][LANES];
    const uint32_t mine = threadIdx.x / LANES, token = blockIdx.x * TOKENS + mine, lane = threadIdx.x % LANES, first = lane * V;
    const bool live = token < a.tokens;                      // (all lanes go along: they are reached by others)
    const T* const row = static_cast<const T*>(a.logits) + (int64_t)(live ? token : a.tokens - 1) * a.row_stride;
    float x[V], bias[V];
    load_elements<DT, V>(row + first, (int64_t)a.experts - first, x);
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = 0.0f;
    if (a.bias) load_elements<DT_F32, V>(a.bias + first, (int64_t)a.experts - first, bias);
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float s = a.sigmoid ? sigmoid(x[i]) : x[i];
        key[i] = first + i < a.experts && x[i] != -INFINITY ? order_of(s + bias[i]) : 0u;
    }
    if (a.groups > 1) {
        const uint32_t per = a.experts / a.groups, lanes = per / V;
        if (per % V == 0 && lanes <= 16 && (lanes & (lanes - 1)) == 0) {
            // a group is 1, 2, 4, 8 or 16 whole lanes: all groups at once
            uint32_t best = 0, second = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                second = max(second, min(best, key[i]));
                best = max(best, key[i]);
            }
            if (lanes > 1) join_best<0xB1>(best, second);
            if (lanes > 2) join_best<0x4E>(best, second);
            if (lanes > 4) join_best<0x141>(best, second);
            if (lanes > 8) join_best<0x140>(best, second);
            uint32_t of_group = a.group_top == 2 ? sum_of_two(best, second) : best;
            bool keep = false;
            for (uint32_t n = 0; n < a.kept; ++n) {
                const uint32_t top = L::max_of(of_group), holder = L::first(of_group == top) % LANES;
                if (top != 0u && lane / lanes == holder / lanes) {
                    keep = true;
                    of_group = 0u;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = keep ? key[i] : 0u;
        } else {
            // groups that end inside a lane: one by one, lane g % LANES keeps the key of group g
            constexpr int PER_LANE = 64 / LANES;
            uint32_t of_group[PER_LANE];
#pragma unroll
            for (int q = 0; q < PER_LANE; ++q) of_group[q] = 0;
            for (uint32_t g = 0; g < a.groups; ++g) {
                uint32_t best = 0, second = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const uint32_t k = first + i - g * per < per ? key[i] : 0u;
                    second = max(second, min(best, k));
                    best = max(best, k);
                }
                uint32_t top = L::max_of(best);
                const bool holds = lane == L::first(best == top) % LANES;
                const uint32_t next = L::max_of(holds ? second : best);
                if (a.group_top == 2) top = sum_of_two(top, next);
#pragma unroll
                for (int q = 0; q < PER_LANE; ++q) of_group[q] = q * LANES + lane == g ? top : of_group[q];
            }
            uint64_t keep = 0;
            for (uint32_t n = 0; n < a.kept; ++n) {
                uint32_t best = 0;
#pragma unroll
                for (int q = 0; q < PER_LANE; ++q) best = max(best, of_group[q]);
                const uint32_t top = L::max_of(best);
                // the lowest group with that key: by q first, then by lane
                bool done = top == 0u;
#pragma unroll
                for (int q = 0; q < PER_LANE; ++q) {
                    const bool here = !done && L::max_of(of_group[q]) == top;
                    const uint32_t holder = L::first(of_group[q] == top) % LANES;
                    if (here) {
                        keep |= 1ull << (q * LANES + holder);
                        if (lane == holder) of_group[q] = 0u;
                        done = true;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = keep >> min((first + i) / per, 63u) & 1u ? key[i] : 0u;
        }
    }
    if (lane < a.topk) picked[mine][lane] = -1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t j = 0; j < a.topk; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i]);
        const uint32_t top = L::max_of(best);
        const bool wins = top != 0u && lane == L::first(best == top) % LANES;
        const uint32_t taken = wins ? top : 1u;              // (1 is nobody's key)
        uint32_t at = 0;
        bool found = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool here = key[i] == taken && !found;
            found |= here;
            at = here ? i : at;
            key[i] = here ? 0u : key[i];
        }
        if (wins) picked[mine][j] = (int32_t)(first + at);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int32_t choice = lane < a.topk ? picked[mine][lane] : -1;
    const bool there = choice >= 0;
    const float l = there ? Elem<DT>::load(row[choice]) : -INFINITY;
    float s, total = 1.0f;
    if (a.sigmoid) {
        s = there ? sigmoid(l) : 0.0f;
        if (a.renormalise) total = L::sum_of(s);
    } else {
        // the largest logit of those in the sum: of the chosen, or of all
        float m = l;
        if (!a.renormalise) {
#pragma unroll
            for (int i = 0; i < V; ++i) m = first + i < a.experts ? fmaxf(m, x[i]) : m;
        }
        m = L::max_of(m);
        m = m == -INFINITY ? 0.0f : m;
        s = there ? expf(l - m) : 0.0f;
        float sum = s;
        if (!a.renormalise) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += first + i < a.experts ? expf(x[i] - m) : 0.0f;
        }
        total = L::sum_of(sum);
    }
    // (every chosen score may have vanished: then so have the weights)
    const float w = !there || total == 0.0f ? 0.0f : a.scale * (s / total);
    if (live && lane < a.topk) {
        a.weights[(uint64_t)token * a.topk + lane] = w;
        a.chosen[(uint64_t)token * a.topk + lane] = choice;
    }
}

// The logits' gradient from the weights' d, with w' = w / scale and p = softmax(x):
//   softmax, renormalised   scale w'_j (d_j - sum w' d)             0 where nothing was chosen
//   softmax                 scale p_i (d_i [chosen] - sum w' d)
//   sigmoid, renormalised   scale (d_j - sum w' d) s_j (1 - s_j) / sum s
//   sigmoid                 scale d_j s_j (1 - s_j)
// The scores are computed again from the logits: they cost less than they would to keep.  4099 tokens of 64 experts: 4.1 us, hardly
// more than a launch takes.
struct RouteGradArgs {
    const void* logits;
    const float* d_weights;
    const int32_t* chosen;
    void* d_logits;
    int64_t row_stride, d_stride;
    uint32_t tokens, experts, topk;
    float scale;
    uint32_t sigmoid, renormalise;
};
template <int DT, int V>
__global__ void __launch_bounds__(64 * kRouteWaves) route_grad_kernel(RouteGradArgs a) {
    using T = typename Elem<DT>::type;
    const uint32_t token = blockIdx.x * kRouteWaves + wave_in_block(), lane = lane_id(), first = lane * V;
    if (token >= a.tokens) return;
    const T* const row = static_cast<const T*>(a.logits) + (int64_t)token * a.row_stride;
    const int32_t mine = lane < a.topk ? a.chosen[(uint64_t)token * a.topk + lane] : -1;
    const bool there = mine >= 0 && (uint32_t)mine < a.experts;
    const float d = there ? a.d_weights[(uint64_t)token * a.topk + lane] : 0.0f;
    const float l = there ? Elem<DT>::load(row[mine]) : -INFINITY;
    float out[V], g = 0.0f;                                  // g: what the chosen logit's gradient has more than its others
    if (a.sigmoid) {
        const float e = expf(-fabsf(l));
        const float s = there ? sigmoid(l) : 0.0f, slope = there ? e / ((1.0f + e) * (1.0f + e)) : 0.0f;
        if (a.renormalise) {
            const float total = wave_sum(s), mean = wave_sum(there ? s * d : 0.0f);
            // (a slope is at most its score: the quotients stay in range however small the scores are)
            g = total == 0.0f ? 0.0f : a.scale * (d - mean / total) * (slope / total);
        } else {
            g = a.scale * d * slope;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = 0.0f;
    } else {
        float x[V], m = l;
        if (!a.renormalise) {
            load_elements<DT, V>(row + first, (int64_t)a.experts - first, x);
#pragma unroll
            for (int i = 0; i < V; ++i) m = first + i < a.experts ? fmaxf(m, x[i]) : m;
        }
        m = wave_max(m);
        m = m == -INFINITY ? 0.0f : m;
        const float s = there ? expf(l - m) : 0.0f;
        float sum = s;
        if (!a.renormalise) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                out[i] = first + i < a.experts ? expf(x[i] - m) : 0.0f;
                sum += out[i];
            }
        }
        const float total = wave_sum(sum);
        const float w = total == 0.0f ? 0.0f : s / total, mean = wave_sum(there ? w * d : 0.0f);
        g = a.scale * w * (a.renormalise ? d - mean : d);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = a.renormalise || total == 0.0f ? 0.0f : -a.scale * (out[i] / total) * mean;
    }
    uint64_t left = __ballot(there);
    while (left) {
        const int j = __builtin_ctzll(left);
        left &= left - 1;
        const uint32_t e = (uint32_t)__builtin_amdgcn_readlane(mine, j);
        const float more = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(g), j));
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] += first + i == e ? more : 0.0f;
    }
    T* const to = static_cast<T*>(a.d_logits) + (int64_t)token * a.d_stride + first;
    store_elements<DT, V>(to, (int64_t)a.experts - first, out);
}

// ---- assignment: a counting sort of the pairs by expert, pairs of an expert in their own order -----
//
// Bucket b < n: expert first + b; bucket n: every other pair.  A wavefront has kSortChunk / kSortWaves
// consecutive pairs: it counts them by bucket, and when it knows how many come before them in each bucket it
// goes through them 64 at a time.  Lanes with the same bucket find each other by ballots over the bucket's
// bits: the order does not depend on anything's timing.
constexpr int kSortWaves = 8, kSortOne = 4096;      // a launch of one block sorts so many pairs
constexpr uint32_t kMostExperts = 1024;

struct AssignArgs {
    const int32_t* chosen;
    int32_t *offsets, *tokens, *slots;
    uint32_t* counts;        // (blocks, n + 1)
    uint32_t pairs, topk, first, n, bits;
    uint32_t share, blocks;  // pairs of a wavefront; thread blocks
};
__device__ __forceinline__ uint32_t bucket_of(const AssignArgs& a, uint32_t pair) {
    const uint32_t b = (uint32_t)a.chosen[pair] - a.first;
    return b < a.n ? b : a.n;
}
// counts of each wavefront's pairs [begin, end) in `mine`
__device__ __forceinline__ void count_pairs(const AssignArgs& a, uint32_t begin, uint32_t end, uint32_t* mine) {
    for (uint32_t p = begin + lane_id(); p < end; p += 256) {
        uint32_t b[4];                   // (asked for together)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) b[i] = bucket_of(a, min(p + i * 64, end - 1));
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (p + i * 64 < end) atomicAdd(mine + b[i], 1u);
    }
}
__device__ __forceinline__ void place_pairs(const AssignArgs& a, uint32_t begin, uint32_t end, uint32_t* next) {
    uint32_t ahead = begin < end ? bucket_of(a, min(begin + lane_id(), end - 1)) : 0u;
    for (uint32_t p0 = begin; p0 < end; p0 += 64) {
        const uint32_t p = p0 + lane_id(), b = ahead;
        const bool in = p < end;
        if (p0 + 64 < end) ahead = bucket_of(a, min(p + 64, end - 1));
        uint64_t same = __ballot(in);
        for (uint32_t i = 0; i < a.bits; ++i) {
            const uint64_t set = __ballot(b >> i & 1u);
            same &= b >> i & 1u ? set : ~set;
        }
        const uint32_t before = __popcll(same & ((1ull << lane_id()) - 1ull));
        const uint32_t at = in ? next[b] + before : 0u;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (in) {
            if (before == 0) next[b] += __popcll(same);
            const bool here = b < a.n;
            a.slots[p] = here ? (int32_t)at : -1;
            a.tokens[at] = here ? (int32_t)(p / a.topk) : -1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}
// exclusive sums of v[0..n), left in v; all threads of the block take part, `sums` is a number for each wavefront
template <int THREADS>
__device__ __forceinline__ void block_scan(uint32_t* v, uint32_t n, uint32_t* sums) {
    const uint32_t t = threadIdx.x, per = (n + THREADS - 1) / THREADS;
    uint32_t total = 0;
    for (uint32_t i = 0; i < per; ++i) {
        const uint32_t at = t * per + i;
        if (at < n) {
            const uint32_t c = v[at];
            v[at] = total;
            total += c;
        }
    }
    const uint32_t upto = sum_below(total);
    if (lane_id() == 63) sums[wave_in_block()] = upto;
    __syncthreads();
    uint32_t base = upto - total;
    for (int w = 0; w < wave_in_block(); ++w) base += sums[w];
    for (uint32_t i = 0; i < per; ++i)
        if (t * per + i < n) v[t * per + i] += base;
    __syncthreads();
}

// few pairs: all of it in one block
__global__ void __launch_bounds__(64 * kSortWaves) assign_one_kernel(AssignArgs a) {
    __shared__ uint32_t next[kSortWaves][kMostExperts + 1], start[kMostExperts + 1], sums[kSortWaves];
    const uint32_t w = wave_in_block(), buckets = a.n + 1;
    for (uint32_t i = threadIdx.x; i < kSortWaves * buckets; i += 64 * kSortWaves) next[i / buckets][i % buckets] = 0u;
    __syncthreads();
    const uint32_t begin = min(w * a.share, a.pairs), end = min(begin + a.share, a.pairs);
    count_pairs(a, begin, end, next[w]);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < buckets; b += 64 * kSortWaves) {
        uint32_t total = 0;
        for (int i = 0; i < kSortWaves; ++i) {
            const uint32_t c = next[i][b];
            next[i][b] = total;
            total += c;
        }
        start[b] = total;
    }
    __syncthreads();
    block_scan<64 * kSortWaves>(start, buckets, sums);
    for (uint32_t b = threadIdx.x; b < buckets; b += 64 * kSortWaves) {
        a.offsets[b] = (int32_t)start[b];
        for (int i = 0; i < kSortWaves; ++i) next[i][b] += start[b];
    }
    __syncthreads();
    place_pairs(a, begin, end, next[w]);
}

// The sum of blocks [i, end)'s counts: a chain of round trips to the cache, with 32 asked for together (65536 x 8 pairs, 256 buckets: 16.2 us a call
// of the whole assignment, calls behind each other; with 16 18.3, with 64 16.3) and what is left over in 16s, too many of them rather than one by one.
__device__ __forceinline__ uint32_t sum_of_counts(const uint32_t* counts, uint32_t buckets, uint32_t i, uint32_t end) {
    uint32_t sum = 0;
    for (; i + 32 <= end; i += 32) {
        uint32_t c[32];
#pragma unroll
        for (uint32_t u = 0; u < 32; ++u) c[u] = counts[(i + u) * buckets];
#pragma unroll
        for (uint32_t u = 0; u < 32; ++u) sum += c[u];
    }
    for (; i < end; i += 16) {
        uint32_t c[16];
#pragma unroll
        for (uint32_t u = 0; u < 16; ++u) c[u] = counts[min(i + u, end - 1) * buckets];
#pragma unroll
        for (uint32_t u = 0; u < 16; ++u) sum += i + u < end ? c[u] : 0u;
    }
    return sum;
}
// Many: a launch counts each block's pairs by bucket, and a second one, in which every block adds up what it needs of
// those counts (all totals, and its own predecessors'), places them: 65536 x 8 pairs, 256 buckets: kernels of 4.8 and 13.6 us, calls behind each other 16 us each; with a launch of
// one block in between that leaves the sums, 49.
__global__ void __launch_bounds__(64 * kSortWaves) assign_count_kernel(AssignArgs a) {
    __shared__ uint32_t all[kMostExperts + 1];
    const uint32_t buckets = a.n + 1;
    for (uint32_t i = threadIdx.x; i < buckets; i += 64 * kSortWaves) all[i] = 0u;
    __syncthreads();
    const uint32_t begin = min((blockIdx.x * kSortWaves + wave_in_block()) * a.share, a.pairs);
    count_pairs(a, begin, min(begin + a.share, a.pairs), all);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < buckets; i += 64 * kSortWaves) a.counts[(uint64_t)blockIdx.x * buckets + i] = all[i];
}
__global__ void __launch_bounds__(64 * kSortWaves) assign_place_kernel(AssignArgs a) {
    __shared__ uint32_t next[kSortWaves][kMostExperts + 1], start[kMostExperts + 1], sums[kSortWaves];
    const uint32_t w = wave_in_block(), buckets = a.n + 1;
    for (uint32_t i = threadIdx.x; i < kSortWaves * buckets; i += 64 * kSortWaves) next[i / buckets][i % buckets] = 0u;
    __syncthreads();
    const uint32_t begin = min((blockIdx.x * kSortWaves + w) * a.share, a.pairs), end = min(begin + a.share, a.pairs);
    count_pairs(a, begin, end, next[w]);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < buckets; b += 64 * kSortWaves) {
        uint32_t before = sum_of_counts(a.counts + b, buckets, 0, blockIdx.x);
        const uint32_t total = before + sum_of_counts(a.counts + b, buckets, blockIdx.x, a.blocks);
        start[b] = total;
        for (int i = 0; i < kSortWaves; ++i) {
            const uint32_t c = next[i][b];
            next[i][b] = before;
            before += c;
        }
    }
    __syncthreads();
    block_scan<64 * kSortWaves>(start, buckets, sums);
    for (uint32_t b = threadIdx.x; b < buckets; b += 64 * kSortWaves) {
        if (blockIdx.x == 0) a.offsets[b] = (int32_t)start[b];
        for (int i = 0; i < kSortWaves; ++i) next[i][b] += start[b];
    }
    __syncthreads();
    place_pairs(a, begin, end, next[w]);
}

// V of a token's lanes: a power of two.
uint32_t values_per_lane(uint32_t experts, uint32_t lanes) {
    uint32_t v = 1;
    while (v * lanes < experts) v *= 2;
    return v;
}
// 16 lanes to a token where they have enough registers, and one for each choice
uint32_t lanes_of(uint32_t experts, uint32_t topk) { return experts <= 256 && topk <= 16 ? 16 : 64; }
template <int DT, int V, int LANES>
int go_route(const RouteArgs& a, hipStream_t stream) {
    return Launch<&route_kernel<DT, V, LANES>>::go((uint32_t)ceil_div(a.tokens, 64 * kRouteWaves / LANES), 64 * kRouteWaves, 0, stream, a);
}
template <int DT, int V, int LANES>
int go_route_grad(const RouteGradArgs& a, hipStream_t stream) {
    return Launch<&route_grad_kernel<DT, V>>::go((uint32_t)ceil_div(a.tokens, kRouteWaves), 64 * kRouteWaves, 0, stream, a);
}
#define MINT_BY_LANE(GO, DT, LANES)                            \
    switch (values_per_lane(a.experts, LANES)) {               \
        case 1: return GO<DT, 1, LANES>(a, stream);            \
        case 2: return GO<DT, 2, LANES>(a, stream);            \
        case 4: return GO<DT, 4, LANES>(a, stream);            \
        case 8: return GO<DT, 8, LANES>(a, stream);            \
        default: return GO<DT, 16, LANES>(a, stream);          \
    }
#define MINT_BY_TYPE(GO, LANES)                                \
    switch (dtype) {                                           \
        case MINT_F16: MINT_BY_LANE(GO, DT_F16, LANES)         \
        case MINT_BF16: MINT_BY_LANE(GO, DT_BF16, LANES)       \
        default: MINT_BY_LANE(GO, DT_F32, LANES)               \
    }
int launch_route(const RouteArgs& a, int dtype, hipStream_t stream) {
    if (lanes_of(a.experts, a.topk) == 16) {
        MINT_BY_TYPE(go_route, 16)
    }
    MINT_BY_TYPE(go_route, 64)
}
int launch_route_grad(const RouteGradArgs& a, int dtype, hipStream_t stream) { MINT_BY_TYPE(go_route_grad, 64) }

// A launch has fewer than 2^32 threads, and a token up to 64 of them: more tokens take several launches.
constexpr uint64_t kTokensOfLaunch = 1ull << 25;
template <typename F>
int in_launches(uint64_t tokens, const F& go) {
    int err = MINT_OK;
    for (uint64_t t = 0; t < tokens && err == MINT_OK; t += kTokensOfLaunch) err = go(t, (uint32_t)std::min(tokens - t, kTokensOfLaunch));
    return err;
}
// element i of numbers of a type
const void* element(uint64_t base, int64_t i, int dtype) { return reinterpret_cast<const void*>(base + i * (dtype == MINT_F32 ? 4 : 2)); }

bool routable(uint64_t tokens, uint32_t experts, uint32_t topk, int dtype, int score) {
    return experts >= 1 && experts <= kMostExperts && topk >= 1 && topk <= 64 && topk <= experts && tokens < (1ull << 31) &&
           (dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32) && (score == MINT_SCORE_SOFTMAX || score == MINT_SCORE_SIGMOID);
}

}  // namespace
}  // namespace mint

using namespace mint;

extern "C" int mint_route(const mint_route_op* op, void* stream) {
    if (!op || !routable(op->tokens, op->experts, op->topk, op->dtype, op->score)) return MINT_ERR_ARG;
    if (op->groups < 1 || op->groups > 64 || op->experts % op->groups || op->kept < 1 || op->kept > op->groups ||
        op->group_top < 1 || op->group_top > 2)
        return MINT_ERR_GEOMETRY;
    if (op->tokens == 0) return MINT_OK;
    if (!op->logits || !op->weights || !op->chosen) return MINT_ERR_ARG;
    return in_launches(op->tokens, [&](uint64_t t, uint32_t n) {
        const RouteArgs a = {element(op->logits, (int64_t)t * op->row_stride, op->dtype), reinterpret_cast<const float*>(op->bias),
                             reinterpret_cast<float*>(op->weights) + t * op->topk, reinterpret_cast<int32_t*>(op->chosen) + t * op->topk, op->row_stride,
                             n, op->experts, op->topk, op->groups, op->kept, op->group_top, op->scale,
                             op->score == MINT_SCORE_SIGMOID, op->renormalise != 0};
        return launch_route(a, op->dtype, static_cast<hipStream_t>(stream));
    });
}

extern "C" int mint_route_grad(const mint_route_op* op, uint64_t d_weights, uint64_t d_logits, int64_t d_stride, void* stream) {
    if (!op || !routable(op->tokens, op->experts, op->topk, op->dtype, op->score)) return MINT_ERR_ARG;
    if (op->tokens == 0) return MINT_OK;
    if (!op->logits || !op->chosen || !d_weights || !d_logits) return MINT_ERR_ARG;
    return in_launches(op->tokens, [&](uint64_t t, uint32_t n) {
        const RouteGradArgs a = {element(op->logits, (int64_t)t * op->row_stride, op->dtype), reinterpret_cast<const float*>(d_weights) + t * op->topk,
                                 reinterpret_cast<const int32_t*>(op->chosen) + t * op->topk,
                                 const_cast<void*>(element(d_logits, (int64_t)t * d_stride, op->dtype)), op->row_stride, d_stride,
                                 n, op->experts, op->topk, op->scale,
                                 op->score == MINT_SCORE_SIGMOID, op->renormalise != 0};
        return launch_route_grad(a, op->dtype, static_cast<hipStream_t>(stream));
    });
}

namespace {
// pairs of a wavefront and thread blocks: 256 blocks at most (each reads the counts of all)
void shares(uint64_t pairs, uint32_t* share, uint32_t* blocks) {
    const uint64_t waves = pairs <= kSortOne ? kSortWaves : std::min<uint64_t>(256 * kSortWaves, ceil_div(pairs, 128));
    *share = (uint32_t)(ceil_div(ceil_div(pairs, waves), 64) * 64);
    *blocks = pairs ? (uint32_t)ceil_div(pairs, (uint64_t)*share * kSortWaves) : 1;
}
}  // namespace

extern "C" size_t mint_assign_workspace(uint64_t pairs, uint32_t experts) {
    if (pairs <= kSortOne || pairs > 0x7FFFFFFFull) return 0;
    uint32_t share, blocks;
    shares(pairs, &share, &blocks);
    return blocks * ((size_t)experts + 1) * 4;
}

extern "C" int mint_assign(const void* chosen, uint64_t tokens, uint32_t topk, uint32_t first, uint32_t experts, void* offsets,
                           void* order, void* slots, void* workspace, size_t workspace_bytes, void* stream) {
    if (topk < 1 || experts < 1 || experts > kMostExperts || first > 0x7FFFFFFFu - experts || !offsets) return MINT_ERR_ARG;
    if (tokens > 0x7FFFFFFFull / topk) return MINT_ERR_TOO_LARGE;
    const uint64_t pairs = tokens * topk;
    if (pairs && (!chosen || !order || !slots)) return MINT_ERR_ARG;
    const size_t need = mint_assign_workspace(pairs, experts);
    if (need > workspace_bytes || (need && !workspace)) return MINT_ERR_STAGING;
    uint32_t bits = 0, share, blocks;
    while (experts >> bits) ++bits;
    shares(pairs, &share, &blocks);
    const AssignArgs a = {static_cast<const int32_t*>(chosen), static_cast<int32_t*>(offsets), static_cast<int32_t*>(order),
                          static_cast<int32_t*>(slots), static_cast<uint32_t*>(workspace), (uint32_t)pairs, topk, first, experts, bits, share, blocks};
    const auto s = static_cast<hipStream_t>(stream);
    if (!need) return Launch<&assign_one_kernel>::go(1, 64 * kSortWaves, 0, s, a);
    const int err = Launch<&assign_count_kernel>::go(blocks, 64 * kSortWaves, 0, s, a);
    return err == MINT_OK ? Launch<&assign_place_kernel>::go(blocks, 64 * kSortWaves, 0, s, a) : err;
}
