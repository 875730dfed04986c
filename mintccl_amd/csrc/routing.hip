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
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

struct RouteArgs {
    const void* logits;
    const float* bias;
    float* weights;
    int32_t* chosen;
    int64_t row_stride;
    uint32_t tokens, experts, topk, groups, kept, group_top;
    float scale;
    uint32_t whole;          // a lane's logits may be loaded as one vector
    uint32_t sigmoid, renormalise;
};

// A lane has V consecutive experts, so that among equal keys the lowest lane has the lowest expert.
template <int DT, int V>
__global__ void __launch_bounds__(64 * kRouteWaves) route_kernel(RouteArgs a) {
    using T = typename Elem<DT>::type;
    const uint32_t token = blockIdx.x * kRouteWaves + wave_in_block(), lane = lane_id(), first = lane * V;
    if (token >= a.tokens) return;
    const T* const row = static_cast<const T*>(a.logits) + (int64_t)token * a.row_stride;
    float x[V];
    load_elements<DT, V>(row + first, a.whole && first + V <= a.experts, (int64_t)a.experts - first, x);
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float s = a.sigmoid ? sigmoid(x[i]) : x[i];
        const float b = a.bias && first + i < a.experts ? a.bias[first + i] : 0.0f;
        key[i] = first + i < a.experts && x[i] != -INFINITY ? order_of(s + b) : 0u;
    }
    if (a.groups > 1) {
        const uint32_t per = a.experts / a.groups;
        uint32_t of_group = 0;                               // lane g: the key of group g
        for (uint32_t g = 0; g < a.groups; ++g) {
            uint32_t best = 0, second = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const uint32_t k = first + i - g * per < per ? key[i] : 0u;
                second = max(second, min(best, k));
                best = max(best, k);
            }
            uint32_t top = wave_max(best);
            if (a.group_top == 2 && top != 0u) {
                const uint32_t holder = __builtin_ctzll(__ballot(best == top));
                const uint32_t next = wave_max(lane == holder ? second : best);
                if (next != 0u) top = order_of(number_of(top) + number_of(next));
            }
            if (lane == g) of_group = top;
        }
        uint64_t keep = 0;
        for (uint32_t n = 0; n < a.kept; ++n) {
            const uint32_t top = wave_max(of_group);
            if (top == 0u) break;
            const uint32_t g = __builtin_ctzll(__ballot(of_group == top));
            keep |= 1ull << g;
            if (lane == g) of_group = 0u;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = keep >> min((first + i) / per, 63u) & 1u ? key[i] : 0u;
    }
    int32_t mine = -1;                                       // lane j: the j-th choice
    for (uint32_t j = 0; j < a.topk; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i]);
        const uint32_t top = wave_max(best);
        if (top == 0u) break;
        const uint32_t holder = __builtin_ctzll(__ballot(best == top));
        uint32_t at = 0;
#pragma unroll
        for (int i = V - 1; i >= 0; --i) at = key[i] == top ? i : at;
        const int32_t e = __builtin_amdgcn_readlane((int)(first + at), holder);
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = first + i == (uint32_t)e ? 0u : key[i];
        if (lane == j) mine = e;
    }
    const bool there = mine >= 0;
    const float l = there ? Elem<DT>::load(row[mine]) : -INFINITY;
    float s, total = 1.0f;
    if (a.sigmoid) {
        s = there ? sigmoid(l) : 0.0f;
        if (a.renormalise) total = wave_sum(s);
    } else {
        // the largest logit of those in the sum: of the chosen, or of all
        float m = l;
        if (!a.renormalise) {
#pragma unroll
            for (int i = 0; i < V; ++i) m = first + i < a.experts ? fmaxf(m, x[i]) : m;
        }
        m = wave_max(m);
        m = m == -INFINITY ? 0.0f : m;
        s = there ? expf(l - m) : 0.0f;
        float sum = s;
        if (!a.renormalise) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += first + i < a.experts ? expf(x[i] - m) : 0.0f;
        }
        total = wave_sum(sum);
    }
    // (every chosen score may have vanished: then so have the weights)
    const float w = !there || total == 0.0f ? 0.0f : a.scale * (s / total);
    if (lane < a.topk) {
        a.weights[(uint64_t)token * a.topk + lane] = w;
        a.chosen[(uint64_t)token * a.topk + lane] = mine;
    }
}

// The logits' gradient from the weights' d, with w' = w / scale and p = softmax(x):
//   softmax, renormalised   scale w'_j (d_j - sum w' d)             0 where nothing was chosen
//   softmax                 scale p_i (d_i [chosen] - sum w' d)
//   sigmoid, renormalised   scale (d_j - sum w' d) s_j (1 - s_j) / sum s
//   sigmoid                 scale d_j s_j (1 - s_j)
// The scores are computed again from the logits: they cost less than they would to keep.
struct RouteGradArgs {
    const void* logits;
    const float* d_weights;
    const int32_t* chosen;
    void* d_logits;
    int64_t row_stride, d_stride;
    uint32_t tokens, experts, topk;
    float scale;
    uint32_t whole, d_whole, sigmoid, renormalise;
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
            g = total == 0.0f ? 0.0f : a.scale * ((d - mean / total) / total) * slope;
        } else {
            g = a.scale * d * slope;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = 0.0f;
    } else {
        float x[V], m = l;
        if (!a.renormalise) {
            load_elements<DT, V>(row + first, a.whole && first + V <= a.experts, (int64_t)a.experts - first, x);
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
    store_elements<DT, V>(to, a.d_whole && first + V <= a.experts, (int64_t)a.experts - first, out);
}

// ---- assignment: a counting sort of the pairs by expert, pairs of an expert in their own order -----
//
// Bucket b < n: expert first + b; bucket n: every other pair.  A wavefront has kSortChunk / kSortWaves
// consecutive pairs: it counts them by bucket, and when it knows how many come before them in each bucket it
// goes through them 64 at a time.  Lanes with the same bucket find each other by ballots over the bucket's
// bits: the order does not depend on anything's timing.
constexpr int kSortWaves = 8, kSortChunk = 4096, kSortOne = 16384;     // pairs of a block; of a launch of one block
constexpr uint32_t kMostExperts = 1024;

struct AssignArgs {
    const int32_t* chosen;
    int32_t *offsets, *tokens, *slots;
    uint32_t* counts;        // (blocks, n + 1), then the places where they begin
    uint32_t pairs, topk, first, n, bits;
};
__device__ __forceinline__ uint32_t bucket_of(const AssignArgs& a, uint32_t pair) {
    const uint32_t b = (uint32_t)a.chosen[pair] - a.first;
    return b < a.n ? b : a.n;
}
// counts of each wavefront's pairs [begin, end) in `mine`
__device__ __forceinline__ void count_pairs(const AssignArgs& a, uint32_t begin, uint32_t end, uint32_t* mine) {
    for (uint32_t p = begin + lane_id(); p < end; p += 64) atomicAdd(mine + bucket_of(a, p), 1u);
}
__device__ __forceinline__ void place_pairs(const AssignArgs& a, uint32_t begin, uint32_t end, uint32_t* next) {
    for (uint32_t p0 = begin; p0 < end; p0 += 64) {
        const uint32_t p = p0 + lane_id();
        const bool in = p < end;
        const uint32_t b = in ? bucket_of(a, p) : 0u;
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
// exclusive sums of v[0..n) over the block's threads, left in v; all threads take part
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
    sums[t] = total;
    __syncthreads();
    for (uint32_t d = 1; d < THREADS; d <<= 1) {
        const uint32_t other = t >= d ? sums[t - d] : 0u;
        __syncthreads();
        sums[t] += other;
        __syncthreads();
    }
    const uint32_t base = sums[t] - total;
    for (uint32_t i = 0; i < per; ++i)
        if (t * per + i < n) v[t * per + i] += base;
    __syncthreads();
}

// few pairs: all of it in one block
__global__ void __launch_bounds__(64 * kSortWaves) assign_one_kernel(AssignArgs a) {
    __shared__ uint32_t next[kSortWaves][kMostExperts + 1], start[kMostExperts + 1], sums[64 * kSortWaves];
    const uint32_t w = wave_in_block(), buckets = a.n + 1;
    for (uint32_t i = threadIdx.x; i < kSortWaves * buckets; i += 64 * kSortWaves) next[i / buckets][i % buckets] = 0u;
    __syncthreads();
    const uint32_t share = ((a.pairs + kSortWaves - 1) / kSortWaves + 63) & ~63u;
    const uint32_t begin = min(w * share, a.pairs), end = min(begin + share, a.pairs);
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

__global__ void __launch_bounds__(64 * kSortWaves) assign_count_kernel(AssignArgs a) {
    __shared__ uint32_t all[kMostExperts + 1];
    const uint32_t buckets = a.n + 1;
    for (uint32_t i = threadIdx.x; i < buckets; i += 64 * kSortWaves) all[i] = 0u;
    __syncthreads();
    const uint32_t begin = blockIdx.x * kSortChunk + wave_in_block() * (kSortChunk / kSortWaves);
    count_pairs(a, min(begin, a.pairs), min(begin + kSortChunk / kSortWaves, a.pairs), all);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < buckets; i += 64 * kSortWaves) a.counts[(uint64_t)blockIdx.x * buckets + i] = all[i];
}
// counts of all blocks -> where each block's pairs of each bucket begin; one block
__global__ void __launch_bounds__(1024) assign_scan_kernel(AssignArgs a, uint32_t blocks) {
    __shared__ uint32_t start[kMostExperts + 1], sums[1024];
    const uint32_t buckets = a.n + 1;
    for (uint32_t b = threadIdx.x; b < buckets; b += 1024) {
        uint32_t total = 0;
        for (uint32_t i = 0; i < blocks; ++i) {
            const uint64_t at = (uint64_t)i * buckets + b;
            const uint32_t c = a.counts[at];
            a.counts[at] = total;
            total += c;
        }
        start[b] = total;
    }
    __syncthreads();
    block_scan<1024>(start, buckets, sums);
    for (uint32_t b = threadIdx.x; b < buckets; b += 1024) a.offsets[b] = (int32_t)start[b];
}
__global__ void __launch_bounds__(64 * kSortWaves) assign_place_kernel(AssignArgs a) {
    __shared__ uint32_t next[kSortWaves][kMostExperts + 1];
    const uint32_t w = wave_in_block(), buckets = a.n + 1;
    for (uint32_t i = threadIdx.x; i < kSortWaves * buckets; i += 64 * kSortWaves) next[i / buckets][i % buckets] = 0u;
    __syncthreads();
    const uint32_t begin = min(blockIdx.x * kSortChunk + w * (kSortChunk / kSortWaves), a.pairs);
    const uint32_t end = min(begin + kSortChunk / kSortWaves, a.pairs);
    count_pairs(a, begin, end, next[w]);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < buckets; b += 64 * kSortWaves) {
        uint32_t total = (uint32_t)a.offsets[b] + a.counts[(uint64_t)blockIdx.x * buckets + b];
        for (int i = 0; i < kSortWaves; ++i) {
            const uint32_t c = next[i][b];
            next[i][b] = total;
            total += c;
        }
    }
    __syncthreads();
    place_pairs(a, begin, end, next[w]);
}

uint32_t values_per_lane(uint32_t experts) {
    uint32_t v = 1;
    while (v * 64 < experts) v *= 2;
    return v;
}
template <int DT, int V>
int go_route(const RouteArgs& a, hipStream_t stream) {
    return Launch<&route_kernel<DT, V>>::go((uint32_t)ceil_div(a.tokens, kRouteWaves), 64 * kRouteWaves, 0, stream, a);
}
template <int DT, int V>
int go_route_grad(const RouteGradArgs& a, hipStream_t stream) {
    return Launch<&route_grad_kernel<DT, V>>::go((uint32_t)ceil_div(a.tokens, kRouteWaves), 64 * kRouteWaves, 0, stream, a);
}
#define MINT_BY_LANE(GO, DT)                            \
    switch (values_per_lane(a.experts)) {               \
        case 1: return GO<DT, 1>(a, stream);            \
        case 2: return GO<DT, 2>(a, stream);            \
        case 4: return GO<DT, 4>(a, stream);            \
        case 8: return GO<DT, 8>(a, stream);            \
        default: return GO<DT, 16>(a, stream);          \
    }
#define MINT_BY_TYPE(GO)                                \
    switch (dtype) {                                    \
        case MINT_F16: MINT_BY_LANE(GO, DT_F16)         \
        case MINT_BF16: MINT_BY_LANE(GO, DT_BF16)       \
        default: MINT_BY_LANE(GO, DT_F32)               \
    }
int launch_route(const RouteArgs& a, int dtype, hipStream_t stream) { MINT_BY_TYPE(go_route) }
int launch_route_grad(const RouteGradArgs& a, int dtype, hipStream_t stream) { MINT_BY_TYPE(go_route_grad) }

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
    const uint32_t vector = values_per_lane(op->experts) * element_bytes(op->dtype);
    const bool whole = aligned_to(reinterpret_cast<void*>(op->logits), vector) && op->row_stride * element_bytes(op->dtype) % vector == 0;
    const RouteArgs a = {reinterpret_cast<const void*>(op->logits), reinterpret_cast<const float*>(op->bias),
                         reinterpret_cast<float*>(op->weights), reinterpret_cast<int32_t*>(op->chosen), op->row_stride,
                         (uint32_t)op->tokens, op->experts, op->topk, op->groups, op->kept, op->group_top, op->scale, whole,
                         op->score == MINT_SCORE_SIGMOID, op->renormalise != 0};
    return launch_route(a, op->dtype, static_cast<hipStream_t>(stream));
}

extern "C" int mint_route_grad(const mint_route_op* op, uint64_t d_weights, uint64_t d_logits, int64_t d_stride, void* stream) {
    if (!op || !routable(op->tokens, op->experts, op->topk, op->dtype, op->score)) return MINT_ERR_ARG;
    if (op->tokens == 0) return MINT_OK;
    if (!op->logits || !op->chosen || !d_weights || !d_logits) return MINT_ERR_ARG;
    const uint32_t size = element_bytes(op->dtype), vector = values_per_lane(op->experts) * size;
    const bool whole = aligned_to(reinterpret_cast<void*>(op->logits), vector) && op->row_stride * size % vector == 0;
    const bool d_whole = aligned_to(reinterpret_cast<void*>(d_logits), vector) && d_stride * size % vector == 0;
    const RouteGradArgs a = {reinterpret_cast<const void*>(op->logits), reinterpret_cast<const float*>(d_weights),
                             reinterpret_cast<const int32_t*>(op->chosen), reinterpret_cast<void*>(d_logits), op->row_stride, d_stride,
                             (uint32_t)op->tokens, op->experts, op->topk, op->scale, whole, d_whole,
                             op->score == MINT_SCORE_SIGMOID, op->renormalise != 0};
    return launch_route_grad(a, op->dtype, static_cast<hipStream_t>(stream));
}

extern "C" size_t mint_assign_workspace(uint64_t pairs, uint32_t experts) {
    return pairs <= kSortOne ? 0 : ceil_div(pairs, kSortChunk) * ((size_t)experts + 1) * 4;
}

extern "C" int mint_assign(const void* chosen, uint64_t tokens, uint32_t topk, uint32_t first, uint32_t experts, void* offsets,
                           void* order, void* slots, void* workspace, size_t workspace_bytes, void* stream) {
    if (topk < 1 || experts < 1 || experts > kMostExperts || first > 0x7FFFFFFFu - experts || !offsets) return MINT_ERR_ARG;
    if (tokens > 0x7FFFFFFFull / topk) return MINT_ERR_TOO_LARGE;
    const uint64_t pairs = tokens * topk;
    if (pairs && (!chosen || !order || !slots)) return MINT_ERR_ARG;
    const size_t need = mint_assign_workspace(pairs, experts);
    if (need > workspace_bytes || (need && !workspace)) return MINT_ERR_STAGING;
    uint32_t bits = 0;
    while (experts >> bits) ++bits;
    const AssignArgs a = {static_cast<const int32_t*>(chosen), static_cast<int32_t*>(offsets), static_cast<int32_t*>(order),
                          static_cast<int32_t*>(slots), static_cast<uint32_t*>(workspace), (uint32_t)pairs, topk, first, experts, bits};
    const auto s = static_cast<hipStream_t>(stream);
    if (!need) return Launch<&assign_one_kernel>::go(1, 64 * kSortWaves, 0, s, a);
    const uint32_t blocks = (uint32_t)ceil_div(pairs, kSortChunk);
    int err = Launch<&assign_count_kernel>::go(blocks, 64 * kSortWaves, 0, s, a);
    if (err == MINT_OK) err = Launch<&assign_scan_kernel>::go(1, 1024, 0, s, a, blocks);
    if (err == MINT_OK) err = Launch<&assign_place_kernel>::go(blocks, 64 * kSortWaves, 0, s, a);
    return err;
}
