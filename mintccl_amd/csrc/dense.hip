// Dense matrix products in 16 and 32 bits with what surrounds them, and their gradients.
//
//   z = x w^T + b      out = residual + a(z)
//   d_z = d a'(z)      d_b = sum over rows of d_z      d_x = d_z w      d_w = d_z^T x
//
// The three products are one kernel: the result's rows come from one operand, its columns from the other, and each of them
// lies in memory either with the depth along its rows ("along": x and w of the first product) or across them ("across": w of d_x, both
// of d_w).  Sums are in 32 bits in a fixed order; z and d_z are rounded once each to the operands' type, out once to its own.
#include "activations.hpp"

#include <algorithm>

namespace mint {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// 32 bytes of an operand's row or column as the matrix instructions take them: a lane has 16 bytes of the first half of the
// depth's block and 16 of the second.
template <int DT>
struct Pair {
    u32x4 v[2];
    static __device__ __forceinline__ f32x4 multiply(const Pair& a, const Pair& b, f32x4 c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (DT == DT_BF16) {
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v[h]), __builtin_bit_cast(bf16x8, b.v[h]), c, 0, 0, 0);
            } else if constexpr (DT == DT_F16) {
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v[h]), __builtin_bit_cast(f16x8, b.v[h]), c, 0, 0, 0);
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[h][t]), __uint_as_float(b.v[h][t]), c, 0, 0, 0);
            }
        }
        return c;
    }
};
template <int DT>
constexpr uint32_t kSize = sizeof(typename Elem<DT>::type);
template <int DT>
constexpr uint32_t kBlock = 128 / kSize<DT>;            // numbers of the depth that go by together

__device__ __forceinline__ void to_lds16(const uint8_t* from, uint32_t lds) {
    __builtin_amdgcn_global_load_lds((MINT_GLOBAL const void*)as_global(from), (MINT_LDS void*)(uintptr_t)lds, 16, 0, 0);
}
__device__ __forceinline__ u32x4 lds16(uint32_t at) { return *(MINT_LDS const u32x4*)(uintptr_t)at; }
// the first `left` bytes, zeros behind
__device__ __forceinline__ u32x4 first_of(u32x4 v, int64_t left) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t bytes = left - 4 * i;
        v[i] &= bytes >= 4 ? 0xFFFFFFFFu : bytes <= 0 ? 0u : (1u << 8 * bytes) - 1u;
    }
    return v;
}
// 16 bytes at any address of which the first `left` are there (whole numbers of SIZE bytes)
template <uint32_t SIZE>
__device__ __forceinline__ u32x4 piece_of(const uint8_t* from, int64_t left) {
    if (left >= 16) return *(MINT_GLOBAL const u32x4_any*)as_global(from);
    u32x4 v = {0, 0, 0, 0};
    if constexpr (SIZE == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (left >= 4 * i + 4) v[i] = *(MINT_GLOBAL const uint32_t*)as_global(from + 4 * i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (left >= 2 * i + 2) v[i / 2] |= (uint32_t)*(MINT_GLOBAL const uint16_t*)as_global(from + 2 * i) << (i % 2 * 16);
    }
    return v;
}
// All but the N latest of a wavefront's loads are done; then all wavefronts meet.
template <int N>
__device__ __forceinline__ void meet() {
    if constexpr (N == 0) {
        __syncthreads();
    } else {
        __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 15 << 8);
        compiler_fence();
        __builtin_amdgcn_s_barrier();
        compiler_fence();
    }
}

// An operand: `n` rows or columns of the result.  ALONG: row i of it at p + i * stride, the depth along it; else depth d at p + d * stride.
struct Side {
    const uint8_t* p;
    int64_t stride;              // bytes
    uint32_t n;
};
// B of them in LDS, a block of the depth: B * 128 bytes either way, in pieces of 16.
//   along    a row of 128 bytes for each of them, pieces turned by the row's number: the lanes that a 16-byte read serves
//            together are of different rows
//   across   a row of B numbers for each number of the depth; a lane's numbers of one column are gathered by the
//            transposing reads (16 bits: 16 lanes have four rows of 16 numbers), or one by one (32 bits).  The groups of 16 numbers are
//            turned by the row's number likewise
template <int DT, int B, bool ALONG>
struct Staged {
    static constexpr uint32_t SIZE = kSize<DT>, PIECES = ALONG ? 8 : B * SIZE / 16;      // of an LDS row
    static __device__ __forceinline__ uint32_t turn(uint32_t row) {
        if constexpr (ALONG) return (row >> 1) & 7u;
        else if constexpr (SIZE == 4) return (row >> 2 & 3u) * 4;
        else if constexpr (PIECES == 8) return ((row >> 1 & 1u) | (row >> 2 & 2u)) * 2;
        else return ((row & 3u) | (row >> 1 & 4u)) * 2;
    }
    // where unit u (16 bytes in LDS, in order) comes from: its LDS row and its piece of the row in memory
    static __device__ __forceinline__ uint32_t row_of(uint32_t u) { return u / PIECES; }
    static __device__ __forceinline__ uint32_t piece_of(uint32_t u) { return (u % PIECES) ^ turn(u / PIECES); }

    // A lane's part of the g-th 16 of them.
    uint32_t base;               // along: the lane's first piece of the first 16; across: the lane's numbers of its LDS row's first 16
    uint32_t turned;             // across: what the number of the 16 is turned by in that row
    __device__ __forceinline__ explicit Staged(uint32_t lane) {
        const uint32_t r16 = lane & 15u, part = lane >> 4;
        if constexpr (ALONG) {
            base = r16 * 128 + ((part ^ turn(r16)) * 16);        // (16 rows on the turning is the same)
            turned = 0;
        } else if constexpr (SIZE == 4) {
            base = part * 4 * (B * 4) + r16 * 4;
            turned = part;
        } else {
            const uint32_t row = part * 8 + (r16 >> 2);          // (4 and 32 rows on the turning is the same)
            base = row * (B * 2) + (r16 & 3u) * 8;
            turned = turn(row) / 2;
        }
    }
    __device__ __forceinline__ Pair<DT> load(uint32_t at, uint32_t g) const {
        Pair<DT> p;
        if constexpr (ALONG) {
            p.v[0] = lds16(at + g * 2048 + base);
            p.v[1] = lds16(at + g * 2048 + (base ^ 64u));
        } else if constexpr (SIZE == 4) {
            const uint32_t from = at + base + (g ^ turned) * 64;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < 4; ++t) p.v[h][t] = *(MINT_LDS const uint32_t*)(uintptr_t)(from + (h * 16 + t) * (B * 4));
        } else {
            const uint32_t from = at + base + (g ^ turned) * 32;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                i16x4 q[2];
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    q[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MINT_LDS i16x4*)(uintptr_t)(from + (h * 32 + j * 4) * (B * 2)));
                const u32x2 lo = __builtin_bit_cast(u32x2, q[0]), hi = __builtin_bit_cast(u32x2, q[1]);
                p.v[h] = u32x4{lo.x, lo.y, hi.x, hi.y};
            }
        }
        return p;
    }
};

struct Finish {
    const void *bias, *residual;         // either may be 0
    void *out, *z;                       // z may be 0
    int64_t residual_stride, out_stride, z_stride;      // elements
    int out_dtype, activation;
};
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t at, int64_t left, float (&v)[8]) {
    load_elements<DT, 8>(static_cast<const typename Elem<DT>::type*>(p) + at, left, v);
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, int64_t left, const float (&v)[8]) {
    store_elements<DT, 8>(static_cast<typename Elem<DT>::type*>(p) + at, left, v);
}
// Eight sums of a row of the result become what is stored.  Results are of the operands' type or in 32 bits.
template <int DT>
__device__ __forceinline__ void finish8(const Finish& f, uint32_t row, uint32_t col, uint32_t cols, float (&v)[8]) {
    const int64_t left = (int64_t)cols - col;
    float more[8];
    if (f.bias) {
        load8<DT>(f.bias, col, left, more);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += more[i];
    }
    if (f.z) store8<DT>(f.z, (int64_t)row * f.z_stride + col, left, v);
    if (f.activation != MINT_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activated(f.activation, v[i]);
    }
    const bool wide = f.out_dtype == MINT_F32;
    if (f.residual) {
        if (wide) load8<DT_F32>(f.residual, (int64_t)row * f.residual_stride + col, left, more);
        else load8<DT>(f.residual, (int64_t)row * f.residual_stride + col, left, more);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += more[i];
    }
    if (wide) store8<DT_F32>(f.out, (int64_t)row * f.out_stride + col, left, v);
    else store8<DT>(f.out, (int64_t)row * f.out_stride + col, left, v);
}

struct DenseArgs {
    Side x, w;                           // the result's rows and columns
    Finish f;
    uint32_t depth, row_tiles, col_tiles;
    uint32_t parts;                      // thread blocks that share a tile's depth; more than one: their sums go to
    float* sums;                         // (parts, rows, cols)
};

// A thread block has BM rows and BN columns of the result, a wavefront BM / WM rows and 64 columns of them.  The depth goes by in blocks of
// 128 bytes; while one is multiplied the next STAGES - 1 ones are on their way into LDS.  DIRECT: rows in memory begin at
// multiples of 16 bytes, and their pieces go straight into LDS; else they pass through registers.
template <int DT, int BM, int BN, int WM, int STAGES, bool X_ALONG, bool W_ALONG, bool DIRECT>
__global__ void __launch_bounds__(64 * WM * (BN / 64)) dense_kernel(DenseArgs a) {
    constexpr int WN = BN / 64, WAVES = WM * WN, MT = BM / WM / 16, NT = 4, XI = BM / 8 / WAVES, WI = BN / 8 / WAVES, ALL = XI + WI;
    constexpr uint32_t SIZE = kSize<DT>, K = kBlock<DT>, kX = BM * 128, kStage = (BM + BN) * 128;
    constexpr uint32_t SLABS = MT < 4 ? MT : 4, PITCH = 68;               // of the sums' way out: slabs of 16 rows of 64 columns
    constexpr uint32_t kOut = WAVES * SLABS * 16 * PITCH * 4, kLds = STAGES * kStage > kOut ? STAGES * kStage : kOut;
    static_assert(XI * 8 * WAVES == BM && WI * 8 * WAVES == BN, "every wavefront brings as much");
    static_assert(kLds <= 160 * 1024, "it fits LDS");
    using SX = Staged<DT, BM, X_ALONG>;
    using SW = Staged<DT, BN, W_ALONG>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_in_block()), wm = wave / WN, wn = wave % WN;
    const uint32_t base = (uint32_t)(uintptr_t)(MINT_LDS uint8_t*)lds;

    // The hardware deals thread blocks to the eight XCDs in turn: each takes an eighth of the tiles that lie together, in
    // columns of GROUP row tiles, so that those at work at a time share operands in its L2.
    constexpr uint32_t GROUP = 4;
    const uint32_t total = a.row_tiles * a.col_tiles * a.parts, xcd = blockIdx.x & 7u, nth = blockIdx.x >> 3;
    if (nth >= total / 8 + (xcd < total % 8)) return;
    const uint32_t all_id = xcd * (total / 8) + min(xcd, total % 8) + nth, id = all_id / a.parts, part = all_id % a.parts;
    const uint32_t group = id / (GROUP * a.col_tiles), in_group = id % (GROUP * a.col_tiles), height = min(GROUP, a.row_tiles - group * GROUP);
    const uint32_t m0 = (group * GROUP + in_group % height) * BM, n0 = in_group / height * BN;

    // this part's blocks of the depth; the last of all may not be whole
    const uint32_t blocks = (a.depth + K - 1) / K, share = (blocks + a.parts - 1) / a.parts, b0 = min(part * share, blocks);
    const uint32_t steps = min(share, blocks - b0), tail = a.depth % K, full = steps && tail && b0 + steps == blocks ? steps - 1 : steps;

    // The 16 bytes that this lane brings with instruction n of the operand: from there, and how much of them is there
    const auto unit = [&](int n, int each) MINT_INLINE_LAMBDA { return (wave * each + n) * 64 + lane; };
    const auto start = [&](const Side& s, uint32_t first, bool along, uint32_t row, uint32_t piece) MINT_INLINE_LAMBDA {
        if (along) return s.p + (int64_t)min(first + row, s.n - 1) * s.stride + ((int64_t)b0 * 128 + piece * 16);
        // (a piece behind the last one: that one instead)
        return s.p + ((int64_t)b0 * K + row) * s.stride + min((int64_t)first * SIZE + piece * 16, ((int64_t)s.n * SIZE - 1) / 16 * 16);
    };
    const uint8_t *from_x[XI], *from_w[WI];
    const int64_t step_x = X_ALONG ? 128 : (int64_t)K * a.x.stride, step_w = W_ALONG ? 128 : (int64_t)K * a.w.stride;
    if (steps) {
#pragma unroll
        for (int n = 0; n < XI; ++n) from_x[n] = start(a.x, m0, X_ALONG, SX::row_of(unit(n, XI)), SX::piece_of(unit(n, XI)));
#pragma unroll
        for (int n = 0; n < WI; ++n) from_w[n] = start(a.w, n0, W_ALONG, SW::row_of(unit(n, WI)), SW::piece_of(unit(n, WI)));
    }

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    const SX sx(lane);
    const SW sw(lane);
    const auto multiply = [&](uint32_t at, const auto& meanwhile) MINT_INLINE_LAMBDA {
        const Pair<DT> w[NT] = {sw.load(at + kX, wn * 4), sw.load(at + kX, wn * 4 + 1), sw.load(at + kX, wn * 4 + 2), sw.load(at + kX, wn * 4 + 3)};
        Pair<DT> x = sx.load(at, wm * MT);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            // (the next block's loads go out between the products: all at once they would stand in each other's way)
            constexpr int PIECES = MT > 1 ? (ALL * 2 + MT - 1) / MT : ALL;
#pragma unroll
            for (int n = 0; n < PIECES; ++n)
                if (i * PIECES + n < ALL) meanwhile(i * PIECES + n);
            Pair<DT> next = x;
            if (i + 1 < MT) next = sx.load(at, wm * MT + i + 1);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = Pair<DT>::multiply(w[j], x, acc[i][j]);
            x = next;
        }
    };

    if constexpr (DIRECT) {
        const auto bring = [&](uint32_t at, int n) MINT_INLINE_LAMBDA {
            if (n < XI) {
                to_lds16(from_x[n], at + (wave * XI + n) * 1024);
                from_x[n] += step_x;
            } else {
                to_lds16(from_w[n - XI], at + kX + (wave * WI + (n - XI)) * 1024);
                from_w[n - XI] += step_w;
            }
        };
        // The depth's last block where it is not whole comes like the others, what lies behind the depth from the block's beginning; then
        // it is cleared in LDS.
        const auto bring_tail = [&](uint32_t at) MINT_INLINE_LAMBDA {
            const auto inside = [&](const uint8_t* from, bool along, uint32_t row, uint32_t piece, int64_t stride) MINT_INLINE_LAMBDA {
                if (along) return piece * 16 < tail * SIZE ? from : from - piece * 16;
                return row < tail ? from : from - (int64_t)row * stride;
            };
#pragma unroll
            for (int n = 0; n < XI; ++n)
                to_lds16(inside(from_x[n], X_ALONG, SX::row_of(unit(n, XI)), SX::piece_of(unit(n, XI)), a.x.stride), at + (wave * XI + n) * 1024);
#pragma unroll
            for (int n = 0; n < WI; ++n)
                to_lds16(inside(from_w[n], W_ALONG, SW::row_of(unit(n, WI)), SW::piece_of(unit(n, WI)), a.w.stride), at + kX + (wave * WI + n) * 1024);
        };
        const auto clear_tail = [&](uint32_t at) MINT_INLINE_LAMBDA {
            const auto clear = [&](bool along, uint32_t row, uint32_t piece, uint32_t to) MINT_INLINE_LAMBDA {
                const auto v = (MINT_LDS u32x4*)(uintptr_t)to;
                *v = first_of(*v, along ? (int64_t)(tail * SIZE) - piece * 16 : row < tail ? 16 : 0);
            };
#pragma unroll
            for (int n = 0; n < XI; ++n) clear(X_ALONG, SX::row_of(unit(n, XI)), SX::piece_of(unit(n, XI)), at + unit(n, XI) * 16);
#pragma unroll
            for (int n = 0; n < WI; ++n) clear(W_ALONG, SW::row_of(unit(n, WI)), SW::piece_of(unit(n, WI)), at + kX + unit(n, WI) * 16);
        };
        uint32_t b = 0, at = base, ahead = base + (STAGES - 1) * kStage;
        const auto after = [&](uint32_t stage) MINT_INLINE_LAMBDA { return stage + kStage == base + STAGES * kStage ? base : stage + kStage; };
        const auto bring_all = [&](uint32_t to) MINT_INLINE_LAMBDA {
#pragma unroll
            for (int n = 0; n < ALL; ++n) bring(to, n);
        };
#pragma unroll
        for (int st = 0; st < STAGES - 1; ++st) {
            if ((uint32_t)st < full) bring_all(base + st * kStage);
            else if ((uint32_t)st == full && full < steps) bring_tail(base + st * kStage);
        }
        for (; b + STAGES - 1 < full; ++b) {
            meet<(STAGES - 2) * ALL>();
            multiply(at, [&](int n) MINT_INLINE_LAMBDA { bring(ahead, n); });
            at = after(at);
            ahead = after(ahead);
        }
        for (; b < steps; ++b) {
            __syncthreads();             // (waits for the loads into LDS too)
            if (b + STAGES - 1 == full && full < steps) bring_tail(ahead);
            if (b == full) {
                clear_tail(at);
                __syncthreads();
            }
            multiply(at, [](int) MINT_INLINE_LAMBDA {});
            at = after(at);
            ahead = after(ahead);
        }
    } else {
        u32x4 held[ALL];
        const auto fetch = [&](uint32_t b) MINT_INLINE_LAMBDA {
            const uint32_t d0 = (b0 + b) * K;            // (depth that is there from here on)
            const auto one = [&](const Side& s, bool along, uint32_t first, uint32_t row, uint32_t piece) MINT_INLINE_LAMBDA {
                if (along)
                    return piece_of<SIZE>(s.p + (int64_t)min(first + row, s.n - 1) * s.stride + ((int64_t)d0 * SIZE + piece * 16), ((int64_t)a.depth - d0) * SIZE - piece * 16);
                const int64_t left = ((int64_t)s.n - first) * SIZE - piece * 16;
                return piece_of<SIZE>(s.p + (int64_t)min(d0 + row, a.depth - 1) * s.stride + ((int64_t)first * SIZE + piece * 16), d0 + row < a.depth ? left : 0);
            };
#pragma unroll
            for (int n = 0; n < XI; ++n) held[n] = one(a.x, X_ALONG, m0, SX::row_of(unit(n, XI)), SX::piece_of(unit(n, XI)));
#pragma unroll
            for (int n = 0; n < WI; ++n) held[XI + n] = one(a.w, W_ALONG, n0, SW::row_of(unit(n, WI)), SW::piece_of(unit(n, WI)));
        };
        if (steps) fetch(0);
        for (uint32_t b = 0; b < steps; ++b) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < XI; ++n) *(MINT_LDS u32x4*)(uintptr_t)(base + unit(n, XI) * 16) = held[n];
#pragma unroll
            for (int n = 0; n < WI; ++n) *(MINT_LDS u32x4*)(uintptr_t)(base + kX + unit(n, WI) * 16) = held[XI + n];
            __syncthreads();
            if (b + 1 < steps) fetch(b + 1);
            multiply(base, [](int) MINT_INLINE_LAMBDA {});
        }
    }

    // The sums' way out: a lane has four columns of 16 rows each; through LDS it gets eight of a row, and eight lanes side by side 64.
    __syncthreads();
    float* const room = reinterpret_cast<float*>(lds) + wave * (SLABS * 16 * PITCH);
    const uint32_t r16 = lane & 15u, quarter = lane >> 4, col = n0 + wn * 64 + (lane & 7u) * 8;
#pragma unroll
    for (int s0 = 0; s0 < MT; s0 += SLABS) {
#pragma unroll
        for (int s = 0; s < (int)SLABS; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j) *reinterpret_cast<f32x4*>(room + (s * 16 + r16) * PITCH + j * 16 + quarter * 4) = acc[s0 + s][j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (uint32_t p = 0; p < SLABS * 2; ++p) {
            const uint32_t in = p * 8 + (lane >> 3), row = m0 + wm * (BM / WM) + s0 * 16 + in;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(room + in * PITCH + (lane & 7u) * 8), hi = *reinterpret_cast<const f32x4*>(room + in * PITCH + (lane & 7u) * 8 + 4);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (row < a.x.n && col < a.w.n) {
                if (a.parts > 1) store_elements<DT_F32, 8>(a.sums + ((uint64_t)part * a.x.n + row) * a.w.n + col, (int64_t)a.w.n - col, v);
                else finish8<DT>(a.f, row, col, a.w.n, v);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// The parts' sums, added up in their order.
template <int DT>
__global__ void __launch_bounds__(256) dense_join_kernel(DenseArgs a) {
    const uint32_t per_row = (a.w.n + 7) / 8;
    const uint64_t unit = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t row = (uint32_t)(unit / per_row), col = (uint32_t)(unit % per_row) * 8;
    if (row >= a.x.n) return;
    float sum[8] = {};
    for (uint32_t p0 = 0; p0 < a.parts; p0 += 4) {
        float v[4][8];
#pragma unroll
        for (uint32_t p = 0; p < 4; ++p)
            load_elements<DT_F32, 8>(a.sums + ((uint64_t)min(p0 + p, a.parts - 1) * a.x.n + row) * a.w.n + col, (int64_t)a.w.n - col, v[p]);
#pragma unroll
        for (uint32_t p = 0; p < 4; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += p0 + p < a.parts ? v[p][i] : 0.0f;
    }
    finish8<DT>(a.f, row, col, a.w.n, sum);
}

// ---- products of few rows ------------------------------------------------------------
// Both operands along.  A wavefront has 16 columns and every KWAYS-th block of the depth, straight from memory into registers: it asks for AHEAD
// blocks before it multiplies the first.  The KWAYS wavefronts' sums of a column are added up in LDS, in their order.
constexpr int kThinWaves = 8;
template <int DT, int MT, int KWAYS>
__global__ void __launch_bounds__(64 * kThinWaves) dense_thin_kernel(DenseArgs a) {
    constexpr int WAVES = kThinWaves, BM = 16 * MT, BN = 16 * (WAVES / KWAYS), AHEAD = 4;
    constexpr uint32_t SIZE = kSize<DT>, K = kBlock<DT>;
    __shared__ __attribute__((aligned(16))) float sums[WAVES][BM][20];
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_in_block()), r16 = lane & 15u, part = lane >> 4, way = wave % KWAYS;
    const uint32_t m0 = blockIdx.x / a.col_tiles * BM, n0 = blockIdx.x % a.col_tiles * BN, n = n0 + wave / KWAYS * 16;
    const uint32_t steps = (a.depth + K - 1) / K;
    const uint8_t* const w = a.w.p + (int64_t)min(n + r16, a.w.n - 1) * a.w.stride + part * 16;
    const uint8_t* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = a.x.p + (int64_t)min(m0 + i * 16 + r16, a.x.n - 1) * a.x.stride + part * 16;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    const auto load = [&](const uint8_t* row, uint32_t b) MINT_INLINE_LAMBDA {
        Pair<DT> p;
        const int64_t left = ((int64_t)a.depth - (int64_t)b * K) * SIZE - part * 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) p.v[h] = piece_of<SIZE>(row + (int64_t)b * 128 + h * 64, left - h * 64);
        return p;
    };
    const uint32_t full = a.depth / K;
    uint32_t b = way;
    for (; b + (AHEAD - 1) * KWAYS < full; b += AHEAD * KWAYS) {
        Pair<DT> wv[AHEAD], xv[AHEAD][MT];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                wv[u].v[h] = *(MINT_GLOBAL const u32x4_any*)as_global(w + (int64_t)(b + u * KWAYS) * 128 + h * 64);
#pragma unroll
                for (int i = 0; i < MT; ++i) xv[u][i].v[h] = *(MINT_GLOBAL const u32x4_any*)as_global(x[i] + (int64_t)(b + u * KWAYS) * 128 + h * 64);
            }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = Pair<DT>::multiply(wv[u], xv[u][i], acc[i]);
    }
    for (; b < steps; b += KWAYS) {
        const Pair<DT> wv = load(w, b);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = Pair<DT>::multiply(wv, load(x[i], b), acc[i]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) *reinterpret_cast<f32x4*>(&sums[wave][i * 16 + r16][part * 4]) = acc[i];
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < BM * BN / 8; at += 64 * WAVES) {
        const uint32_t m = at / (BN / 8), c = at % (BN / 8) * 8;
        if (m0 + m >= a.x.n || n0 + c >= a.w.n) continue;
        float v[8] = {};
#pragma unroll
        for (int k = 0; k < KWAYS; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += sums[c / 16 * KWAYS + k][m][c % 16 + i];
        finish8<DT>(a.f, m0 + m, n0 + c, a.w.n, v);
    }
}

// ---- the gradient in front of the activation, and the bias's -----------------------------
struct ActivationGradArgs {
    const void *d, *z;                   // z 0: no activation
    void* d_z;                           // 0: not wanted
    float* sums;                         // (groups, cols), or 0
    int64_t d_stride, z_stride, d_z_stride;
    uint32_t rows, cols, chunks, groups;
    int activation;
};
// A wavefront has 512 columns of every groups-th row.
constexpr int kGradWaves = 4;
template <int D, int DT>
__global__ void __launch_bounds__(64 * kGradWaves) activation_grad_kernel(ActivationGradArgs a) {
    const uint64_t unit = (uint64_t)blockIdx.x * kGradWaves + wave_in_block();
    const uint32_t group = (uint32_t)(unit / a.chunks), col = ((uint32_t)(unit % a.chunks) * 64 + lane_id()) * 8;
    if (group >= a.groups || col >= a.cols) return;
    const int64_t left = (int64_t)a.cols - col;
    float sum[8] = {};
    for (uint64_t row = group; row < a.rows; row += a.groups) {
        float d[8], z[8];
        load8<D>(a.d, (int64_t)row * a.d_stride + col, left, d);
        if (a.z) {
            load8<DT>(a.z, (int64_t)row * a.z_stride + col, left, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= slope_of(a.activation, z[i]);
        }
        if (a.d_z) store8<DT>(a.d_z, (int64_t)row * a.d_z_stride + col, left, d);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += d[i];
    }
    if (a.sums) store_elements<DT_F32, 8>(a.sums + (uint64_t)group * a.cols + col, left, sum);
}
// A thread block has 64 columns, and a wavefront every 16th group's sums of them.
constexpr int kBiasWaves = 16;
template <int DT>
__global__ void __launch_bounds__(64 * kBiasWaves) bias_grad_kernel(const float* sums, void* d_bias, uint32_t cols, uint32_t groups) {
    __shared__ float part[kBiasWaves][64];
    const uint32_t col = blockIdx.x * 64 + lane_id(), from = min(col, cols - 1), wave = wave_in_block();
    float sum = 0.0f;
    for (uint32_t g0 = wave; g0 < groups; g0 += kBiasWaves * 8) {
        float v[8];
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) v[u] = *as_global(sums + (uint64_t)min(g0 + u * kBiasWaves, groups - 1) * cols + from);
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) sum += g0 + u * kBiasWaves < groups ? v[u] : 0.0f;
    }
    part[wave][lane_id()] = sum;
    __syncthreads();
    if (wave != 0 || col >= cols) return;
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kBiasWaves; ++w) sum += part[w][lane_id()];
    *as_global(static_cast<typename Elem<DT>::type*>(d_bias) + col) = Elem<DT>::round(sum);
}

// ---- the launches --------------------------------------------------------------------
bool known(int dtype) { return dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32; }
constexpr uint64_t kMost = 0x7FFFFFFF - 256;
uint32_t size_of(int dtype) { return dtype == MINT_F32 ? 4 : 2; }

struct Choice {
    int tile;                    // 0: few rows; else rows of a tile, and its columns
    int cols;
    uint32_t parts;
};
Choice choose(const mint_dense_op& op) {
    const bool along = op.form == MINT_DENSE_PRODUCT;
    if (along && op.rows <= 32) return {0, 0, 1};
    const auto tiles = [&](uint64_t bm, uint64_t bn) { return ceil_div(op.rows, bm) * ceil_div(op.cols, bn); };
    const uint64_t blocks = ceil_div(op.depth * size_of(op.dtype), 128);
    const auto parts = [&](uint64_t n) { return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(256 / std::max<uint64_t>(n, 1), blocks / 8)); };
    if (op.dtype != MINT_F32 && tiles(256, 256) >= 200) return {256, 256, 1};
    if (op.dtype != MINT_F32 && tiles(128, 256) >= 200) return {128, 256, 1};
    if (tiles(128, 128) >= 100) return {128, 128, parts(tiles(128, 128))};
    return {64, 64, parts(tiles(64, 64))};
}
bool direct(const mint_dense_op& op) {
    const int64_t size = size_of(op.dtype);
    // (a stride is looked at only where there is more than one row)
    const uint64_t x_rows = op.form == MINT_DENSE_WEIGHT_GRAD ? op.depth : op.rows, w_rows = op.form == MINT_DENSE_PRODUCT ? op.cols : op.depth;
    return op.x % 16 == 0 && op.w % 16 == 0 && (x_rows <= 1 || op.x_stride * size % 16 == 0) && (w_rows <= 1 || op.w_stride * size % 16 == 0);
}
template <int DT, int BM, int BN, int WM, int STAGES, bool X_ALONG, bool W_ALONG, bool DIRECT>
int go_tiles(DenseArgs a, hipStream_t s) {
    a.row_tiles = (uint32_t)ceil_div(a.x.n, BM);
    a.col_tiles = (uint32_t)ceil_div(a.w.n, BN);
    const uint64_t blocks = ceil_div((uint64_t)a.row_tiles * a.col_tiles * a.parts, 8) * 8;
    if (blocks > 0x7FFFFFFFull / (64 * WM * (BN / 64))) return MINT_ERR_TOO_LARGE;
    return Launch<&dense_kernel<DT, BM, BN, WM, STAGES, X_ALONG, W_ALONG, DIRECT>>::go((uint32_t)blocks, 64 * WM * (BN / 64), 0, s, a);
}
template <int DT, bool X_ALONG, bool W_ALONG>
int go_form(const DenseArgs& a, const Choice& c, bool is_direct, hipStream_t s) {
    if (!is_direct) {
        if (c.tile >= 128) return go_tiles<DT, 128, 128, 4, 1, X_ALONG, W_ALONG, false>(a, s);
        return go_tiles<DT, 64, 64, 4, 1, X_ALONG, W_ALONG, false>(a, s);
    }
    if constexpr (DT != DT_F32) {
        if (c.tile == 256) return go_tiles<DT, 256, 256, 2, 2, X_ALONG, W_ALONG, true>(a, s);
        if (c.cols == 256) return go_tiles<DT, 128, 256, 2, 3, X_ALONG, W_ALONG, true>(a, s);
    }
    if (c.tile == 128) return go_tiles<DT, 128, 128, 4, 3, X_ALONG, W_ALONG, true>(a, s);
    return go_tiles<DT, 64, 64, 4, 4, X_ALONG, W_ALONG, true>(a, s);
}
template <int DT, int MT, int KWAYS>
int go_thin(DenseArgs a, hipStream_t s) {
    a.col_tiles = (uint32_t)ceil_div(a.w.n, 16 * (kThinWaves / KWAYS));
    const uint64_t blocks = ceil_div(a.x.n, 16 * MT) * a.col_tiles;
    if (blocks > 0x7FFFFFFFull / (64 * kThinWaves)) return MINT_ERR_TOO_LARGE;
    return Launch<&dense_thin_kernel<DT, MT, KWAYS>>::go((uint32_t)blocks, 64 * kThinWaves, 0, s, a);
}
template <int DT>
int go_dense(const mint_dense_op& op, const DenseArgs& a, const Choice& c, hipStream_t s) {
    if (c.tile == 0) {
        const bool few = ceil_div(op.cols, 16) <= 768;
        if (op.rows <= 16) return few ? go_thin<DT, 1, 8>(a, s) : go_thin<DT, 1, 2>(a, s);
        return few ? go_thin<DT, 2, 8>(a, s) : go_thin<DT, 2, 2>(a, s);
    }
    const bool is_direct = direct(op);
    int err;
    switch (op.form) {
        case MINT_DENSE_PRODUCT: err = go_form<DT, true, true>(a, c, is_direct, s); break;
        case MINT_DENSE_INPUT_GRAD: err = go_form<DT, true, false>(a, c, is_direct, s); break;
        default: err = go_form<DT, false, false>(a, c, is_direct, s); break;
    }
    if (err != MINT_OK || a.parts == 1) return err;
    const uint64_t blocks = ceil_div((uint64_t)a.x.n * ceil_div(a.w.n, 8), 256);
    if (blocks > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    return Launch<&dense_join_kernel<DT>>::go((uint32_t)blocks, 256, 0, s, a);
}
// groups of rows whose sums a wavefront keeps: as many as fill the device
uint32_t grad_groups(uint64_t rows, uint64_t cols) {
    const uint64_t chunks = ceil_div(cols, 512);
    return (uint32_t)std::min<uint64_t>(rows, std::max<uint64_t>(16, 4096 / std::max<uint64_t>(chunks, 1)));
}

}  // namespace
}  // namespace mint

using namespace mint;

extern "C" size_t mint_dense_workspace(const mint_dense_op* op) {
    if (!op || !known(op->dtype) || op->rows == 0 || op->cols == 0 || op->rows > kMost || op->cols > kMost || op->depth > kMost) return 0;
    const Choice c = choose(*op);
    return c.parts > 1 ? (size_t)c.parts * op->rows * op->cols * 4 : 0;
}

extern "C" int mint_dense(const mint_dense_op* op, void* stream) {
    if (!op || !known(op->dtype) || !(op->out_dtype == op->dtype || op->out_dtype == MINT_F32) || op->form < MINT_DENSE_PRODUCT ||
        op->form > MINT_DENSE_WEIGHT_GRAD || !activation_known(op->activation))
        return MINT_ERR_ARG;
    if (op->form != MINT_DENSE_PRODUCT && (op->bias || op->residual || op->z || op->activation)) return MINT_ERR_ARG;
    if (op->rows > kMost || op->cols > kMost || op->depth > kMost) return MINT_ERR_TOO_LARGE;
    if (op->rows == 0 || op->cols == 0) return MINT_OK;
    if (!op->out || (op->depth && (!op->x || !op->w))) return MINT_ERR_ARG;
    const Choice c = choose(*op);
    const size_t need = mint_dense_workspace(op);
    if (need && (!op->workspace || op->workspace_bytes < need)) return MINT_ERR_STAGING;
    if (need && op->workspace % 16) return MINT_ERR_ALIGN;
    const int64_t size = size_of(op->dtype);
    const DenseArgs a = {{reinterpret_cast<const uint8_t*>(op->x), op->x_stride * size, (uint32_t)op->rows},
                         {reinterpret_cast<const uint8_t*>(op->w), op->w_stride * size, (uint32_t)op->cols},
                         {reinterpret_cast<const void*>(op->bias), reinterpret_cast<const void*>(op->residual), reinterpret_cast<void*>(op->out),
                          reinterpret_cast<void*>(op->z), op->residual_stride, op->out_stride, op->z_stride, op->out_dtype, op->activation},
                         (uint32_t)op->depth, 0, 0, c.parts, reinterpret_cast<float*>(op->workspace)};
    const auto s = static_cast<hipStream_t>(stream);
    switch (op->dtype) {
        case MINT_F16: return go_dense<DT_F16>(*op, a, c, s);
        case MINT_BF16: return go_dense<DT_BF16>(*op, a, c, s);
        default: return go_dense<DT_F32>(*op, a, c, s);
    }
}

extern "C" size_t mint_activation_grad_workspace(uint64_t rows, uint64_t cols) {
    return rows && cols && rows <= kMost && cols <= kMost ? (size_t)grad_groups(rows, cols) * cols * 4 : 0;
}

extern "C" int mint_activation_grad(const mint_activation_grad_op* op, void* stream) {
    if (!op || !known(op->dtype) || !(op->d_dtype == op->dtype || op->d_dtype == MINT_F32) || !activation_known(op->activation)) return MINT_ERR_ARG;
    if (op->rows > kMost || op->cols > kMost) return MINT_ERR_TOO_LARGE;
    if (op->cols == 0) return MINT_OK;
    if (op->rows && (!op->d || (op->activation != MINT_ACT_NONE && !op->z))) return MINT_ERR_ARG;
    const size_t need = op->d_bias ? mint_activation_grad_workspace(op->rows, op->cols) : 0;
    if (need && (!op->workspace || op->workspace_bytes < need)) return MINT_ERR_STAGING;
    if (need && op->workspace % 4) return MINT_ERR_ALIGN;
    const uint32_t chunks = (uint32_t)ceil_div(op->cols, 512), groups = grad_groups(op->rows, op->cols);
    const ActivationGradArgs a = {reinterpret_cast<const void*>(op->d), op->activation != MINT_ACT_NONE ? reinterpret_cast<const void*>(op->z) : nullptr,
                                  reinterpret_cast<void*>(op->d_z), need ? reinterpret_cast<float*>(op->workspace) : nullptr, op->d_stride,
                                  op->z_stride, op->d_z_stride, (uint32_t)op->rows, (uint32_t)op->cols, chunks, groups, op->activation};
    const auto s = static_cast<hipStream_t>(stream);
    const uint64_t blocks = ceil_div((uint64_t)chunks * groups, kGradWaves);
    if (blocks > 0x7FFFFFFFull / (64 * kGradWaves)) return MINT_ERR_TOO_LARGE;
    if (op->rows && (a.d_z || a.sums)) {
        int err;
        switch (op->dtype) {
            case MINT_F16: err = op->d_dtype == MINT_F16 ? Launch<&activation_grad_kernel<DT_F16, DT_F16>>::go((uint32_t)blocks, 64 * kGradWaves, 0, s, a)
                                                         : Launch<&activation_grad_kernel<DT_F32, DT_F16>>::go((uint32_t)blocks, 64 * kGradWaves, 0, s, a); break;
            case MINT_BF16: err = op->d_dtype == MINT_BF16 ? Launch<&activation_grad_kernel<DT_BF16, DT_BF16>>::go((uint32_t)blocks, 64 * kGradWaves, 0, s, a)
                                                           : Launch<&activation_grad_kernel<DT_F32, DT_BF16>>::go((uint32_t)blocks, 64 * kGradWaves, 0, s, a); break;
            default: err = Launch<&activation_grad_kernel<DT_F32, DT_F32>>::go((uint32_t)blocks, 64 * kGradWaves, 0, s, a); break;
        }
        if (err != MINT_OK) return err;
    }
    if (!op->d_bias) return MINT_OK;
    // (of no rows the sums are zeros)
    const float* const sums = a.sums;
    void* const d_bias = reinterpret_cast<void*>(op->d_bias);
    const uint32_t n = op->rows ? groups : 0u, grid = (uint32_t)ceil_div(op->cols, 64);
    switch (op->dtype) {
        case MINT_F16: return Launch<&bias_grad_kernel<DT_F16>>::go(grid, 64 * kBiasWaves, 0, s, sums, d_bias, a.cols, n);
        case MINT_BF16: return Launch<&bias_grad_kernel<DT_BF16>>::go(grid, 64 * kBiasWaves, 0, s, sums, d_bias, a.cols, n);
        default: return Launch<&bias_grad_kernel<DT_F32>>::go(grid, 64 * kBiasWaves, 0, s, sums, d_bias, a.cols, n);
    }
}
