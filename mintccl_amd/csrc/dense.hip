// Dense matrix products in 16 and 32 bits with what surrounds them, and their gradients.
//
//   z = x w^T + b      out = residual + a(z)
//   d_z = d a'(z)      d_b = sum over rows of d_z      d_x = d_z w      d_w = d_z^T x
//
// The three products are one kernel: the result's rows come from one operand, its columns from the other, and each of them
// lies in memory either with the depth along its rows ("along": x and w of the first product) or across them ("across": w of d_x, both
// of d_w).  Sums are in 32 bits in a fixed order; out is rounded once to its own type, and z and d_z once each to the operands': d_z is an operand, which the matrix
// instructions take in 16 bits, and z the largest thing that is kept (in 32 bits it would be twice the bytes, written and read again).  In bf16 gradients are then 2.4e-3
// off in 2-norm for the 1.7e-3 that their own rounding makes (8192 x 8192 x 4096, silu).
#include "activations.hpp"

#include <algorithm>

namespace mint {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// 16 bytes of an operand's row or column, of which four lanes have a step's part of the depth, as the matrix instructions take them: in 32 bits
// number T of them, else all.
template <int DT>
constexpr int kTurns = DT == DT_F32 ? 4 : 1;
template <int DT, int T>
__device__ __forceinline__ f32x4 multiply_add(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == DT_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (DT == DT_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[T]), __uint_as_float(b[T]), c, 0, 0, 0);
}
// c[n] += a[n] b for N sums, one behind the other (those of one sum would wait for each other)
template <int DT, int N>
__device__ __forceinline__ void multiply_add(const u32x4 (&a)[N], u32x4 b, f32x4 (&c)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) c[n] = multiply_add<DT, 0>(a[n], b, c[n]);
    if constexpr (kTurns<DT> > 1) {
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = multiply_add<DT, 1>(a[n], b, c[n]);
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = multiply_add<DT, 2>(a[n], b, c[n]);
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = multiply_add<DT, 3>(a[n], b, c[n]);
    }
}
template <int DT>
constexpr uint32_t kSize = sizeof(typename Elem<DT>::type);
template <int DT>
constexpr uint32_t kHalf = 64 / kSize<DT>;              // numbers of the depth that go by in a step
template <int DT>
constexpr uint32_t kBlock = 2 * kHalf<DT>;              // ... and in a block, two steps

using LdsBytes = MINT_LDS uint8_t*;
// 16 bytes of a lane's own, at a 32-bit offset from where the wavefront's are, into LDS, the lanes' side by side.  (By the buffer's form: for
// the global one the compiler holds every read of LDS back until all such loads, and all reads, are done.)
__device__ __forceinline__ void to_lds16(const uint8_t* from, uint32_t offset, LdsBytes to) {
    const auto whole = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(from), 0, 0xFFFFFFFFu, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(whole, (MINT_LDS void*)to, 16, offset, 0, 0, 0);
}
__device__ __forceinline__ u32x4 lds16(LdsBytes at) { return *(MINT_LDS const u32x4*)at; }
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
// All but the N latest of a wavefront's loads are done.
template <int N>
__device__ __forceinline__ void wait_loads() {
    compiler_fence();
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 15 << 8);
    compiler_fence();
}
// All wavefronts meet, what they read from LDS and wrote there behind them.
__device__ __forceinline__ void meet() {
    compiler_fence();
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);          // (LDS only)
    __builtin_amdgcn_s_barrier();
    compiler_fence();
}

// An operand: `n` rows or columns of the result.  ALONG: row i of it at p + i * stride, the depth along it; else depth d at p + d * stride.
struct Side {
    const uint8_t* p;
    int64_t stride;              // bytes
    uint32_t n;
};
// B of them in LDS, a part of the depth, in pieces of 16 bytes.
//   along    a block: a row of 128 bytes for each of them, its pieces turned so that the 16 lanes that a 16-byte read serves together (0 - 3,
//            12 - 15 and 20 - 27 of 32, then the others; 16 lanes side by side are 16 rows) are on different banks.  (Half a block at a time would
//            be 64 bytes of a row with each request: 8192 x 8192 x 4096 485 us for 440)
//   across   a step's half: a row of B numbers for each number of the depth; a lane's numbers of one column are gathered by the
//            transposing reads (16 bits: 16 lanes have four rows of 16 numbers), or one by one (32 bits).  Which 16 numbers lie
//            where in a row is turned by the row's number, so that those reads have different banks too
template <int DT, int B, bool ALONG>
struct Staged {
    static constexpr uint32_t SIZE = kSize<DT>, PIECES = ALONG ? 8 : B * SIZE / 16, BYTES = B * (ALONG ? 128 : 64);
    static __device__ __forceinline__ uint32_t turn(uint32_t row) {
        if constexpr (ALONG) return (row >> 1) & 7u;
        else if constexpr (SIZE == 4) return (row >> 2 & 3u) * 4;
        else if constexpr (PIECES == 8) return ((row >> 1 & 1u) | (row >> 2 & 2u)) * 2;
        else return ((row & 3u) | (row >> 1 & 4u)) * 2;
    }
    // where 16 bytes in LDS, the u-th, come from: their row and their piece of that row
    static __device__ __forceinline__ uint32_t row_of(uint32_t u) { return u / PIECES; }
    static __device__ __forceinline__ uint32_t piece_of(uint32_t u) { return (u % PIECES) ^ turn(u / PIECES); }

    // A lane's part of the g-th 16 of them, of a half of the depth's block.
    uint32_t base;               // along: the lane's piece of the first 16; across: the lane's numbers of its row's first 16
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
            const uint32_t row = part * 8 + (r16 >> 2);          // (4 rows on the turning is the same)
            base = row * (B * 2) + (r16 & 3u) * 8;
            turned = turn(row) / 2;
        }
    }
    __device__ __forceinline__ u32x4 load(LdsBytes at, uint32_t g, uint32_t half) const {
        if constexpr (ALONG) {
            return lds16(at + (g * 2048 + (base ^ half * 64)));
        } else if constexpr (SIZE == 4) {
            const LdsBytes from = at + (base + (g ^ turned) * 64);
            u32x4 v;
#pragma unroll
            for (int t = 0; t < 4; ++t) v[t] = *(MINT_LDS const uint32_t*)(from + t * (B * 4));
            return v;
        } else {
            const LdsBytes from = at + (base + (g ^ turned) * 32);
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MINT_LDS i16x4*)from));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MINT_LDS i16x4*)(from + 4 * (B * 2))));
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        }
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
template <int DT>
__device__ __forceinline__ void bias8(const Finish& f, uint32_t col, uint32_t cols, float (&bias)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bias[i] = 0.0f;
    if (f.bias && col < cols) load8<DT>(f.bias, col, (int64_t)cols - col, bias);
}
template <int DT>
__device__ __forceinline__ void residual8(const Finish& f, uint32_t row, uint32_t col, uint32_t cols, float (&more)[8]) {
    const int64_t left = (int64_t)cols - col;
    if (f.out_dtype == MINT_F32) load8<DT_F32>(f.residual, (int64_t)row * f.residual_stride + col, left, more);
    else load8<DT>(f.residual, (int64_t)row * f.residual_stride + col, left, more);
}
// Eight sums of a row of the result become what is stored.  Results are of the operands' type or in 32 bits.
template <int DT>
__device__ __forceinline__ void finish8(const Finish& f, uint32_t row, uint32_t col, uint32_t cols, const float (&bias)[8], const float (&more)[8], float (&v)[8]) {
    const int64_t left = (int64_t)cols - col;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += bias[i];
    if (f.z) store8<DT>(f.z, (int64_t)row * f.z_stride + col, left, v);
    if (f.activation != MINT_ACT_NONE) activate(f.activation, v);
    if (f.residual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += more[i];
    }
    if (f.out_dtype == MINT_F32) store8<DT_F32>(f.out, (int64_t)row * f.out_stride + col, left, v);
    else store8<DT>(f.out, (int64_t)row * f.out_stride + col, left, v);
}

struct DenseArgs {
    Side x, w;                           // the result's rows and columns
    Finish f;
    uint32_t depth, row_tiles, col_tiles;
    uint32_t parts;                      // thread blocks that share a tile's depth; more than one: their sums go to
    float* sums;                         // (parts, rows, cols)
};

// One operand of a tile, on its way from memory into a ring of N places in LDS.  A unit is a block of the depth (along) or half of one.
template <int DT, int B, int WAVES, int N, bool ALONG>
struct Ring {
    using S = Staged<DT, B, ALONG>;
    static constexpr int EACH = S::BYTES / 1024 / WAVES;         // instructions of a wavefront for a unit
    static constexpr uint32_t SIZE = kSize<DT>, UNIT = ALONG ? kBlock<DT> : kHalf<DT>, BYTES = S::BYTES;
    static_assert(EACH * 1024 * WAVES == BYTES, "every wavefront brings as much");
    const uint8_t* from;         // the unit to ask for, the same for the wavefront ...
    uint32_t at[EACH];           // ... and what the lane brings of it
    int64_t stride;
    uint32_t left;               // of the depth, from that unit on
    uint32_t wave, lane;
    LdsBytes base, ask;

    __device__ __forceinline__ uint32_t unit(int n) const { return (wave * EACH + n) * 64 + lane; }
    __device__ __forceinline__ Ring(const Side& s, uint32_t first, uint32_t depth0, uint32_t depth, LdsBytes to, uint32_t w, uint32_t l)
        : stride(s.stride), left(depth), wave(w), lane(l), base(to), ask(to) {
        from = ALONG ? s.p + (int64_t)first * stride + (int64_t)depth0 * SIZE : s.p + (int64_t)depth0 * stride + (int64_t)first * SIZE;
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const uint32_t row = S::row_of(unit(n)), piece = S::piece_of(unit(n)) * 16;
            // (rows behind the operand's last one: that one instead; in the place of a piece behind a row's last one, that one)
            at[n] = ALONG ? min(row, s.n - 1 - first) * (uint32_t)stride + piece : row * (uint32_t)stride + min(piece, (min(s.n - first, 4096u) * SIZE - 1) / 16 * 16);
        }
    }
    __device__ __forceinline__ LdsBytes on(LdsBytes p) const { return p + BYTES == base + N * BYTES ? base : p + BYTES; }
    __device__ __forceinline__ void advance() {
        from += ALONG ? 128 : (int64_t)UNIT * stride;
        left -= min(left, UNIT);
        ask = on(ask);
    }
    // piece n of a whole unit, into `to`; the last one goes on
    __device__ __forceinline__ void bring(LdsBytes to, int n) {
        to_lds16(from, at[n], to + (wave * EACH + n) * 1024);
        if (n == EACH - 1) advance();
    }
    // All of a unit that may not be whole: what lies behind the depth comes from the unit's beginning.  The depth's units behind its last number are
    // cleared only.  Its own pieces are cleared, when they are there, by whoever brought them; `there` is what it has.
    __device__ __forceinline__ void bring_any(LdsBytes to, uint32_t& there) {
        there = left;
        if (left) {
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                const uint32_t row = S::row_of(unit(n)), piece = S::piece_of(unit(n)) * 16;
                const uint32_t back = ALONG ? piece < min(left, UNIT) * SIZE ? 0u : piece : row < left ? 0u : row * (uint32_t)stride;
                to_lds16(from, at[n] - back, to + (wave * EACH + n) * 1024);
            }
        }
        advance();
    }
    __device__ __forceinline__ void clear(LdsBytes to, uint32_t there) const {
        if (there >= UNIT) return;
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const auto v = (MINT_LDS u32x4*)(to + unit(n) * 16);
            const int64_t bytes = ALONG ? (int64_t)(there * SIZE) - S::piece_of(unit(n)) * 16 : S::row_of(unit(n)) < there ? 16 : 0;
            *v = first_of(*v, bytes);
        }
    }
};

// A thread block has BM rows and BN columns of the result, a wavefront BM / WM rows and 64 columns of them.  The depth goes by in blocks of
// 128 bytes, two steps each, in rings of NX and NW places.  In a step
//   - what the last step read of x last is multiplied, while the first of this one is read: no one waits behind the meeting
//   - the rest follows, each operand read some products ahead, and w's for the next step
//   - units of x NX - 1 on and of w NW on are asked for, into places that are no longer read: w's of a step has been read before it
// and at its end the wavefronts meet when what the next step reads has come: asked for two steps before and more.  DIRECT: rows in memory
// begin at multiples of 16 bytes (or were copied there), and their pieces go straight into LDS; else they pass through registers, a block at a time.
template <int DT, int BM, int BN, int WM, int NX, int NW, bool X_ALONG, bool W_ALONG>
struct Tile {
    static constexpr int WN = BN / 64, WAVES = WM * WN, MT = BM / WM / 16, NT = 4;
    static constexpr int LAG = MT > 2 ? 2 : 1;                            // rows of products that are left to the next step
    static constexpr uint32_t K = kBlock<DT>;
    using X = Ring<DT, BM, WAVES, NX, X_ALONG>;
    using W = Ring<DT, BN, WAVES, NW, W_ALONG>;
    static constexpr uint32_t kStages = NX * X::BYTES + NW * W::BYTES;
    static constexpr uint32_t SLABS = MT < 4 ? MT : 4, PITCH = 68;        // of the sums' way out: slabs of 16 rows of 64 columns
    static constexpr uint32_t kOut = WAVES * SLABS * 16 * PITCH * 4;

    // What is asked for in a step (0: a block's first), x's before w's, and how much of it may be on its way when the step ends.
    static constexpr int asks_x(int step) { return X_ALONG ? (step & 1 ? 0 : X::EACH) : X::EACH; }
    static constexpr int asks_w(int step) { return W_ALONG ? (step & 1 ? W::EACH : 0) : W::EACH; }
    static constexpr int later(int first, int end) {                      // asked in steps [first, end]
        int n = 0;
        for (int s = first; s <= end; ++s) n += asks_x(s & 1) + asks_w(s & 1);
        return n;
    }
    static constexpr int under_way(int step) {
        const int s = 64 + step;                                          // (any block)
        int most = 63;
        // w of step s + 2 is read in the next step, x of step s + 1 too
        const int w_asked = W_ALONG ? (step ? -1 : s + 3 - 2 * NW) : s + 2 - NW, x_asked = X_ALONG ? (step ? s + 3 - 2 * NX : -1) : s + 2 - NX;
        if (w_asked >= 0 && later(w_asked + 1, s) < most) most = later(w_asked + 1, s);
        if (x_asked >= 0 && later(x_asked + 1, s) + asks_w(x_asked & 1) < most) most = later(x_asked + 1, s) + asks_w(x_asked & 1);
        return most;
    }
    // blocks that are asked for ahead of the one at work
    static constexpr int x_ahead = X_ALONG ? NX - 1 : NX / 2, w_ahead = W_ALONG ? NW : (NW + 1) / 2, LEAD = x_ahead > w_ahead ? x_ahead : w_ahead;

    const DenseArgs& a;
    uint32_t lane, wave, m0, n0, depth0, depth, blocks;
    typename X::S sx;
    typename W::S sw;
    f32x4 acc[MT][NT];

    __device__ __forceinline__ uint32_t wm() const { return wave / WN; }
    __device__ __forceinline__ uint32_t wn() const { return wave % WN; }
    // part `part` of `parts`: whole blocks of the depth, as many for each (some may be behind its end); the last of all may not be whole
    __device__ __forceinline__ Tile(const DenseArgs& args, uint32_t m, uint32_t n, uint32_t part, uint32_t parts)
        : a(args), lane(lane_id()), wave(__builtin_amdgcn_readfirstlane(wave_in_block()) % WAVES), m0(m), n0(n), sx(lane), sw(lane) {
        blocks = ((a.depth + K - 1) / K + parts - 1) / parts;
        depth0 = min(part * blocks * K, a.depth);
        depth = min(blocks * K, a.depth - depth0);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ u32x4 load_x(LdsBytes at, int i, uint32_t half) const { return sx.load(at, wm() * MT + i, half); }
    __device__ __forceinline__ u32x4 load_w(LdsBytes at, int j, uint32_t half) const { return sw.load(at, wn() * 4 + j, half); }
    __device__ __forceinline__ void products(int i, const u32x4 (&w)[NT], u32x4 x) {
        multiply_add<DT, NT>(w, x, acc[i]);
        __builtin_amdgcn_sched_barrier(0);
    }
    // A step: of the block at x_at with `w`, which has been read.  `before` has w of the step before, which is still wanted for what it left (in `lag`), and
    // takes that of the next one, at w_at.
    template <typename F>
    __device__ __forceinline__ void step(LdsBytes x_at, uint32_t x_half, LdsBytes w_at, uint32_t w_half, u32x4 (&w)[NT], u32x4 (&before)[NT], u32x4 (&lag)[LAG],
                                         int asks, const F& meanwhile) {
        constexpr int FIRST = MT > LAG ? LAG + 1 : MT, SLOTS = MT > LAG ? MT - LAG : 1, READS = SLOTS > 2 ? (NT + SLOTS - 2) / (SLOTS - 1) : NT;
        u32x4 x[MT];
#pragma unroll
        for (int i = 0; i < FIRST; ++i) x[i] = load_x(x_at, i, x_half);
        const int pieces = (asks + SLOTS - 1) / SLOTS;
#pragma unroll
        for (int i = 0; i < LAG; ++i) products(MT - LAG + i, before, lag[i]);
        // (nothing is read during the last products: the meeting waits for the reads, so that what is asked for behind it may lie where they read)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            if (i + FIRST < MT) x[i + FIRST] = load_x(x_at, i + FIRST, x_half);
            // (the loads go out between the products: all at once they would stand in each other's way)
#pragma unroll
            for (int n = 0; n < pieces; ++n)
                if (i * pieces + n < asks) meanwhile(i * pieces + n);
#pragma unroll
            for (int n = 0; n < READS; ++n)
                if (i * READS + n < NT) before[i * READS + n] = load_w(w_at, i * READS + n, w_half);
            if (i < MT - LAG) products(i, w, x[i]);
        }
#pragma unroll
        for (int i = 0; i < LAG; ++i) lag[i] = x[MT - LAG + i];
    }
    // The two steps of a block, where all that they ask for is whole.  Reads are from four places (a block along the depth has two of them alike), what is
    // asked for goes to four; w's of the second step may be where the first one read, behind a meeting.  That no read is of what is on
    // its way is what the compiler has to know, or it waits for all of that.
    __device__ __forceinline__ void block(X& rx, W& rw, LdsBytes __restrict x0, LdsBytes __restrict x1, LdsBytes __restrict w0, LdsBytes __restrict w1,
                                          LdsBytes __restrict to_x0, LdsBytes __restrict to_x1, LdsBytes __restrict to_w0, LdsBytes __restrict to_w1,
                                          u32x4 (&w)[NT], u32x4 (&other)[NT], u32x4 (&lag)[LAG]) {
        step(x0, 0, w0, 1, w, other, lag, asks_x(0) + asks_w(0), [&](int n) MINT_INLINE_LAMBDA {
            if (n < asks_x(0)) rx.bring(to_x0, n);
            else rw.bring(to_w0, n - asks_x(0));
        });
        wait_loads<under_way(0)>();
        meet();
        step(x1, 1, w1, 0, other, w, lag, asks_x(1) + asks_w(1), [&](int n) MINT_INLINE_LAMBDA {
            if (n < asks_x(1)) rx.bring(to_x1, n);
            else rw.bring(to_w1, n - asks_x(1));
        });
        wait_loads<under_way(1)>();
        meet();
    }
    __device__ __forceinline__ void run_direct(LdsBytes lds) {
        const uint32_t full = depth / K;
        if (!blocks) return;
        X rx(a.x, m0, depth0, depth, lds, wave, lane);
        W rw(a.w, n0, depth0, depth, lds + NX * X::BYTES, wave, lane);
        const auto bring_x = [&]() MINT_INLINE_LAMBDA {
            const LdsBytes to = rx.ask;
            uint32_t there;
            rx.bring_any(to, there);
            return there;
        };
        {
            uint32_t x_there[NX - 1], w_there[NW];
#pragma unroll
            for (int u = 0; u < NX - 1; ++u) x_there[u] = bring_x();
#pragma unroll
            for (int u = 0; u < NW; ++u) {
                const LdsBytes to = rw.ask;
                rw.bring_any(to, w_there[u]);
            }
            wait_loads<0>();
#pragma unroll
            for (int u = 0; u < NX - 1; ++u) rx.clear(rx.base + u * X::BYTES, x_there[u]);
#pragma unroll
            for (int u = 0; u < NW; ++u) rw.clear(rw.base + u * W::BYTES, w_there[u]);
        }
        meet();
        u32x4 w[NT], other[NT], lag[LAG];
        LdsBytes x_at = rx.base, w_at = rw.base;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            w[j] = load_w(w_at, j, 0);
            other[j] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < LAG; ++i) lag[i] = u32x4{0, 0, 0, 0};
        meet();
        uint32_t b = 0;
#pragma unroll 1
        for (; b + LEAD < full; ++b) {
            const LdsBytes x1 = X_ALONG ? x_at : rx.on(x_at), w0 = W_ALONG ? w_at : rw.on(w_at), w1 = rw.on(w0);
            // (where a unit is a block one of the two steps asks for it)
            const LdsBytes to_x0 = rx.ask, to_x1 = rx.on(to_x0), to_w0 = rw.ask, to_w1 = W_ALONG ? to_w0 : rw.on(to_w0);
            block(rx, rw, x_at, x1, w0, w1, to_x0, to_x1, to_w0, to_w1, w, other, lag);
            x_at = rx.on(x1);
            w_at = w1;
        }
        // the last blocks: what they ask for, if anything, may not be whole, and everything is waited for
#pragma unroll 1
        for (; b < blocks; ++b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const LdsBytes to_x = rx.ask, to_w = rw.ask;
                uint32_t x_there = X::UNIT, w_there = W::UNIT;
                if (asks_x(h)) rx.bring_any(to_x, x_there);
                if (asks_w(h)) rw.bring_any(to_w, w_there);
                const LdsBytes next_w = W_ALONG && h == 0 ? w_at : rw.on(w_at);
                step(x_at, h, next_w, 1 - h, h ? other : w, h ? w : other, lag, 0, [](int) MINT_INLINE_LAMBDA {});
                wait_loads<0>();
                rx.clear(to_x, x_there);
                rw.clear(to_w, w_there);
                meet();
                if (!X_ALONG || h) x_at = rx.on(x_at);
                w_at = next_w;
            }
        }
#pragma unroll
        for (int i = 0; i < LAG; ++i) products(MT - LAG + i, other, lag[i]);
    }
    // (the places: two blocks in turn, so that there is one meeting to a block)
    static constexpr uint32_t kHeldX = BM * 128, kHeld = (BM + BN) * 128;
    __device__ __forceinline__ void run_held(LdsBytes lds) {
        constexpr uint32_t SIZE = kSize<DT>;
        constexpr int XI = BM / 8 / WAVES, WI = BN / 8 / WAVES;          // pieces of a lane
        u32x4 held[XI + WI];
        // of the u-th 16 bytes of an operand's block: its row and piece (across: the second half's behind the first one's)
        const auto fetch = [&](uint32_t b) MINT_INLINE_LAMBDA {
            const uint32_t d0 = depth0 + b * K;                          // (the depth from here on)
            const auto one = [&](const Side& s, bool along, uint32_t first, uint32_t row, uint32_t piece) MINT_INLINE_LAMBDA {
                if (along)
                    return ::mint::piece_of<SIZE>(s.p + (int64_t)min(first + row, s.n - 1) * s.stride + ((int64_t)d0 * SIZE + piece * 16),
                                                  ((int64_t)(depth0 + depth) - d0) * SIZE - piece * 16);
                const int64_t left = ((int64_t)s.n - first) * SIZE - piece * 16;
                return ::mint::piece_of<SIZE>(s.p + (int64_t)min(d0 + row, a.depth - 1) * s.stride + ((int64_t)first * SIZE + piece * 16),
                                              d0 + row < depth0 + depth ? left : 0);
            };
#pragma unroll
            for (int n = 0; n < XI; ++n) {
                const uint32_t u = (wave * XI + n) * 64 + lane;
                held[n] = one(a.x, X_ALONG, m0, X::S::row_of(u), X::S::piece_of(u));
            }
#pragma unroll
            for (int n = 0; n < WI; ++n) {
                const uint32_t u = (wave * WI + n) * 64 + lane;
                held[XI + n] = one(a.w, W_ALONG, n0, W::S::row_of(u), W::S::piece_of(u));
            }
        };
        if (blocks) fetch(0);
#pragma unroll 1
        for (uint32_t b = 0; b < blocks; ++b) {
            const LdsBytes at = lds + (b & 1u) * kHeld;
#pragma unroll
            for (int n = 0; n < XI; ++n) *(MINT_LDS u32x4*)(at + ((wave * XI + n) * 64 + lane) * 16) = held[n];
#pragma unroll
            for (int n = 0; n < WI; ++n) *(MINT_LDS u32x4*)(at + (kHeldX + ((wave * WI + n) * 64 + lane) * 16)) = held[XI + n];
            __syncthreads();
            if (b + 1 < blocks) fetch(b + 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 w[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) w[j] = load_w(at + (kHeldX + (W_ALONG ? 0 : h * BN * 64)), j, h);
#pragma unroll
                for (int i = 0; i < MT; ++i) products(i, w, load_x(at + (X_ALONG ? 0 : h * BM * 64), i, h));
            }
        }
    }
};

// SPLIT sets of wavefronts, each with a part of the depth and LDS of its own, where tiles leave few wavefronts on a compute unit; their sums are
// added up in LDS, in the parts' order.
//
// Bound by the matrix instructions where there are tiles enough for all compute units, then by the last round of tiles and its way out.  bf16, 8192 x 8192 x
// 4096: x w^T 440 us (1.25 PFLOP/s), d_z w 428, d_z^T x 446 (a library's 436, 436, 496); with bias, an activation of the result and z stored 460.
// 2048 x 4096 x 4096 with a residual and a result in 32 bits 73 (the library's bare product 60): one round of tiles, whose way out no other hides.  f32, 4096 x 256 x
// 4096: 67 (128 TFLOP/s; its four sets' sums added up and stored by one of them 69.6; the library's 69), in the first milliseconds of work 75 (the library's 80).  f32
// with the depth across, 4096^3: x w^T 942 us, d_z w 954, d_z^T x 971 (146, 144 and 142 TFLOP/s, the library 915 each): four reads of LDS for one.
// Not direct, 50 x 5001 x 2500 f16: 13.4, and 5.3 for the parts' sums (a library's 20.2).
template <int DT, int BM, int BN, int WM, int NX, int NW, int SPLIT, bool X_ALONG, bool W_ALONG, bool DIRECT>
__global__ void __launch_bounds__(64 * WM * (BN / 64) * SPLIT) dense_kernel(DenseArgs a) {
    using T = Tile<DT, BM, BN, WM, NX, NW, X_ALONG, W_ALONG>;
    constexpr uint32_t SLABS = T::SLABS, PITCH = T::PITCH, kRoom = DIRECT ? T::kStages : 2 * T::kHeld;
    constexpr uint32_t kRows = BM / WM, kAll = SPLIT * T::WAVES * kRows * PITCH * 4, kOut = SPLIT > 1 ? kAll : T::kOut;
    constexpr uint32_t kLds = SPLIT * kRoom > kOut ? SPLIT * kRoom : kOut;
    static_assert(kLds <= 160 * 1024, "it fits LDS");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    // The hardware deals thread blocks to the eight XCDs in turn: each takes an eighth of the tiles that lie together, in
    // columns of GROUP row tiles, so that those at work at a time share operands in its L2.
    constexpr uint32_t GROUP = 4;
    const uint32_t total = a.row_tiles * a.col_tiles * a.parts, xcd = blockIdx.x & 7u, nth = blockIdx.x >> 3;
    if (nth >= total / 8 + (xcd < total % 8)) return;
    const uint32_t all_id = xcd * (total / 8) + min(xcd, total % 8) + nth, id = all_id / a.parts, part = all_id % a.parts;
    const uint32_t group = id / (GROUP * a.col_tiles), in_group = id % (GROUP * a.col_tiles), height = min(GROUP, a.row_tiles - group * GROUP);
    const uint32_t m0 = (group * GROUP + in_group % height) * BM, n0 = in_group / height * BN;
    const uint32_t way = SPLIT > 1 ? (uint32_t)__builtin_amdgcn_readfirstlane(wave_in_block()) / T::WAVES : 0u;
    T t(a, m0, n0, part * SPLIT + way, a.parts * SPLIT);
    if constexpr (DIRECT) t.run_direct((LdsBytes)lds + way * kRoom);
    else t.run_held((LdsBytes)lds + way * kRoom);
    if constexpr (SPLIT > 1) {
        // All sets' sums go to LDS, and all of their threads add up eight of a row at a time.
        constexpr int THREADS = 64 * T::WAVES * SPLIT, UNITS = BM * BN / 8 / THREADS;
        static_assert(UNITS * THREADS * 8 == BM * BN, "every thread has as many");
        float* const all = reinterpret_cast<float*>(lds);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T::MT; ++i)
#pragma unroll
            for (int j = 0; j < T::NT; ++j)
                *reinterpret_cast<f32x4*>(all + ((way * T::WAVES + t.wave) * kRows + i * 16 + (t.lane & 15u)) * PITCH + j * 16 + (t.lane >> 4) * 4) = t.acc[i][j];
        __syncthreads();
        const uint32_t eight = threadIdx.x % (BN / 8), col = n0 + eight * 8;
        if (col >= a.w.n) return;
        float bias[8];
        bias8<DT>(a.f, col, a.w.n, bias);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const uint32_t in = u * (THREADS / (BN / 8)) + threadIdx.x / (BN / 8), row = m0 + in;
            if (row >= a.x.n) return;
            float more[8], v[8] = {};
            if (a.f.residual && a.parts == 1) residual8<DT>(a.f, row, col, a.w.n, more);
#pragma unroll
            for (int k = 0; k < SPLIT; ++k) {
                const float* const from = all + ((k * T::WAVES + in / kRows * T::WN + eight / 8) * kRows + in % kRows) * PITCH + (eight & 7u) * 8;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += i < 4 ? lo[i & 3] : hi[i & 3];
            }
            if (a.parts > 1) store_elements<DT_F32, 8>(a.sums + ((uint64_t)part * a.x.n + row) * a.w.n + col, (int64_t)a.w.n - col, v);
            else finish8<DT>(a.f, row, col, a.w.n, bias, more, v);
        }
        return;
    }

    // The sums' way out: a lane has four columns of 16 rows each; through LDS it gets eight of a row, and eight lanes side by side 64.
    __syncthreads();
    const uint32_t lane = t.lane;
    float* const room = reinterpret_cast<float*>(lds) + t.wave * (SLABS * 16 * PITCH);
    const uint32_t r16 = lane & 15u, quarter = lane >> 4, col = n0 + t.wn() * 64 + (lane & 7u) * 8, row0 = m0 + t.wm() * (BM / WM) + (lane >> 3);
    float bias[8];
    bias8<DT>(a.f, col, a.w.n, bias);
#pragma unroll
    for (int s0 = 0; s0 < T::MT; s0 += SLABS) {
#pragma unroll
        for (int s = 0; s < (int)SLABS; ++s)
#pragma unroll
            for (int j = 0; j < T::NT; ++j) *reinterpret_cast<f32x4*>(room + (s * 16 + r16) * PITCH + j * 16 + quarter * 4) = t.acc[s0 + s][j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // two rows at a time, so that what they read is asked for together
#pragma unroll 1
        for (uint32_t p = 0; p < SLABS * 2; p += 2) {
            float more[2][8], v[2][8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t in = (p + u) * 8, row = row0 + s0 * 16 + in;
                const float* const from = room + (in + (lane >> 3)) * PITCH + (lane & 7u) * 8;
                const f32x4 lo = *reinterpret_cast<const f32x4*>(from), hi = *reinterpret_cast<const f32x4*>(from + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[u][i] = i < 4 ? lo[i & 3] : hi[i & 3];
                if (a.f.residual && a.parts == 1 && row < a.x.n && col < a.w.n) residual8<DT>(a.f, row, col, a.w.n, more[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t row = row0 + s0 * 16 + (p + u) * 8;
                if (row >= a.x.n || col >= a.w.n) continue;
                if (a.parts > 1) store_elements<DT_F32, 8>(a.sums + ((uint64_t)part * a.x.n + row) * a.w.n + col, (int64_t)a.w.n - col, v[u]);
                else finish8<DT>(a.f, row, col, a.w.n, bias, more[u], v[u]);
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
    float sum[8] = {}, bias[8], more[8];
    bias8<DT>(a.f, col, a.w.n, bias);
    if (a.f.residual) residual8<DT>(a.f, row, col, a.w.n, more);
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
    finish8<DT>(a.f, row, col, a.w.n, bias, more, sum);
}

// ---- operands at any address ------------------------------------------------------------
// Rows, copied to multiples of 16 bytes, zeros behind their ends.  Both operands of a product in one launch.  Bound by memory: 4096 x 4095 numbers of 16
// bits each, 134 MB read and written, 26 us, 5.2 TB/s.
struct Copy {
    const uint8_t* from;
    uint8_t* to;
    int64_t stride;
    uint32_t bytes, pieces, units;       // of a row: its length, 16 bytes each; all rows' pieces (0: nothing to do)
};
constexpr int kCopies = 4;               // pieces of a thread
template <uint32_t SIZE>
__global__ void __launch_bounds__(256) copy_kernel(Copy x, Copy w) {
    u32x4 v[kCopies];
    uint8_t* to[kCopies];
#pragma unroll
    for (int u = 0; u < kCopies; ++u) {
        const uint64_t unit = (uint64_t)blockIdx.x * (256 * kCopies) + u * 256 + threadIdx.x;
        const Copy& c = unit < x.units ? x : w;
        const uint64_t at = unit < x.units ? unit : unit - x.units;
        to[u] = nullptr;
        if (at >= c.units) continue;
        const uint32_t row = (uint32_t)at / c.pieces, piece = (uint32_t)at % c.pieces;
        v[u] = piece_of<SIZE>(c.from + row * c.stride + (uint64_t)piece * 16, (int64_t)c.bytes - (int64_t)piece * 16);
        to[u] = c.to + at * 16;
    }
#pragma unroll
    for (int u = 0; u < kCopies; ++u)
        if (to[u]) *(MINT_GLOBAL u32x4*)as_global(to[u]) = v[u];
}

// ---- products of few rows ------------------------------------------------------------
// Both operands along.  A wavefront has 16 columns and one of KWAYS parts of the depth, straight from memory into registers: it asks for AHEAD
// blocks before it multiplies the first.  The KWAYS wavefronts' sums of a column are added up in LDS, in their order.  Bound by w's bytes: one row,
// 4096 columns of 4096 bf16 numbers 9 us, 3.7 TB/s (64 rows, through tiles and LDS, 15.4).
constexpr int kThinWaves = 8;
template <int DT, int MT, int KWAYS>
__global__ void __launch_bounds__(64 * kThinWaves) dense_thin_kernel(DenseArgs a) {
    constexpr int WAVES = kThinWaves, BM = 16 * MT, BN = 16 * (WAVES / KWAYS), AHEAD = 8;
    constexpr uint32_t SIZE = kSize<DT>, K = kHalf<DT>;
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
        return piece_of<SIZE>(row + (int64_t)b * 64, ((int64_t)a.depth - (int64_t)b * K) * SIZE - part * 16);
    };
    // (a wavefront's are side by side: two of them are a line of memory)
    const uint32_t share = (steps + KWAYS * 2 - 1) / (KWAYS * 2) * 2, full = a.depth / K, end = min(way * share + share, steps), whole = min(end, full);
    uint32_t b = way * share;
    for (; b + AHEAD <= whole; b += AHEAD) {
        u32x4 wv[AHEAD], xv[AHEAD][MT];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            wv[u] = *(MINT_GLOBAL const u32x4_any*)as_global(w + (int64_t)(b + u) * 64);
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[u][i] = *(MINT_GLOBAL const u32x4_any*)as_global(x[i] + (int64_t)(b + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) multiply_add<DT, MT>(xv[u], wv[u], acc);
    }
    for (; b < end; ++b) {
        const u32x4 wv = load(w, b);
        u32x4 xv[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) xv[i] = load(x[i], b);
        multiply_add<DT, MT>(xv, wv, acc);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[wave][i * 16 + part * 4 + k][r16] = acc[i][k];
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < BM * BN / 8; at += 64 * WAVES) {
        const uint32_t m = at / (BN / 8), c = at % (BN / 8) * 8;
        if (m0 + m >= a.x.n || n0 + c >= a.w.n) continue;
        float v[8] = {}, bias[8], more[8];
        bias8<DT>(a.f, n0 + c, a.w.n, bias);
        if (a.f.residual) residual8<DT>(a.f, m0 + m, n0 + c, a.w.n, more);
#pragma unroll
        for (int k = 0; k < KWAYS; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += sums[c / 16 * KWAYS + k][m][c % 16 + i];
        finish8<DT>(a.f, m0 + m, n0 + c, a.w.n, bias, more, v);
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
// A wavefront has 512 columns of every groups-th row.  Bound by memory: 8192 x 8192 bf16 80 us for 403 MB, 5.0 TB/s, and 4.9 for the bias's sums.  Fewer columns leave
// lanes without work: 65536 x 256 46 us for 101 MB.
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
            slopes(a.activation, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= z[i];
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
    const uint32_t col = block_in_grid() * 64 + lane_id(), from = min(col, cols - 1), wave = wave_in_block();
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

// Which tiles, and how many thread blocks share one.  What a launch takes by this, us: 2.5, and for each round over the compute units a beginning and an
// end and so much for a block of the depth (128 bytes), less of both in a last round of `few` tiles; sums that pass through memory take another launch and their bytes. Measured (bf16
// if not said otherwise, operands used in turn), and the rule's choice behind =:
//   4096 x 256 x 4096 f32       64 x 64 in four sets 67, in two 76, 128 x 128 134 (two parts)            = 64 x 64 in four sets
//   512 x 4096 x 4096           64 x 64 in two sets 30.0, 128 x 128 in two sets 30.9, in two parts of them 31.1 = the last of these
//   1024 x 4096 x 4096          128 x 128 in two sets 37.5, in one 40.5, 128 x 256 49                    = 128 x 128 in two sets
//   2048 x 4096 x 4096          128 x 256 62, 128 x 128 66, 256 x 256 79                                 = 128 x 256
//   8192 x 1024 x 512           128 x 128 17.4, 128 x 256 18.1, 256 x 256 23.2                           = 128 x 128
//   4096 x 4096 x 512 (d_w)     256 x 256 27.4, 128 x 128 30.2, 128 x 256 36                             = 256 x 256
//   64 x 4096 x 4096            64 x 64 in four sets 16.3, two parts of them 15.6, four 15.2             = four
//   3000 x 2000 x 4000 f32      128 x 128 in two parts 372, 64 x 64 in two sets 389, 128 x 128 in one 463 = 128 x 128 in two parts
//   700 x 3000 x 5000           128 x 256 in three parts 45, 128 x 128 in three 48, in two sets 54       = 128 x 128 in two sets (rows that begin inside
//                               lines of 128 bytes, which the model does not know of)
// The gradients go by the same figures, though 32-bit operands across the depth are read from LDS a number at a time:
//   4096 x 4096 x 256 f32 (d_x) 128 x 128 77, 64 x 64 in two sets 100                                    = 128 x 128
//   256 x 4096 x 4096 f32 (d_w) 64 x 64 in four sets 72, in two 86, 128 x 128 139 (two parts)            = 64 x 64 in four sets
//   8192 x 1024 x 1024 f32 (d_x) 128 x 128 130, 64 x 64 in two sets 150                                  = 128 x 128
//   1024 x 1024 x 8192 f32 (d_w) 64 x 64 in four sets 136, 128 x 128 in two sets and four parts 140, in four parts 143 = the second of these
//   128 x 2048 x 4099 f32 (d_w) 64 x 64 in two sets and four parts 32.3, in four sets and four parts 32.9 = the first of these
enum { kThin, k64Four, k64Two, k128, k128Two, k128x256, k256, kHeld };
struct Choice {
    int tile;
    uint32_t parts;
    float time;
    bool copies;                             // of the operands that are not at multiples of 16 bytes
};
struct Cost {
    int tile;
    uint32_t rows, cols, round, most;        // tiles of a round; most tiles that it is for
    float begin, block, block32;             // us; 32-bit operands' (0: not for them)
    uint32_t few;                            // so few tiles have a compute unit (or memory) to themselves, and take
    float few_begin, few_block, few_block32;
};
constexpr Cost kCosts[] = {{k64Four, 64, 64, 256, 256, 3.5f, 0.22f, 0.53f, 0, 0, 0, 0},
                           {k64Two, 64, 64, 512, ~0u, 3.5f, 0.42f, 1.02f, 256, 3.5f, 0.25f, 0.55f},
                           {k128, 128, 128, 512, ~0u, 6.0f, 0.89f, 3.65f, 256, 4.0f, 0.48f, 1.9f},
                           {k128Two, 128, 128, 256, 256, 6.0f, 0.39f, 1.8f, 0, 0, 0, 0},
                           {k128x256, 128, 256, 256, ~0u, 7.5f, 0.78f, 0.0f, 0, 0, 0, 0},
                           {k256, 256, 256, 256, ~0u, 10.5f, 1.34f, 0.0f, 128, 10.5f, 1.03f, 0.0f}};
// Operands that are not at multiples of 16 bytes: through registers, or copied first.  4096 x 4095 x 4095: x w^T 213 through registers, 162 copied, d_z w 351 and
// 146, d_z^T x 597 and 156; 1000 x 1001 x 1003 f32, x w^T 33 and 39; 300 x 1001 x 701 f16 10.4 and 17.
constexpr Cost kHeldCosts[] = {{kHeld, 64, 64, 512, ~0u, 3.5f, 0.8f, 1.3f, 256, 3.5f, 0.8f, 0.85f}};
constexpr float kHeldForms[] = {1.0f, 1.6f, 2.7f}, kHeldForms32[] = {1.0f, 1.1f, 1.15f};     // ... a block takes, by form
constexpr float kCopyBegin = 6.0f, kCopyRate = 3.5e6f;       // us; bytes per us, read and written
template <int N>
Choice cheapest(const Cost (&costs)[N], const mint_dense_op& op, float of_block = 1.0f) {
    const uint64_t blocks = ceil_div(op.depth * size_of(op.dtype), 128);
    Choice best = {costs[0].tile, 1, 0.0f, false};
    float least = 1e30f;
    for (const Cost& c : costs) {
        const float block = (op.dtype == MINT_F32 ? c.block32 : c.block) * of_block, few = (op.dtype == MINT_F32 ? c.few_block32 : c.few_block) * of_block;
        const uint64_t tiles = ceil_div(op.rows, c.rows) * ceil_div(op.cols, c.cols);
        if (block == 0.0f || tiles > c.most) continue;
        const uint64_t most = std::max<uint64_t>(std::min<uint64_t>(2 * c.round / tiles, blocks / 8), 1);
        for (uint64_t parts = 1, each; parts <= most; parts = each > 1 ? ceil_div(blocks, each - 1) : most + 1) {
            each = ceil_div(blocks, parts);                  // (more parts of as many blocks only cost more: on to the next ones of fewer)
            const uint64_t rounds = tiles * parts / c.round, rest = tiles * parts % c.round;
            if (tiles * parts > c.most) break;
            float t = (float)rounds * (c.begin + (float)each * block);
            if (rest) t += rest <= c.few ? c.few_begin + (float)each * few : c.begin + (float)each * block;
            if (parts > 1) t += 2.5f + (float)(op.rows * op.cols) * (float)parts * (8.0f / 4.5e6f);
            if (t < least) {
                least = t;
                best = {c.tile, (uint32_t)parts, t, false};
            }
        }
    }
    return best;
}
// an operand as it lies in memory
struct Operand {
    uint64_t p;
    int64_t stride;                          // bytes
    uint64_t rows, bytes;                    // ... of a row
    uint64_t pieces() const { return ceil_div(bytes, 16); }
    // (a stride is looked at only where there is more than one row; a tile's rows have to be in reach of 32 bits)
    static constexpr int64_t kFar = 1ll << 23;
    bool direct() const { return p % 16 == 0 && (rows <= 1 || (stride % 16 == 0 && stride >= 0 && stride < kFar)); }
    // (a copy is 4 GiB at most: an operand that fills the memory goes through registers)
    bool copied() const { return pieces() * 16 < (uint64_t)kFar && rows * pieces() <= 1ull << 28; }
    uint64_t room() const { return direct() ? 0 : rows * pieces() * 16; }
};
Operand x_of(const mint_dense_op& op) {
    const uint64_t size = size_of(op.dtype), across = op.form == MINT_DENSE_WEIGHT_GRAD;
    return {op.x, op.x_stride * (int64_t)size, across ? op.depth : op.rows, (across ? op.rows : op.depth) * size};
}
Operand w_of(const mint_dense_op& op) {
    const uint64_t size = size_of(op.dtype), across = op.form != MINT_DENSE_PRODUCT;
    return {op.w, op.w_stride * (int64_t)size, across ? op.depth : op.cols, (across ? op.cols : op.depth) * size};
}
// Up to 32 rows go to the kernel for few rows.  us, 1, 16 and 32 rows, weights from memory, and what tiles take:
//   4096 columns of 4096 numbers, bf16   8.8, 11.1, 14.5    tiles 14.0, 15.1, 15.6     (33 rows 20.3, tiles 15.6)
//   the same in f32                      15.1, 18.0, 27.1   tiles 28.7, 29.3, 29.3     (33 rows 39.6, tiles 28.7)
//   8192 of 512, bf16                    4.6, 5.3, 6.2      tiles 7.5, 7.6, 7.8
//   256 of 4096, bf16                    6.7, 9.3, 12.8     tiles 9.8, 10.1, 10.1
//   11000 of 4096, bf16                  19.6, 28.9, 40.8   tiles 24.4, 24.5, 24.7
//   1024 of 16384, bf16                  22, 33, 47         tiles 17.8, 17.1, 17.4
// So from about 16 rows on the rule costs time where there are many columns or much depth: every wavefront reads x again.
Choice choose(const mint_dense_op& op) {
    if (op.form == MINT_DENSE_PRODUCT && op.rows <= 32) return {kThin, 1, 0.0f, false};
    const Operand x = x_of(op), w = w_of(op);
    const Choice best = cheapest(kCosts, op);
    if (op.depth == 0 || (x.direct() && w.direct())) return best;
    const Choice held = cheapest(kHeldCosts, op, (op.dtype == MINT_F32 ? kHeldForms32 : kHeldForms)[op.form]);
    if ((!x.direct() && !x.copied()) || (!w.direct() && !w.copied())) return held;
    if (held.time <= best.time + kCopyBegin + 2.0f * (float)(x.room() + w.room()) / kCopyRate) return held;
    return {best.tile, best.parts, best.time, true};
}
// where in the workspace copies and the parts' sums are
struct Room {
    uint64_t x, w, sums, bytes;
    Room(const mint_dense_op& op, const Choice& c) {
        x = 0;
        w = x + (c.copies ? x_of(op).room() : 0);
        sums = w + (c.copies ? w_of(op).room() : 0);
        bytes = sums + (c.parts > 1 ? (uint64_t)c.parts * op.rows * op.cols * 4 : 0);
    }
};
template <int DT, int BM, int BN, int WM, int NX, int NW, int SPLIT, bool X_ALONG, bool W_ALONG, bool DIRECT>
int go_tiles(DenseArgs a, hipStream_t s) {
    a.row_tiles = (uint32_t)ceil_div(a.x.n, BM);
    a.col_tiles = (uint32_t)ceil_div(a.w.n, BN);
    const uint64_t blocks = ceil_div((uint64_t)a.row_tiles * a.col_tiles * a.parts, 8) * 8;
    if (blocks > 0x7FFFFFFFull / (64 * WM * (BN / 64) * SPLIT)) return MINT_ERR_TOO_LARGE;
    return Launch<&dense_kernel<DT, BM, BN, WM, NX, NW, SPLIT, X_ALONG, W_ALONG, DIRECT>>::go((uint32_t)blocks, 64 * WM * (BN / 64) * SPLIT, 0, s, a);
}
template <int DT, bool XA, bool WA>
int go_form(const DenseArgs& a, int tile, hipStream_t s) {
    constexpr int X2 = XA ? 2 : 4, X3 = XA ? 3 : 5, W2 = WA ? 2 : 4;
    if constexpr (DT != DT_F32) {
        if (tile == k256) return go_tiles<DT, 256, 256, 2, X3, XA == WA && !XA ? 5 : W2, 1, XA, WA, true>(a, s);
        if (tile == k128x256) return go_tiles<DT, 128, 256, 2, XA ? 4 : 8, WA ? 3 : 6, 1, XA, WA, true>(a, s);
    }
    switch (tile) {
        case kHeld: return go_tiles<DT, 64, 64, 4, X2, W2, 2, XA, WA, false>(a, s);
        case k64Four: return go_tiles<DT, 64, 64, 2, X2, W2, 4, XA, WA, true>(a, s);
        case k64Two: return go_tiles<DT, 64, 64, 2, X2, W2, 2, XA, WA, true>(a, s);
        case k128Two: return go_tiles<DT, 128, 128, 2, X2, W2, 2, XA, WA, true>(a, s);
        default: return go_tiles<DT, 128, 128, 4, X3, W2, 1, XA, WA, true>(a, s);
    }
}
template <int DT, int MT, int KWAYS>
int go_thin(DenseArgs a, hipStream_t s) {
    a.col_tiles = (uint32_t)ceil_div(a.w.n, 16 * (kThinWaves / KWAYS));
    const uint64_t blocks = ceil_div(a.x.n, 16 * MT) * a.col_tiles;
    if (blocks > 0x7FFFFFFFull / (64 * kThinWaves)) return MINT_ERR_TOO_LARGE;
    return Launch<&dense_thin_kernel<DT, MT, KWAYS>>::go((uint32_t)blocks, 64 * kThinWaves, 0, s, a);
}
template <int DT>
int go_dense(const mint_dense_op& op, DenseArgs a, const Choice& c, hipStream_t s) {
    if (c.tile == kThin) {
        // Eight wavefronts share the depth of 16 columns, or two each of 64, where there are columns enough.  us, 1, 16 and 32 rows, bf16, eight and two:
        // 4096 columns of 4096 numbers 8.8, 11.1, 14.5 and 22, 31, 45; 16384 of 1024 11.5, 13.1, 16.0 and 8.8, 10.5, 13.9; 14000 of 4096 24, 37, 53
        // and 28, 35, 48; 12304 of 72 3.9, 4.1, 4.2 and 3.2, 3.3, 3.4; but 50000 of 2048 38, 57, 84 and 44, 66, 95.
        const bool few = ceil_div(op.cols, 16) <= 768;
        if (op.rows <= 16) return few ? go_thin<DT, 1, 8>(a, s) : go_thin<DT, 1, 2>(a, s);
        return few ? go_thin<DT, 2, 8>(a, s) : go_thin<DT, 2, 2>(a, s);
    }
    if (c.copies) {
        const auto one = [](const Operand& o, uint8_t* to) {
            const bool any = !o.direct();
            return Copy{reinterpret_cast<const uint8_t*>(o.p), to, o.stride, (uint32_t)o.bytes, (uint32_t)o.pieces(), any ? (uint32_t)(o.rows * o.pieces()) : 0u};
        };
        const Room room(op, c);
        auto* const at = reinterpret_cast<uint8_t*>(op.workspace);
        const Copy x = one(x_of(op), at + room.x), w = one(w_of(op), at + room.w);
        if (x.units) a.x = {x.to, (int64_t)x.pieces * 16, a.x.n};
        if (w.units) a.w = {w.to, (int64_t)w.pieces * 16, a.w.n};
        const uint64_t blocks = ceil_div((uint64_t)x.units + w.units, 256 * kCopies);
        const int err = Launch<&copy_kernel<kSize<DT>>>::go((uint32_t)blocks, 256, 0, s, x, w);
        if (err != MINT_OK) return err;
    }
    int err;
    switch (op.form) {
        case MINT_DENSE_PRODUCT: err = go_form<DT, true, true>(a, c.tile, s); break;
        case MINT_DENSE_INPUT_GRAD: err = go_form<DT, true, false>(a, c.tile, s); break;
        default: err = go_form<DT, false, false>(a, c.tile, s); break;
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
    if (!op || !known(op->dtype) || op->form < MINT_DENSE_PRODUCT || op->form > MINT_DENSE_WEIGHT_GRAD || op->rows == 0 || op->cols == 0 || op->rows > kMost ||
        op->cols > kMost || op->depth > kMost)
        return 0;
    return Room(*op, choose(*op)).bytes;
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
    const Room room(*op, c);
    const size_t need = room.bytes;
    if (need && (!op->workspace || op->workspace_bytes < need)) return MINT_ERR_STAGING;
    if (need && op->workspace % 16) return MINT_ERR_ALIGN;
    const int64_t size = size_of(op->dtype);
    const DenseArgs a = {{reinterpret_cast<const uint8_t*>(op->x), op->x_stride * size, (uint32_t)op->rows},
                         {reinterpret_cast<const uint8_t*>(op->w), op->w_stride * size, (uint32_t)op->cols},
                         {reinterpret_cast<const void*>(op->bias), reinterpret_cast<const void*>(op->residual), reinterpret_cast<void*>(op->out),
                          reinterpret_cast<void*>(op->z), op->residual_stride, op->out_stride, op->z_stride, op->out_dtype, op->activation},
                         (uint32_t)op->depth, 0, 0, c.parts, reinterpret_cast<float*>(op->workspace + room.sums)};
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
    const uint32_t n = op->rows ? groups : 0u;
    const dim3 grid = wide_grid(ceil_div(op->cols, 64));
    switch (op->dtype) {
        case MINT_F16: return Launch<&bias_grad_kernel<DT_F16>>::go(grid, 64 * kBiasWaves, 0, s, sums, d_bias, a.cols, n);
        case MINT_BF16: return Launch<&bias_grad_kernel<DT_BF16>>::go(grid, 64 * kBiasWaves, 0, s, sums, d_bias, a.cols, n);
        default: return Launch<&bias_grad_kernel<DT_F32>>::go(grid, 64 * kBiasWaves, 0, s, sums, d_bias, a.cols, n);
    }
}
