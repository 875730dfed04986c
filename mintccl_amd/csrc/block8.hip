// Products in 8-bit floating point (four exponent bits) with a 32-bit scale for each block of 128.
//
//   of a block B (128 numbers of a row, of a column, or a square of 128 x 128):
//     m = max(2^-96, max |B|)     scale = m / 448     q = rounded to 8 bits(B * (448 / m))
//   c[i, j] = sum over blocks b of  sx[i, b] sw[j, b] * sum_k qx[i, 128 b + k] qw[j, 128 b + k]
//
// where sw is one number for each 128 rows of a weight matrix, and one for each row where the other side of the
// product was rounded by rows too (the weights' gradient).  A block's sum comes from matrix instructions, and is
// scaled and added in 32 bits.
//
// The 8-bit matrix instructions do not keep all of a sum: of eight products at a time, each is cut off at 2^-13 of the largest
// one's power of two before they are added in 32 bits (all their forms).  The largest has 8 bits and stays whole, so eight
// products lose less than 7 * 2^-13 of it, and a sum less than 8.5e-4 of its magnitudes' sum.  What that is in practice hangs on how
// unlike the products are: 1.5e-5 at most in sums of 128 normal numbers' products, 1e-4 and more where some channels are much larger
// than the others, the bound itself where one of eight is 2^13 times the rest (all relative to the magnitudes' sum).  Half an ulp of bf16
// is 2.0e-3 - 3.9e-3: results in bf16 take these instructions.  Half an ulp of f16 is 2.4e-4 - 4.9e-4, less than the bound: results in
// f16, like those in 32 bits, have their 8-bit numbers widened to 16-bit floats, exactly, and take the 16-bit
// instructions, which keep every bit of a product and add in 32 bits (9e-9 of a sum of 128 normal numbers' products), at half the rate.
#include "operators.hpp"

namespace mint {
namespace {

constexpr float kLargest8 = 448.0f, kLeastBlock = 0x1p-96f;

__device__ __forceinline__ uint32_t pack8(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// Magnitudes are compared as the whole numbers that they are in memory: of a NaN and a number the NaN is larger, and stays.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// 16 lanes' 8 numbers each, a block of 128, in 8 bits; the scale comes back
__device__ __forceinline__ float round_block(const float (&v)[8], u32x2& q) {
    uint32_t most = __float_as_uint(kLeastBlock);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, magnitude(v[i]));
    const float m = __uint_as_float(row_max(most)), r = kLargest8 / m;
    q = u32x2{pack8(v[0] * r, v[1] * r, v[2] * r, v[3] * r), pack8(v[4] * r, v[5] * r, v[6] * r, v[7] * r)};
    return m / kLargest8;
}

// ---- groups of rows --------------------------------------------------------------
// Rows [offsets[e], offsets[e + 1]) are expert e's; tiles of `rows` rows do not reach over experts.
struct Groups {
    const int32_t* offsets;      // 0: one group of all rows
    uint32_t experts, rows;      // rows in all
};
struct Tile {
    uint32_t expert, first, begin, end;     // its expert; the expert's first tile; rows [begin, end) of the expert
    bool found;
};
__device__ __forceinline__ uint32_t row_bound(const Groups& g, uint32_t i) {
    return min((uint32_t)max(g.offsets[i], 0), g.rows);
}
// The tiles of expert e, how many there are in all, and the expert of tile `t`.  `rest`: the rows that are no
// expert's follow as those of an expert with number g.experts, the ones before the first expert's and then those behind the last one's.  Every wavefront looks for itself, 64 experts at a time.
__device__ __forceinline__ uint32_t tiles_of(const Groups& g, uint32_t e, uint32_t tile_rows, bool rest, uint32_t& begin, uint32_t& end) {
    begin = end = 0;
    if (e < g.experts + rest) {
        begin = row_bound(g, e);
        end = max(begin, e < g.experts ? row_bound(g, e + 1) : g.rows);
    }
    return (end - begin + tile_rows - 1) / tile_rows;
}
__device__ __forceinline__ uint32_t count_tiles(const Groups& g, uint32_t tile_rows, bool rest) {
    if (!g.offsets) return (g.rows + tile_rows - 1) / tile_rows;
    uint32_t mine = 0, begin, end;
    for (uint32_t e = lane_id(); e < g.experts + rest; e += 64) mine += tiles_of(g, e, tile_rows, rest, begin, end);
    const uint32_t before = rest ? (row_bound(g, 0) + tile_rows - 1) / tile_rows : 0u;
    return (uint32_t)__builtin_amdgcn_readlane((int)sum_below(mine), 63) + before;
}
__device__ __forceinline__ Tile find_tile(const Groups& g, uint32_t t, uint32_t tile_rows, bool rest) {
    Tile r = {0, 0, 0, g.rows, true};
    if (!g.offsets) return r;
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < g.experts; e0 += 64) {
        uint32_t begin, end;
        const uint32_t tiles = tiles_of(g, e0 + lane_id(), tile_rows, false, begin, end), sum = sum_below(tiles);
        const uint64_t behind = __ballot(base + sum > t);
        if (behind) {
            const int at = __builtin_ctzll(behind);
            r.expert = e0 + at;
            r.first = base + (uint32_t)__builtin_amdgcn_readlane((int)(sum - tiles), at);
            r.begin = (uint32_t)__builtin_amdgcn_readlane((int)begin, at);
            r.end = (uint32_t)__builtin_amdgcn_readlane((int)end, at);
            return r;
        }
        base += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
    r.expert = g.experts;
    r.first = base;
    r.end = row_bound(g, 0);
    const uint32_t before = (r.end + tile_rows - 1) / tile_rows;
    if (t - base >= before) {
        r.first = base + before;
        r.begin = row_bound(g, g.experts);
        r.end = g.rows;
    }
    r.found = rest && t - r.first < (r.end - r.begin + tile_rows - 1) / tile_rows;
    return r;
}

// ---- rounding to 8 bits ------------------------------------------------------------
struct RowsArgs {
    const void* x;
    uint8_t* q;
    float* scale;
    int64_t x_stride, q_stride, s_row, s_block;
    uint32_t rows, depth, blocks;            // blocks of a row
    uint32_t clears;
    uint32_t* clear;                         // so many words that the product behind it counts in, or none
};
// 16 lanes have a block of 128 numbers of a row, 16 bytes each.  The last block is filled up with zeros.
// Bound by memory: 8192 x 8192 numbers of 16 bits 40 us (5.1 TB/s), 8192 x 4096 22 (4.7).
template <int DT>
__global__ void __launch_bounds__(256) rows8_kernel(RowsArgs a) {
    using T = typename Elem<DT>::type;
    const uint64_t unit = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < a.clears; i += gridDim.x * 256) a.clear[i] = 0;
    const uint32_t row = (uint32_t)(unit / a.blocks), block = (uint32_t)(unit % a.blocks), at = block * 128 + (threadIdx.x & 15u) * 8;
    if (row >= a.rows) return;
    float v[8];
    load_elements<DT, 8>(static_cast<const T*>(a.x) + row * a.x_stride + at, (int64_t)a.depth - at, v);
    u32x2 q;
    const float scale = round_block(v, q);
    *(MINT_GLOBAL u32x2*)as_global(a.q + row * a.q_stride + at) = q;
    if ((threadIdx.x & 15u) == 0) a.scale[row * a.s_row + block * a.s_block] = scale;
}

struct ColumnsArgs {
    const void* x;
    const int32_t* tokens;       // 0, or the row of x that is row i
    uint8_t* q;                  // (width, q_stride): a column of x is a row of it
    float* scale;                // (blocks, width)
    int64_t x_stride, q_stride;
    Groups groups;
    uint32_t x_rows, width;
};
// A thread block has 64 columns of 128 rows of an expert (fewer where it has no more: zeros follow), which turn in LDS.
// Bound by memory: 65536 rows of 2048 numbers 87 us (4.6 TB/s), 4096 gathered from 16384 rows 162, both in a launch 269 (with a column's blocks side by side in
// the launch 102 and 184; bank conflicts of the turned stores cost nothing).
// Two matrices can share a launch: the columns of the second one come behind the first one's.
template <int DT>
__global__ void __launch_bounds__(256) columns8_kernel(ColumnsArgs a0, ColumnsArgs a1) {
    using T = typename Elem<DT>::type;
    __shared__ __attribute__((aligned(16))) uint8_t turned[64][128 + 16];
    __shared__ uint32_t most[4][64];
    const uint32_t first_tiles = (a0.width + 63) / 64, tiles = first_tiles + (a1.width + 63) / 64;
    const uint32_t block = blockIdx.x / tiles, tile = blockIdx.x % tiles;      // (rows side by side are read side by side)
    const bool second = tile >= first_tiles;
    const ColumnsArgs& a = second ? a1 : a0;
    const uint32_t c0 = (tile - (second ? first_tiles : 0u)) * 64;
    const Tile t = find_tile(a.groups, block, 128, false);
    if (!t.found) return;
    const uint32_t r0 = t.begin + (block - t.first) * 128;
    const uint32_t vec = threadIdx.x & 7u, first = threadIdx.x >> 3, col = c0 + vec * 8;      // rows first + 32 i
    float v[4][8];
    uint32_t m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = __float_as_uint(kLeastBlock);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t row = r0 + first * 4 + i;
        bool there = row < t.end && col < a.width;
        if (there && a.tokens) {
            row = (uint32_t)a.tokens[row];
            there = row < a.x_rows;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (there)
            load_elements<DT, 8>(static_cast<const T*>(a.x) + row * a.x_stride + col, (int64_t)a.width - col, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = max(m[j], magnitude(v[i][j]));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int d = 8; d < 64; d <<= 1) m[j] = max(m[j], (uint32_t)__shfl_xor((int)m[j], d));
        if (lane_id() < 8) most[wave_in_block()][vec * 8 + j] = m[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t c = vec * 8 + j;
        const float all = __uint_as_float(max(max(most[0][c], most[1][c]), max(most[2][c], most[3][c])));
        const float r = kLargest8 / all;
        *reinterpret_cast<uint32_t*>(&turned[c][first * 4]) = pack8(v[0][j] * r, v[1][j] * r, v[2][j] * r, v[3][j] * r);
        if (first == 0 && c0 + c < a.width) a.scale[(uint64_t)block * a.width + c0 + c] = all / kLargest8;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t at = threadIdx.x + i * 256, c = at >> 3, part = at & 7u;
        if (c0 + c < a.width)
            *(MINT_GLOBAL u32x4*)as_global(a.q + (uint64_t)(c0 + c) * a.q_stride + (uint64_t)block * 128 + part * 16) =
                *reinterpret_cast<const u32x4*>(&turned[c][part * 16]);
    }
}

struct SquaresArgs {
    const void* w;
    uint8_t* q;
    float* scale;
    int64_t w_matrix, w_stride, q_matrix, q_stride;
    uint32_t rows, depth, blocks;            // blocks of a row
};
// A thread block has a square of 128 x 128: 16 lanes to a row, eight rows to a thread, read once and held until the square's largest is known.
// Bound by memory: 8192 x 4096 numbers of 16 bits 18 us (5.6 TB/s), 32 matrices of 2048 x 4096 147 (5.5; of 32 bits 230, 5.8).
template <int DT>
__global__ void __launch_bounds__(256) squares8_kernel(SquaresArgs a) {
    using T = typename Elem<DT>::type;
    __shared__ uint32_t most[4];
    const uint32_t square = blockIdx.x, matrix = blockIdx.y, r0 = square / a.blocks * 128 + threadIdx.x / 16, at = square % a.blocks * 128 + (threadIdx.x & 15u) * 8;
    const T* const w = static_cast<const T*>(a.w) + matrix * a.w_matrix;
    float v[8][8];
    uint32_t largest = __float_as_uint(kLeastBlock);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t row = r0 + 16 * i;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row < a.rows)
            load_elements<DT, 8>(w + row * a.w_stride + at, (int64_t)a.depth - at, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) largest = max(largest, magnitude(v[i][j]));
    }
    largest = wave_max(largest);
    if (lane_id() == 0) most[wave_in_block()] = largest;
    __syncthreads();
    const float m = __uint_as_float(max(max(most[0], most[1]), max(most[2], most[3])));
    const float r = kLargest8 / m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t row = r0 + 16 * i;
        const u32x2 p = {pack8(v[i][0] * r, v[i][1] * r, v[i][2] * r, v[i][3] * r), pack8(v[i][4] * r, v[i][5] * r, v[i][6] * r, v[i][7] * r)};
        if (row < a.rows) *(MINT_GLOBAL u32x2*)as_global(a.q + matrix * a.q_matrix + row * a.q_stride + at) = p;
    }
    if (threadIdx.x == 0) a.scale[(uint64_t)matrix * gridDim.x + square] = m / kLargest8;
}

// ---- the product ---------------------------------------------------------------------
struct ProductArgs {
    const uint8_t *x, *w;
    const float *sx, *sw;
    void* out;
    const int32_t* tokens;       // 0, or the row of x that row i of the result is made from (zeros if x has no such row)
    Groups groups;               // experts' rows (or, `along_depth`, experts' blocks of the depth)
    int64_t x_stride, w_stride, w_matrix, out_stride, out_matrix;
    int64_t sx_row, sx_block, sw_matrix, sw_row, sw_block;
    uint32_t x_rows, rows, cols, depth, col_tiles, row_tiles;
    uint32_t parts;              // JOINED: thread blocks that have a part of a tile's depth, a tile's wavefronts' counts of those that are
    uint32_t* arrived;           // done, and their sums
    uint64_t* sums;
};

// Where a row's 16-byte piece lies in its 128 bytes of LDS: turned by the row's number, so that the lanes that a 16-byte read
// serves together (0 - 3, 12 - 15 and 20 - 27 of 32, then the others), each a row, fall on different banks. For that lane groups 0
// and 1 (2 and 3) read pieces that differ in their lowest bit.
__device__ __forceinline__ uint32_t turn(uint32_t row) { return (row >> 1) & 7u; }
// Which column of the result a row of the weights in LDS stands for: a lane gets four consecutive columns of a row from each of
// four matrix instructions, and those of two lie side by side, so that the four lanes that have a row store 64 bytes together.
__device__ __forceinline__ uint32_t column_of(uint32_t row) {
    return (row & ~63u) | (row & 32u) | (row << 1 & 24u) | (row >> 2 & 4u) | (row & 3u);
}

__device__ __forceinline__ void to_lds16(const uint8_t* from, uint32_t lds) {
    __builtin_amdgcn_global_load_lds((MINT_GLOBAL const void*)as_global(from), (MINT_LDS void*)(uintptr_t)lds, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const float* from, uint32_t lds) {
    __builtin_amdgcn_global_load_lds((MINT_GLOBAL const void*)as_global(from), (MINT_LDS void*)(uintptr_t)lds, 4, 0, 0);
}
// the first `left` bytes, zeros behind
__device__ __forceinline__ u32x4 first_of(u32x4 v, int32_t left) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int32_t bytes = left - 4 * i;
        v[i] &= bytes >= 4 ? 0xFFFFFFFFu : bytes <= 0 ? 0u : (1u << 8 * bytes) - 1u;
    }
    return v;
}
// 16 bytes of a row of which the first `left` are there.  (A piece that begins in the row may be read to its end: it is
// aligned, so it lies in the same page.)
__device__ __forceinline__ u32x4 piece_of(const uint8_t* from, int32_t left) {
    u32x4 v = {0, 0, 0, 0};
    if (left > 0) v = *(MINT_GLOBAL const u32x4*)as_global(from);
    return first_of(v, left);
}
__device__ __forceinline__ u32x4 lds16(uint32_t at) { return *(MINT_LDS const u32x4*)(uintptr_t)at; }
__device__ __forceinline__ float lds_float(uint32_t at) { return *(MINT_LDS const float*)(uintptr_t)at; }
// a lane's part of 16 rows: two of a row's eight pieces (the same two of both operands: the order of the depth does not matter)
__device__ __forceinline__ i32x8 piece(uint32_t at0, uint32_t at1) {
    const u32x4 a = lds16(at0), b = lds16(at1);
    return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f16x8 widened(int a, int b) {
    const f16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), v1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const f16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), v3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return f16x8{v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
}
// Whether results of type OUT are made from widened numbers (above).
template <int OUT>
constexpr bool kWidened = OUT != DT_BF16;
// A 16 x 128 piece of an operand as the matrix instructions take it, and their sum over its depth.
template <bool WIDE>
struct Operand {
    i32x8 v;
    __device__ __forceinline__ explicit Operand(i32x8 bits) : v(bits) {}
    static __device__ __forceinline__ f32x4 multiply(const Operand& a, const Operand& b) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
    }
};
template <>
struct Operand<true> {
    f16x8 v[4];
    __device__ __forceinline__ explicit Operand(i32x8 bits) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = widened(bits[2 * i], bits[2 * i + 1]);
    }
    static __device__ __forceinline__ f32x4 multiply(const Operand& a, const Operand& b) {
        f32x4 d = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], d, 0, 0, 0);
        return d;
    }
};

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

constexpr uint32_t DEALT = 32;

// A thread block has BM rows and BN columns of the result, a wavefront 64 columns and BM / WM rows of them.
// The depth goes by in blocks of 128: while one is multiplied the next STAGES - 1 ones' bytes are on their way into LDS.
// SPLIT sets of wavefronts, each with LDS of its own, take the blocks in turn where there are few tiles: a step takes 0.3 us however
// little there is to multiply.  Their sums are added up in LDS at the end.
// JOINED: the same over `parts` thread blocks, where there are fewer tiles than compute units.  A wavefront leaves its sums in memory and
// counts itself; the last one of those that have the same place adds them all up, in the parts' order.  (No one waits for another.)
// Bound by how steadily the matrix instructions are fed: at 8192 x 8192 x 4096 (253 - 266 us, 2.1 - 2.2 PFLOP/s) they are at work for 56 % of the cycles, no read
// of LDS conflicts, and the rest is what a round of tiles takes to begin and to store (6 - 8 us of 65) and the scaling between them.
// The weights are the matrix instruction's first operand, so a lane has consecutive columns of one row of the result (column_of).
template <int OUT, int BM, int BN, int WM, int STAGES, int SPLIT, bool ROWS_W, bool ALONG, bool JOINED>
__global__ void __launch_bounds__(64 * WM * (BN / 64) * SPLIT) product_kernel(ProductArgs a) {
    using Op = Operand<kWidened<OUT>>;
    using T = typename Elem<OUT>::type;
    constexpr int WN = BN / 64, WAVES = WM * WN, MT = BM / WM / 16, NT = 4;
    constexpr uint32_t kX = BM * 128, kW = BN * 128, kSx = BM * 4, kSw = ROWS_W ? BN * 4 : 256, kStage = kX + kW + kSx + kSw;
    static_assert(BM / 64 <= WAVES && BN / 64 <= WAVES, "a wavefront for each 64 scales");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[SPLIT * STAGES * kStage];
    const uint32_t lane = lane_id(), all_waves = __builtin_amdgcn_readfirstlane(wave_in_block()), wave = all_waves % WAVES, wm = wave / WN, wn = wave % WN;
    const uint32_t way = all_waves / WAVES, base = (uint32_t)(uintptr_t)(MINT_LDS uint8_t*)lds + way * STAGES * kStage;

    // The hardware deals thread blocks to the eight XCDs in turn: each takes an eighth of the tiles that lie together, in
    // columns of GROUP row tiles, so that those at work at a time share rows and weights in its L2.  (Along the depth, where experts
    // with many rows have the long tiles, DEALT tiles at a time: with eighths 16384 tokens of 32 experts took 800 - 1060 us.)
    constexpr uint32_t GROUP = 4;
    const uint32_t row_tiles = ALONG ? a.row_tiles * (a.groups.offsets ? a.groups.experts : 1u) : count_tiles(a.groups, BM, true);
    const uint32_t parts = JOINED ? a.parts : 1u, ways = SPLIT * parts;
    const uint32_t total = row_tiles * a.col_tiles * parts, xcd = blockIdx.x & 7u, nth = blockIdx.x >> 3;
    if (!ALONG && nth >= total / 8 + (xcd < total % 8)) return;
    const uint32_t all_id = ALONG ? (nth / DEALT * 8 + xcd) * DEALT + nth % DEALT : xcd * (total / 8) + min(xcd, total % 8) + nth;
    if (all_id >= total) return;
    const uint32_t id = all_id / parts, part_of_depth = all_id % parts, turn_of_way = part_of_depth * SPLIT + way;
    const uint32_t group = id / (GROUP * a.col_tiles), in_group = id % (GROUP * a.col_tiles), height = min(GROUP, row_tiles - group * GROUP);
    const uint32_t row_tile = group * GROUP + in_group % height, n0 = in_group / height * BN;

    // which rows, which weights, which part of the depth
    uint32_t expert, m0, m_end, depth0 = 0, depth = a.depth;
    if (ALONG) {
        expert = row_tile / a.row_tiles;
        m0 = row_tile % a.row_tiles * BM;
        m_end = a.rows;
        if (a.groups.offsets) {
            uint32_t before = 0;         // blocks of 128 of the experts before this one
            for (uint32_t e = lane; e < expert; e += 64) {
                const uint32_t b = row_bound(a.groups, e), n = row_bound(a.groups, e + 1);
                before += n > b ? (n - b + 127) / 128 : 0u;
            }
            const uint32_t b = row_bound(a.groups, expert), n = row_bound(a.groups, expert + 1);
            depth0 = min((uint32_t)__builtin_amdgcn_readlane((int)sum_below(before), 63) * 128, a.depth);      // (whatever the offsets say)
            depth = min(n > b ? (n - b + 127) / 128 * 128 : 0u, a.depth - depth0);
        }
    } else {
        const Tile t = find_tile(a.groups, row_tile, BM, true);
        expert = t.expert;
        m0 = t.begin + (row_tile - t.first) * BM;
        m_end = t.end;
        if (a.groups.offsets && expert == a.groups.experts) depth = 0;
    }
    // whole blocks of the depth and all of them; of those this way has one of `ways`
    const uint32_t full_all = depth / 128, all_steps = (depth + 127) / 128;
    const uint32_t full = (full_all + ways - 1 - turn_of_way) / ways, steps = (all_steps + ways - 1 - turn_of_way) / ways;

    // A wavefront brings 8 rows of 128 bytes with an instruction: the rows it has of x, then of the weights.
    constexpr int XI = BM / 8 / WAVES, WI = BN / 8 / WAVES;
    const uint8_t *from_x[XI], *from_w[WI];
    const float *from_sx = nullptr, *from_sw = nullptr;
    const uint32_t sub = lane >> 3, slot = lane & 7u;
    const auto x_row = [&](uint32_t r) MINT_INLINE_LAMBDA {
        uint32_t row = min(m0 + r, m_end ? m_end - 1 : 0u);
        if (!ALONG && a.tokens) row = (uint32_t)a.tokens[row];
        return min(row, a.x_rows - 1);
    };
    if (steps) {
        depth0 += turn_of_way * 128;
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const uint32_t r = (wave * XI + i) * 8 + sub;
            from_x[i] = a.x + (int64_t)x_row(r) * a.x_stride + depth0 + ((slot ^ turn(r)) * 16);
        }
        const uint8_t* const w0 = a.w + (ALONG ? 0 : (int64_t)expert * a.w_matrix);
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const uint32_t r = (wave * WI + i) * 8 + sub;
            from_w[i] = w0 + (int64_t)min(n0 + column_of(r), a.cols - 1) * a.w_stride + depth0 + ((slot ^ turn(r)) * 16);
        }
        from_sx = a.sx + (int64_t)x_row(wave % (BM / 64) * 64 + lane) * a.sx_row + (int64_t)(depth0 / 128) * a.sx_block;
        // (of a weight matrix lane i has the scale of the columns of wavefront i)
        const uint32_t col = min(n0 + (ROWS_W ? wave % (BN / 64) * 64 + lane : lane * 64), a.cols - 1);
        from_sw = a.sw + (ROWS_W ? (int64_t)col * a.sw_row + (int64_t)(depth0 / 128) * a.sw_block
                                 : (int64_t)expert * a.sw_matrix + (int64_t)(col / 128) * a.sw_row + (int64_t)turn_of_way * a.sw_block);
    }
    // Where loads are counted (STAGES > 2) all wavefronts have the same number of them under way: some bring scales that others bring too.
    constexpr int LOADS = XI + WI + 2;
    const auto bring_scales = [&](uint32_t at) MINT_INLINE_LAMBDA {
        if (STAGES > 2 || wave < BM / 64) {
            to_lds4(from_sx, at + kX + kW + wave % (BM / 64) * 256);
            from_sx += ways * a.sx_block;
        }
        if (STAGES > 2 || (ROWS_W ? wave < BN / 64 : wave == WAVES - 1)) {
            to_lds4(from_sw, at + kX + kW + kSx + (ROWS_W ? wave % (BN / 64) * 256 : 0));
            from_sw += ways * a.sw_block;
        }
    };
    // piece `n` of XI + WI, the scales with the first
    const auto bring = [&](uint32_t at, int n) MINT_INLINE_LAMBDA {
        if (n == 0) bring_scales(at);
        if (n < XI) {
            to_lds16(from_x[n], at + (wave * XI + n) * 1024);
            from_x[n] += ways * 128;
        } else {
            to_lds16(from_w[n - XI], at + kX + (wave * WI + (n - XI)) * 1024);
            from_w[n - XI] += ways * 128;
        }
    };
    // the last block of a depth that is no multiple of 128 (along the rows there is none)
    // It comes like the others, a piece that lies behind the depth from the block's first one; what is not the row's becomes zeros in LDS.
    const auto left_of = [&](uint32_t r) MINT_INLINE_LAMBDA { return (int32_t)(depth % 128) - (int32_t)((slot ^ turn(r)) * 16); };
    const auto bring_tail = [&](uint32_t at) MINT_INLINE_LAMBDA {
        const auto piece_from = [&](const uint8_t* from, uint32_t r) MINT_INLINE_LAMBDA { return left_of(r) > 0 ? from : from - (slot ^ turn(r)) * 16; };
#pragma unroll
        for (int i = 0; i < XI; ++i) to_lds16(piece_from(from_x[i], (wave * XI + i) * 8 + sub), at + (wave * XI + i) * 1024);
#pragma unroll
        for (int i = 0; i < WI; ++i) to_lds16(piece_from(from_w[i], (wave * WI + i) * 8 + sub), at + kX + (wave * WI + i) * 1024);
        bring_scales(at);
    };
    const auto clear_tail = [&](uint32_t at) MINT_INLINE_LAMBDA {
        const auto clear = [&](uint32_t r, uint32_t to) MINT_INLINE_LAMBDA {
            const auto v = (MINT_LDS u32x4*)(uintptr_t)(to + lane * 16);
            *v = first_of(*v, left_of(r));
        };
        for (int i = 0; i < XI; ++i) clear((wave * XI + i) * 8 + sub, at + (wave * XI + i) * 1024);
        for (int i = 0; i < WI; ++i) clear((wave * WI + i) * 8 + sub, at + kX + (wave * WI + i) * 1024);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    const uint32_t r16 = lane & 15u, part = lane >> 4;
    const uint32_t xr = wm * (BM / WM) + r16, wr = wn * 64 + r16;
    const uint32_t x_at = xr * 128 + ((part ^ turn(xr)) * 16), w_at = kX + wr * 128 + ((part ^ turn(wr)) * 16);
    // Which of a lane's rows of the result (bit i: the i-th) are made from rows that x does not have: those are zeros, whatever was brought in
    // their place.
    uint32_t absent = 0;
    if (!ALONG && a.tokens && all_steps) {
#pragma unroll
        for (int i = 0; i < MT; ++i) absent |= ((uint32_t)a.tokens[min(m0 + xr + i * 16, m_end - 1)] >= a.x_rows ? 1u : 0u) << i;
    }
    const uint32_t sx_at = kX + kW + xr * 4, sw_at = kX + kW + kSx + (ROWS_W ? wn * 64 + part * 8 : wn) * 4;
    // The matrix instructions' sums are scaled and added LAG instructions later: the two units work side by side.
    constexpr int LAG = 3;
    const auto multiply = [&](uint32_t at, const auto& meanwhile) MINT_INLINE_LAMBDA {
        f32x4 sw4[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (ROWS_W) sw4[j] = *(MINT_LDS const f32x4*)(uintptr_t)(at + sw_at + (j / 2 * 32 + j % 2 * 4) * 4);
        const uint32_t w0 = at + w_at, w1 = at + (w_at ^ 64u), x0 = at + x_at, x1 = at + (x_at ^ 64u);
        const Op w[NT] = {Op(piece(w0, w1)), Op(piece(w0 + 2048, w1 + 2048)), Op(piece(w0 + 4096, w1 + 4096)), Op(piece(w0 + 6144, w1 + 6144))};
        Op x(piece(x0, x1));
        static_assert(LAG <= NT, "sums of this row and the one before");
        const float sw = ROWS_W ? 1.0f : lds_float(at + sw_at);
        float s[2], next_s = lds_float(at + sx_at);      // of this row of products, and of those whose sums are still to be added
        __builtin_amdgcn_sched_barrier(0);
        f32x4 d[LAG + 1];
        const auto add = [&](int n) MINT_INLINE_LAMBDA {
            const int i = n / NT, j = n % NT;
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][j][k] = fmaf(d[n % (LAG + 1)][k], ROWS_W ? s[i % 2] * sw4[j][k] : s[i % 2], acc[i][j][k]);
        };
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            // (the next block's loads go out between the products: all at once they would stand in each other's way)
            constexpr int PIECES = MT > 1 ? ((XI + WI) * 2 + MT - 1) / MT : XI + WI;
#pragma unroll
            for (int n = 0; n < PIECES; ++n)
                if (i * PIECES + n < XI + WI) meanwhile(i * PIECES + n);
            Op next = x;
            s[i % 2] = next_s * sw;
            if (i + 1 < MT) {
                next = Op(piece(x0 + (i + 1) * 2048, x1 + (i + 1) * 2048));
                next_s = lds_float(at + sx_at + (i + 1) * 64);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = i * NT + j;
                d[n % (LAG + 1)] = Op::multiply(w[j], x);
                if (n >= LAG) add(n - LAG);
                __builtin_amdgcn_sched_barrier(0);       // (left alone the compiler puts every sum right behind its instruction)
            }
            x = next;
        }
#pragma unroll
        for (int n = MT * NT - LAG; n < MT * NT; ++n) add(n);
    };

    if (all_steps) {
        uint32_t b = 0, at = base, ahead = base + (STAGES - 1) * kStage;
        const auto after = [&](uint32_t stage) MINT_INLINE_LAMBDA { return stage + kStage == base + STAGES * kStage ? base : stage + kStage; };
        const auto bring_all = [&](uint32_t to) MINT_INLINE_LAMBDA {
#pragma unroll
            for (int n = 0; n < XI + WI; ++n) bring(to, n);
        };
#pragma unroll
        for (int st = 0; st < STAGES - 1; ++st) {
            if (st < full) bring_all(base + st * kStage);
            if (!ALONG && st == full && full < steps) bring_tail(base + st * kStage);
        }
        // (as long as every way has a block to bring)
        for (; b + STAGES - 1 < full_all / ways; ++b) {
            meet<(STAGES - 2) * LOADS>();
            multiply(at, [&](int n) MINT_INLINE_LAMBDA { bring(ahead, n); });
            at = after(at);
            ahead = after(ahead);
        }
        for (; b < (all_steps + ways - 1) / ways; ++b) {
            __syncthreads();             // (waits for the loads into LDS too)
            if (SPLIT > 1 && b + STAGES - 1 < full) bring_all(ahead);
            if (!ALONG && b + STAGES - 1 == full && full < steps) bring_tail(ahead);
            if (!ALONG && depth % 128 && b == full_all / ways) {
                if (turn_of_way == full_all % ways) clear_tail(at);
                __syncthreads();
            }
            if (SPLIT == 1 || b < steps) multiply(at, [](int) MINT_INLINE_LAMBDA {});
            at = after(at);
            ahead = after(ahead);
        }
    }
    if constexpr (SPLIT > 1) {           // the ways' sums, added up in their order
        static_assert((SPLIT - 1) * BM * BN * 4 <= SPLIT * STAGES * (int)kStage, "they fit LDS");
        f32x4* const sums = reinterpret_cast<f32x4*>(lds);
        __syncthreads();
        if (way) {
#pragma unroll
            for (int n = 0; n < MT * NT; ++n) sums[(((way - 1) * WAVES + wave) * MT * NT + n) * 64 + lane] = acc[n / NT][n % NT];
        }
        __syncthreads();
        if (way) return;
#pragma unroll
        for (int k = 0; k < SPLIT - 1; ++k)
#pragma unroll
            for (int n = 0; n < MT * NT; ++n) acc[n / NT][n % NT] += sums[((k * WAVES + wave) * MT * NT + n) * 64 + lane];
    }

    if constexpr (JOINED) {
        constexpr uint32_t N = MT * NT * 2;                      // words of 64 bits that a lane has
        const uint64_t place = (uint64_t)id * WAVES + wave;
        uint64_t* const sums = a.sums + place * parts * (N * 64) + lane;
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
            const f32x4 v = acc[n / 2 / NT][n / 2 % NT];
            const uint32_t lo = __float_as_uint(v[n % 2 * 2]), hi = __float_as_uint(v[n % 2 * 2 + 1]);
            st64_agent(sums + (part_of_depth * N + n) * 64, (uint64_t)hi << 32 | lo);
        }
        wait_stores_visible();
        uint32_t before = 0;
        if (lane == 0) before = __hip_atomic_fetch_add(a.arrived + place, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if ((uint32_t)__builtin_amdgcn_readfirstlane((int)before) != parts - 1) return;
        compiler_fence();
#pragma unroll
        for (uint32_t n = 0; n < N / 2; ++n) acc[n / NT][n % NT] = f32x4{0, 0, 0, 0};
        for (uint32_t p0 = 0; p0 < parts; p0 += 4) {
            uint64_t v[4][N];
#pragma unroll
            for (uint32_t p = 0; p < 4; ++p)
#pragma unroll
                for (uint32_t n = 0; n < N; ++n) v[p][n] = ld64_agent(sums + (min(p0 + p, parts - 1) * N + n) * 64);
#pragma unroll
            for (uint32_t p = 0; p < 4; ++p)
                if (p0 + p < parts) {
#pragma unroll
                    for (uint32_t n = 0; n < N; ++n) {
                        f32x4& sum = acc[n / 2 / NT][n / 2 % NT];
                        sum[n % 2 * 2] += __uint_as_float((uint32_t)v[p][n]);
                        sum[n % 2 * 2 + 1] += __uint_as_float((uint32_t)(v[p][n] >> 32));
                    }
                }
        }
    }

    T* const out = static_cast<T*>(a.out) + (ALONG ? (int64_t)expert * a.out_matrix : 0);
    const uint32_t col = n0 + wn * 64 + part * 8;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const uint32_t row = m0 + xr + i * 16;
        if (row >= m_end) continue;
        T* const to = out + (int64_t)row * a.out_stride;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = absent >> i & 1u ? 0.0f : acc[i][h * 2 + k / 4][k % 4];
            const uint32_t c = col + h * 32;
            if (c < a.cols) store_elements<OUT, 8>(to + c, (int64_t)a.cols - c, v);
        }
    }
}

// ---- products of few rows ------------------------------------------------------------
// Bound by reading the weights: 16 MT rows need them once (1 x 4096 x 4096: 5.4 us, most of it the launch and one round trip to
// memory; 8 rows over 64 experts of 1024 x 2048, of which 34 have any: 71 MB in 16.1, 4.4 TB/s).  Those weights come from the last-level cache in part: with
// as many others in between that all of them come from memory, 6.6 us and 19.5 (3.8 TB/s).  A wavefront has 16 columns and every KWAYS-th block of the
// depth, straight from memory into registers: it asks for AHEAD blocks before it multiplies the first, which is what
// keeps enough bytes on their way.  The KWAYS wavefronts' sums of a column are added up in LDS, in their order.
// Activations that are not in 8 bits yet (X) are rounded by the thread block, CHUNK numbers of each row at a time, while the first weights
// travel, and read from LDS: every thread block does that again, but it takes less than another launch.
constexpr int kThinWaves = 8;

// The 32 bytes that a lane has of a block of a row: 16 from `part` * 16 on, and 16 from there + 64 on (the four lanes of
// a row read 64 bytes together).
struct Strip {
    u32x4 v[2];
    // `left` bytes of the row from `from` (the lane's first) on
    __device__ __forceinline__ void load(const uint8_t* from, bool whole, int32_t left) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (whole) v[k] = *(MINT_GLOBAL const u32x4*)as_global(from + k * 64);
            else v[k] = piece_of(from + k * 64, left - k * 64);
        }
    }
    __device__ __forceinline__ i32x8 bits() const {
        return i32x8{(int)v[0].x, (int)v[0].y, (int)v[0].z, (int)v[0].w, (int)v[1].x, (int)v[1].y, (int)v[1].z, (int)v[1].w};
    }
};

// X: the activations' type, DT_BYTES if they are in 8 bits
template <int OUT, int X, int MT, int KWAYS>
__global__ void __launch_bounds__(64 * kThinWaves, 4) thin_kernel(ProductArgs a) {
    using Op = Operand<kWidened<OUT>>;
    using T = typename Elem<OUT>::type;
    constexpr bool ROUND = X != DT_BYTES;
    constexpr int WAVES = kThinWaves, BM = 16 * MT, BN = 16 * (WAVES / KWAYS), AHEAD = 4 / MT;
    constexpr uint32_t CHUNK = 32, XROW = CHUNK * 128 + 16;         // blocks; bytes of a row in LDS
    static_assert(!ROUND || MT == 1, "rounded rows fit LDS");
    __shared__ float sums[WAVES][BM][17];
    __shared__ __attribute__((aligned(16))) uint8_t xs[ROUND ? 16 * XROW : 16];
    __shared__ float xscale[ROUND ? CHUNK : 1][16];
    __shared__ bool gone[16];                                       // ROUND: rows that x does not have
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_in_block()), r16 = lane & 15u, part = lane >> 4;
    const uint32_t way = wave % KWAYS, row_tile = blockIdx.x / a.col_tiles, n0 = blockIdx.x % a.col_tiles * BN, n = n0 + wave / KWAYS * 16;
    const Tile t = find_tile(a.groups, row_tile, BM, true);
    if (!t.found) return;
    const uint32_t m0 = t.begin + (row_tile - t.first) * BM, rows = min(t.end - m0, (uint32_t)BM);
    const uint32_t steps = a.groups.offsets && t.expert == a.groups.experts ? 0u : (a.depth + 127) / 128;

    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    const auto x_row = [&](uint32_t i) MINT_INLINE_LAMBDA {
        const uint32_t row = m0 + min(i, rows - 1);       // (lanes beyond the last row have that one too: what they make is not stored)
        return a.tokens ? (uint32_t)a.tokens[row] : row;
    };
    const uint8_t* const w = a.w + (int64_t)t.expert * a.w_matrix + (int64_t)min(n + r16, a.cols - 1) * a.w_stride + part * 16;
    const float* const sw = a.sw + (int64_t)t.expert * a.sw_matrix + (int64_t)(min(n, a.cols - 1) / 128) * a.sw_row;
    // (a row that x does not have is read as its last one, and makes zeros)
    uint32_t row[MT];
    bool absent[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        row[i] = ROUND || !steps ? 0u : x_row(i * 16 + r16);
        absent[i] = !ROUND && row[i] >= a.x_rows;
        row[i] = min(row[i], a.x_rows - 1);
    }

    // blocks of the depth from `first` on, CHUNK of them at most where they are rounded here
    for (uint32_t first = 0; first < steps; first += CHUNK) {
        const uint32_t end = ROUND ? min(first + CHUNK, steps) : steps;
        for (uint32_t b0 = first + way, round = 0; b0 < end || (ROUND && round == 0); b0 += KWAYS * AHEAD, ++round) {
            Strip wv[AHEAD], xv[AHEAD][MT];
            float s_x[AHEAD][MT], s_w[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                // (in the place of a block behind the last the first is asked for again, and not multiplied)
                const uint32_t b = min(b0 + u * KWAYS < end ? b0 + u * KWAYS : b0, end - 1), at = b * 128 + part * 16;
                const bool whole = b * 128 + 128 <= a.depth;
                const int32_t left = (int32_t)a.depth - (int32_t)at;
                wv[u].load(w + b * 128, whole, left);
                s_w[u] = sw[(int64_t)b * a.sw_block];
                if constexpr (!ROUND) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        xv[u][i].load(a.x + (int64_t)row[i] * a.x_stride + at, whole, left);
                        s_x[u][i] = a.sx[(int64_t)row[i] * a.sx_row + (int64_t)b * a.sx_block];
                    }
                }
            }
            if constexpr (ROUND) {
                if (round == 0) {
                    if (first) __syncthreads();          // (all are done with the chunk before)
                    using TX = typename Elem<X>::type;
                    const uint32_t blocks = end - first;
                    for (uint32_t unit = threadIdx.x / 16; unit < rows * blocks; unit += WAVES * 4) {
                        const uint32_t i = unit / blocks, b = unit % blocks, at = (first + b) * 128 + r16 * 8;
                        const uint32_t from = x_row(i);
                        float v[8];
                        load_elements<X, 8>(reinterpret_cast<const TX*>(a.x) + (int64_t)(a.tokens ? min(from, a.x_rows - 1) : from) * a.x_stride + at, (int64_t)a.depth - at, v);
                        u32x2 q;
                        const float s = round_block(v, q);
                        *reinterpret_cast<u32x2*>(xs + i * XROW + b * 128 + r16 * 8) = q;
                        if (r16 == 0) xscale[b][i] = s;
                        if (a.tokens && r16 == 0 && b == 0) gone[i] = from >= a.x_rows;
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const uint32_t b = min(b0 + u * KWAYS < end ? b0 + u * KWAYS : b0, end - 1) - first;
#pragma unroll
                    for (int k = 0; k < 2; ++k) xv[u][0].v[k] = *reinterpret_cast<const u32x4*>(xs + r16 * XROW + b * 128 + part * 16 + k * 64);
                    s_x[u][0] = xscale[b][r16];
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (b0 + u * KWAYS >= end) break;
                const Op wo(wv[u].bits());
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const f32x4 d = Op::multiply(wo, Op(xv[u][i].bits()));
                    const float s = s_x[u][i] * s_w[u];
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[i][k] = fmaf(d[k], s, acc[i][k]);
                }
            }
        }
        if (!ROUND) break;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const bool zero = ROUND ? a.tokens && steps && gone[r16] : absent[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[wave][i * 16 + r16][part * 4 + k] = zero ? 0.0f : acc[i][k];
    }
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < BM * BN; at += 64 * WAVES) {
        const uint32_t m = at / BN, c = at % BN;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < KWAYS; ++i) sum += sums[c / 16 * KWAYS + i][m][c % 16];
        if (m < rows && n0 + c < a.cols) *as_global(static_cast<T*>(a.out) + (int64_t)(m0 + m) * a.out_stride + n0 + c) = Elem<OUT>::round(sum);
    }
}

// How many tiles of `tile_rows` rows there are at most: an expert's last one, and those of the rows before and behind the experts', may have a
// single row.
uint64_t most_row_tiles(const ProductArgs& a, uint32_t tile_rows) {
    if (!a.groups.offsets) return ceil_div(a.rows, tile_rows);
    return std::min<uint64_t>(a.rows, (a.rows + ((uint64_t)a.groups.experts + 2) * (tile_rows - 1)) / tile_rows);
}
template <int OUT, int BM, int BN, int WM, int STAGES, int SPLIT, bool ROWS_W, bool ALONG, bool JOINED = false>
int go_tiles(ProductArgs a, uint32_t matrices, hipStream_t stream) {
    a.col_tiles = (uint32_t)ceil_div(a.cols, BN);
    a.row_tiles = (uint32_t)ceil_div(a.rows, BM);
    const uint64_t blocks = (ALONG ? (uint64_t)a.row_tiles * matrices : most_row_tiles(a, BM)) * a.col_tiles * (JOINED ? a.parts : 1);
    if (blocks + 8 * DEALT > 0x7FFFFFFFull / (64 * WM * (BN / 64) * SPLIT)) return MINT_ERR_TOO_LARGE;
    if (!blocks) return MINT_OK;
    constexpr uint32_t all = ALONG ? 8 * DEALT : 8;
    return Launch<&product_kernel<OUT, BM, BN, WM, STAGES, SPLIT, ROWS_W, ALONG, JOINED>>::go((uint32_t)(ceil_div(blocks, all) * all), 64 * WM * (BN / 64) * SPLIT, 0,
                                                                                     stream, a);
}
// The tiles whose rounds over the compute units take least: tiles / (those at work at a time), rounded up, times what a round
// takes for a block of the depth.  Measured, us:
//   64 x 64     0.32 up to 256 tiles, the depth dealt to two times four wavefronts, three blocks under way for each (weights used in turn, 64 x 4096
//               x 4096: 11.3; one block under way and dealt to four 11.9, to two 14.0, undealt 18.8; eight in one row 12.9), else 0.5 for 512, dealt to two with
//               one block under way and two thread blocks to a compute unit (512 x 4096 x 4096: 17.3; undealt 20.2, three under way 19.3); up to a depth of 1024
//               undealt (64 x 4096 x 1024: 5.2, dealt 5.3; 512 x 4096 x 512: 4.9, dealt 5.7)
//   128 x 128   0.72 up to 256 tiles, two blocks under way (1024 x 4096 x 4096: 23.0, one 26.5, three 23.2; dealt to two 23.7); 1.29
//               for 512, two thread blocks to a compute unit, which start while others work (11532 rows of 64 experts x 1408 x 2048: 72, 128 x 256 69)
//   128 x 256   1.2, two blocks of the depth under way (2048 x 4096 x 4096: 39, 128 x 128 45)
//   256 x 256   2.0 (8192 x 8192 x 4096: 260, 128 x 256 315; 65536 rows of 32 experts x 2048 x 4096: 573, 128 x 256 656)
template <int OUT, bool ROWS_W, bool ALONG>
int go_product(const ProductArgs& a, uint32_t matrices, hipStream_t stream) {
    const auto tiles = [&](uint32_t bm, uint32_t bn) {
        const uint64_t rows = ALONG ? ceil_div(a.rows, bm) * matrices : ceil_div(a.rows, bm) + (a.groups.offsets ? a.groups.experts / 2 : 0);
        return rows * ceil_div(a.cols, bn);
    };
    const uint64_t n64 = tiles(64, 64), n128 = tiles(128, 128);
    const float t64 = n64 <= 256 ? 0.32f : 0.5f * ceil_div(n64, 512), t128 = n128 <= 256 ? 0.72f : 1.29f * ceil_div(n128, 512),
                wide = 1.2f * ceil_div(tiles(128, 256), 256), large = 2.0f * ceil_div(tiles(256, 256), 256);
    // (operands widened to 16 bits leave no registers for more wavefronts or larger tiles)
    constexpr bool WIDE = kWidened<OUT>;
    const uint64_t blocks = ceil_div(a.depth, 128) / (ALONG && matrices ? matrices : 1);
    if (t64 <= t128 && t64 <= wide && t64 <= large) {
        if constexpr (!ALONG)
            if (a.parts > 1) return go_tiles<OUT, 64, 64, 4, WIDE ? 2 : 4, 2, ROWS_W, ALONG, true>(a, matrices, stream);
        if (blocks <= 8) return go_tiles<OUT, 64, 64, 4, 2, 1, ROWS_W, ALONG>(a, matrices, stream);
        if (!WIDE && n64 <= 256) return go_tiles<OUT, 64, 64, 4, WIDE ? 2 : 4, 2, ROWS_W, ALONG>(a, matrices, stream);
        return go_tiles<OUT, 64, 64, 4, 2, 2, ROWS_W, ALONG>(a, matrices, stream);
    }
    if constexpr (WIDE) {
        return go_tiles<OUT, 128, 256, 2, 3, 1, ROWS_W, ALONG>(a, matrices, stream);
    } else {
        if (t128 <= wide && t128 <= large) {
            if (n128 <= 256) return go_tiles<OUT, 128, 128, 4, 3, 1, ROWS_W, ALONG>(a, matrices, stream);
            return go_tiles<OUT, 128, 128, 4, 2, 1, ROWS_W, ALONG>(a, matrices, stream);
        }
        if (wide <= large) return go_tiles<OUT, 128, 256, 2, 3, 1, ROWS_W, ALONG>(a, matrices, stream);
        return go_tiles<OUT, 256, 256, 2, 2, 1, ROWS_W, ALONG>(a, matrices, stream);
    }
}

// Where a product of one matrix has tiles of 64 x 64 for at most half of the compute units and a long depth: thread blocks to a tile. Rounded
// before, us, with one and with these (and with widened operands): 64 x 4096 x 4096 14.1 and 12.4 (18.1 and 13.1), 40 x 2048 x 8192 19.0 and 13.7,
// 100 x 1000 x 8000 19.4 and 13.6, 128 x 4096 x 4096 14.4 and 13.2, 50 x 5000 x 2500 11.5 and 11.6 (14.1 and 12.2), 48 x 7168 x 2048 10.0 and 11.2.
uint32_t parts_of(uint64_t rows, uint64_t cols, uint64_t depth, int dtype) {
    const uint64_t tiles = ceil_div(rows, 64) * ceil_div(cols, 64), blocks = ceil_div(depth, 128);
    if (tiles == 0 || tiles > 128 || blocks < (dtype == MINT_BF16 ? 32 : 20)) return 1;
    return (uint32_t)std::min<uint64_t>(256 / tiles, blocks / 6);
}
// Few rows: at most 32 for each weight matrix, on the average (24 x 4096 x 4096: 7.8 us, with tiles of 64 x 64 9.4; at 64 rows
// 12.8 and 9.5).
bool few_rows(uint64_t rows, uint32_t matrices) { return rows <= 32ull * matrices; }
// ... and so few that the rounding is done on the way: 256 blocks of 128 for each weight matrix (all thread blocks
// do that work again, 0.5 us for 32 blocks, and save a launch: with a depth and 4096 columns of 4096, 1 row 5.7 us for 10.3, 8 rows 9.2
// for 10.6, 12 rows 11.6 for 10.5)
bool rounded_on_the_way(uint64_t rows, uint64_t depth, uint32_t matrices) {
    return rows <= 16ull * matrices && rows * ceil_div(depth, 128) <= 256ull * matrices;
}
template <int OUT, int X, int MT, int KWAYS>
int go_thin_ways(ProductArgs a, hipStream_t stream) {
    a.col_tiles = (uint32_t)ceil_div(a.cols, 16 * (kThinWaves / KWAYS));
    const uint64_t blocks = most_row_tiles(a, 16 * MT) * a.col_tiles;
    if (blocks > 0x7FFFFFFFull / (64 * kThinWaves)) return MINT_ERR_TOO_LARGE;
    return Launch<&thin_kernel<OUT, X, MT, KWAYS>>::go((uint32_t)blocks, 64 * kThinWaves, 0, stream, a);
}
// The depth is dealt to eight wavefronts where 16 columns to a thread block leave few of those, else to two.
template <int OUT, int X, int MT>
int go_thin(const ProductArgs& a, hipStream_t stream) {
    const uint64_t blocks = (ceil_div(a.rows, 16 * MT) + (a.groups.offsets ? a.groups.experts / 2 : 0)) * ceil_div(a.cols, 16);
    if (blocks <= 768) return go_thin_ways<OUT, X, MT, 8>(a, stream);
    return go_thin_ways<OUT, X, MT, 2>(a, stream);
}
template <int OUT>
int go_rows(const ProductArgs& a, int x_dtype, uint32_t matrices, hipStream_t stream) {
    switch (x_dtype) {
        case MINT_F16: return go_thin<OUT, DT_F16, 1>(a, stream);
        case MINT_BF16: return go_thin<OUT, DT_BF16, 1>(a, stream);
        case MINT_F32: return go_thin<OUT, DT_F32, 1>(a, stream);
        default: break;
    }
    if (a.rows <= 16ull * matrices) return go_thin<OUT, DT_BYTES, 1>(a, stream);
    if (few_rows(a.rows, matrices)) return go_thin<OUT, DT_BYTES, 2>(a, stream);
    return go_product<OUT, false, false>(a, 1, stream);
}

bool known(int dtype) { return dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32; }
constexpr uint64_t kMostRows = 0x7FFFFFFF - 128;

}  // namespace
}  // namespace mint

using namespace mint;

namespace {
int go_rows8(const void* x, int64_t x_stride, uint64_t rows, uint64_t depth, int dtype, void* q, int64_t q_stride, void* scale, int64_t s_row,
             int64_t s_block, uint32_t* clear, uint32_t clears, void* stream) {
    if (!known(dtype)) return MINT_ERR_ARG;
    if (rows > kMostRows || depth > kMostRows) return MINT_ERR_TOO_LARGE;
    if (rows == 0 || depth == 0) return MINT_OK;
    if (!x || !q || !scale) return MINT_ERR_ARG;
    const uint64_t per_row = ceil_div(depth, 128);
    if (!aligned_to(q, 16) || q_stride % 16) return MINT_ERR_ALIGN;
    if (q_stride < (int64_t)(per_row * 128)) return MINT_ERR_GEOMETRY;
    const uint64_t blocks = ceil_div(rows * per_row, 16);
    if (blocks > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    const RowsArgs a = {x, static_cast<uint8_t*>(q), static_cast<float*>(scale), x_stride, q_stride, s_row, s_block, (uint32_t)rows,
                        (uint32_t)depth, (uint32_t)per_row, clears, clear};
    const auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case MINT_F16: return Launch<&rows8_kernel<DT_F16>>::go((uint32_t)blocks, 256, 0, s, a);
        case MINT_BF16: return Launch<&rows8_kernel<DT_BF16>>::go((uint32_t)blocks, 256, 0, s, a);
        default: return Launch<&rows8_kernel<DT_F32>>::go((uint32_t)blocks, 256, 0, s, a);
    }
}
}  // namespace

extern "C" int mint_rows8(const void* x, int64_t x_stride, uint64_t rows, uint64_t depth, int dtype, void* q, int64_t q_stride,
                          void* scale, int64_t s_row, int64_t s_block, void* stream) {
    return go_rows8(x, x_stride, rows, depth, dtype, q, q_stride, scale, s_row, s_block, nullptr, 0, stream);
}

extern "C" size_t mint_columns8_blocks(uint64_t rows, uint32_t experts) { return ceil_div(rows, 128) + experts; }

namespace {
int go_columns(const ColumnsArgs& a, const ColumnsArgs& b, int dtype, uint32_t blocks, hipStream_t s) {
    const uint64_t all = (uint64_t)blocks * (ceil_div(a.width, 64) + ceil_div(b.width, 64));
    if (all > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    const uint32_t grid = (uint32_t)all;
    switch (dtype) {
        case MINT_F16: return Launch<&columns8_kernel<DT_F16>>::go(grid, 256, 0, s, a, b);
        case MINT_BF16: return Launch<&columns8_kernel<DT_BF16>>::go(grid, 256, 0, s, a, b);
        default: return Launch<&columns8_kernel<DT_F32>>::go(grid, 256, 0, s, a, b);
    }
}
}  // namespace

extern "C" int mint_columns8(const void* x, int64_t x_stride, uint64_t x_rows, uint64_t width, int dtype, const void* tokens, uint64_t rows,
                             const void* offsets, uint32_t experts, void* q, int64_t q_stride, void* scale, void* stream) {
    if (!known(dtype) || (!offsets && experts)) return MINT_ERR_ARG;
    if (rows > kMostRows || x_rows > kMostRows || width > kMostRows) return MINT_ERR_TOO_LARGE;
    if (rows == 0 || width == 0) return MINT_OK;
    if (!x || !q || !scale || (!tokens && x_rows < rows) || x_rows == 0) return MINT_ERR_ARG;
    const uint64_t blocks = mint_columns8_blocks(rows, experts);
    if (!aligned_to(q, 16) || q_stride % 16) return MINT_ERR_ALIGN;
    if (q_stride < (int64_t)(blocks * 128)) return MINT_ERR_GEOMETRY;
    if (blocks > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    const ColumnsArgs a = {x, static_cast<const int32_t*>(tokens), static_cast<uint8_t*>(q), static_cast<float*>(scale), x_stride, q_stride,
                           {static_cast<const int32_t*>(offsets), experts, (uint32_t)rows}, (uint32_t)x_rows, (uint32_t)width};
    return go_columns(a, ColumnsArgs{}, dtype, (uint32_t)blocks, static_cast<hipStream_t>(stream));
}

namespace {
// 8-bit numbers and scales of both sides, one behind the other: (cols, blocks * 128), (depth, blocks * 128), scales
struct GradientRoom {
    uint64_t blocks, x, scales, x_scales, bytes;
    explicit GradientRoom(const mint_weight_grad_op& op) {
        blocks = mint_columns8_blocks(op.rows, op.experts);
        x = op.cols * blocks * 128;
        scales = x + op.depth * blocks * 128;
        x_scales = scales + blocks * op.cols * 4;
        bytes = x_scales + blocks * op.depth * 4;
    }
};
}  // namespace

extern "C" size_t mint_weight_grad8_workspace(const mint_weight_grad_op* op) { return op && op->rows ? GradientRoom(*op).bytes : 0; }

extern "C" int mint_weight_grad8(const mint_weight_grad_op* op, void* stream) {
    if (!op || !known(op->dtype) || !known(op->d_dtype) || !known(op->x_dtype) || (!op->offsets && op->experts)) return MINT_ERR_ARG;
    if (op->rows > kMostRows || op->x_rows > kMostRows || op->cols > kMostRows || op->depth > kMostRows || op->experts > 65535)
        return MINT_ERR_TOO_LARGE;
    if (op->cols == 0 || op->depth == 0) return MINT_OK;
    if (!op->out || (op->rows && (!op->d || !op->x || op->x_rows == 0 || (!op->tokens && op->x_rows < op->rows)))) return MINT_ERR_ARG;
    const GradientRoom room(*op);
    if (room.blocks > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    auto* const q = reinterpret_cast<uint8_t*>(op->workspace);
    const int64_t wide = (int64_t)room.blocks * 128;
    if (op->rows) {
        if (!q || op->workspace_bytes < room.bytes) return MINT_ERR_STAGING;
        if (!aligned_to(q, 16)) return MINT_ERR_ALIGN;
        const Groups groups = {reinterpret_cast<const int32_t*>(op->offsets), op->experts, (uint32_t)op->rows};
        const ColumnsArgs d = {reinterpret_cast<const void*>(op->d), nullptr, q, reinterpret_cast<float*>(q + room.scales), op->d_stride, wide, groups,
                               (uint32_t)op->rows, (uint32_t)op->cols};
        const ColumnsArgs x = {reinterpret_cast<const void*>(op->x), reinterpret_cast<const int32_t*>(op->tokens), q + room.x,
                               reinterpret_cast<float*>(q + room.x_scales), op->x_stride, wide, groups, (uint32_t)op->x_rows, (uint32_t)op->depth};
        const auto s = static_cast<hipStream_t>(stream);
        int err;
        if (op->d_dtype == op->x_dtype) {
            err = go_columns(d, x, op->d_dtype, (uint32_t)room.blocks, s);
        } else {
            err = go_columns(d, ColumnsArgs{}, op->d_dtype, (uint32_t)room.blocks, s);
            if (err == MINT_OK) err = go_columns(x, ColumnsArgs{}, op->x_dtype, (uint32_t)room.blocks, s);
        }
        if (err != MINT_OK) return err;
    }
    mint_product_op p = {};
    p.kind = MINT_PRODUCT_GRADIENT;
    p.dtype = op->dtype;
    p.x_dtype = MINT_BYTES;
    p.x = reinterpret_cast<uint64_t>(q);
    p.w = reinterpret_cast<uint64_t>(q + room.x);
    p.sx = reinterpret_cast<uint64_t>(q + room.scales);
    p.sw = reinterpret_cast<uint64_t>(q + room.x_scales);
    p.out = op->out;
    p.offsets = op->offsets;
    p.rows = p.x_rows = op->cols;
    p.cols = op->depth;
    p.depth = op->rows ? (uint64_t)wide : 0;
    p.group_rows = op->rows;
    p.x_stride = p.w_stride = wide;
    p.out_stride = op->out_stride;
    p.out_matrix = op->out_matrix;
    p.sx_row = p.sw_row = 1;
    p.sx_block = (int64_t)op->cols;
    p.sw_block = (int64_t)op->depth;
    p.experts = op->experts;
    return mint_product8(&p, stream);
}

extern "C" int mint_squares8(const void* w, int64_t w_matrix, int64_t w_stride, uint32_t matrices, uint64_t rows, uint64_t depth, int dtype,
                             void* q, int64_t q_matrix, int64_t q_stride, void* scale, void* stream) {
    if (!known(dtype)) return MINT_ERR_ARG;
    if (rows > kMostRows || depth > kMostRows || matrices > 65535) return MINT_ERR_TOO_LARGE;
    if (rows == 0 || depth == 0 || matrices == 0) return MINT_OK;
    if (!w || !q || !scale) return MINT_ERR_ARG;
    const uint64_t per_row = ceil_div(depth, 128), blocks = per_row * ceil_div(rows, 128);
    if (!aligned_to(q, 16) || q_stride % 16 || q_matrix % 16) return MINT_ERR_ALIGN;
    if (q_stride < (int64_t)(per_row * 128)) return MINT_ERR_GEOMETRY;
    if (blocks > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    const SquaresArgs a = {w, static_cast<uint8_t*>(q), static_cast<float*>(scale), w_matrix, w_stride, q_matrix, q_stride, (uint32_t)rows,
                           (uint32_t)depth, (uint32_t)per_row};
    const auto s = static_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)blocks, matrices);
    switch (dtype) {
        case MINT_F16: return Launch<&squares8_kernel<DT_F16>>::go(grid, 256, 0, s, a);
        case MINT_BF16: return Launch<&squares8_kernel<DT_BF16>>::go(grid, 256, 0, s, a);
        default: return Launch<&squares8_kernel<DT_F32>>::go(grid, 256, 0, s, a);
    }
}

namespace {
uint32_t matrices_of(const mint_product_op& op) { return op.offsets ? op.experts : 1; }
// What a product needs: 8-bit numbers and scales of activations that come as they are, where rounding them takes a launch of its
// own, and behind them the sums of a tile's parts and their counts (which that launch clears, or one that does nothing else: a product
// has the same bits whoever rounded its rows)
struct ProductRoom {
    uint64_t rounded = 0, sums_at = 0, sums = 0, clears = 0, bytes = 0;
    uint32_t parts = 1;
    explicit ProductRoom(const mint_product_op& op) {
        if (op.kind != MINT_PRODUCT_ROWS) return;
        if (op.x_dtype != MINT_BYTES && !rounded_on_the_way(op.rows, op.depth, matrices_of(op)))
            bytes = rounded = op.x_rows * ceil_div(op.depth, 128) * 132;
        if (op.offsets || few_rows(op.rows, 1)) return;
        parts = parts_of(op.rows, op.cols, op.depth, op.dtype);
        if (parts == 1) return;
        const uint64_t tiles = ceil_div(op.rows, 64) * ceil_div(op.cols, 64);
        sums_at = ceil_div(rounded, 16) * 16;
        sums = tiles * parts * (64 * 64 * 4);
        clears = tiles * 4;
        bytes = sums_at + sums + clears * 4;
    }
};
}  // namespace

extern "C" size_t mint_product8_workspace(const mint_product_op* op) { return op ? ProductRoom(*op).bytes : 0; }

extern "C" int mint_product8(const mint_product_op* op, void* stream) {
    if (!op || !known(op->dtype) || (op->kind != MINT_PRODUCT_ROWS && op->kind != MINT_PRODUCT_GRADIENT)) return MINT_ERR_ARG;
    const bool along = op->kind == MINT_PRODUCT_GRADIENT, raw = op->x_dtype != MINT_BYTES;
    if (raw && (along || !known(op->x_dtype))) return MINT_ERR_ARG;
    if (op->rows > kMostRows || op->cols > kMostRows || op->depth > kMostRows || op->x_rows > kMostRows || op->experts > 65535)
        return MINT_ERR_TOO_LARGE;
    if (op->rows == 0 || op->cols == 0) return MINT_OK;
    if (!op->out || (!op->offsets && op->experts)) return MINT_ERR_ARG;
    // (nothing to multiply: the result is zeros, and neither operand is read)
    const bool some = op->depth != 0;
    if (some && (!op->x || !op->w || (!raw && !op->sx) || !op->sw || op->x_rows == 0)) return MINT_ERR_ARG;
    if (some && (along || !op->tokens) && op->x_rows < op->rows) return MINT_ERR_ARG;
    if (some && ((!raw && (!aligned_to(reinterpret_cast<void*>(op->x), 16) || op->x_stride % 16)) || !aligned_to(reinterpret_cast<void*>(op->w), 16) ||
                 op->w_stride % 16 || op->w_matrix % 16))
        return MINT_ERR_ALIGN;
    if (along && op->depth % 128) return MINT_ERR_GEOMETRY;
    const ProductRoom room(*op);
    const size_t need = room.bytes;
    if (need && (op->workspace_bytes < need || !op->workspace)) return MINT_ERR_STAGING;
    if (need && !aligned_to(reinterpret_cast<void*>(op->workspace), 16)) return MINT_ERR_ALIGN;
    const auto s = static_cast<hipStream_t>(stream);
    ProductArgs a = {reinterpret_cast<const uint8_t*>(op->x), reinterpret_cast<const uint8_t*>(op->w),
                     reinterpret_cast<const float*>(op->sx), reinterpret_cast<const float*>(op->sw), reinterpret_cast<void*>(op->out),
                     reinterpret_cast<const int32_t*>(op->tokens),
                     {reinterpret_cast<const int32_t*>(op->offsets), op->experts, (uint32_t)(along ? op->group_rows : op->rows)},
                     op->x_stride, op->w_stride, op->w_matrix, op->out_stride, op->out_matrix, op->sx_row, op->sx_block, op->sw_matrix,
                     op->sw_row, op->sw_block, (uint32_t)op->x_rows, (uint32_t)op->rows, (uint32_t)op->cols, (uint32_t)op->depth, 0, 0, 1, nullptr, nullptr};
    const uint32_t matrices = matrices_of(*op);
    int x_dtype = op->x_dtype;
    if (need && some) {
        a.parts = room.parts;
        a.sums = reinterpret_cast<uint64_t*>(op->workspace + room.sums_at);
        a.arrived = reinterpret_cast<uint32_t*>(op->workspace + room.sums_at + room.sums);
    }
    if (room.clears && !room.rounded && some) {
        const RowsArgs none = {nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, 0, 1, (uint32_t)room.clears, a.arrived};
        const int err = Launch<&rows8_kernel<DT_F32>>::go((uint32_t)ceil_div(room.clears, 256), 256, 0, s, none);
        if (err != MINT_OK) return err;
    }
    if (room.rounded && some) {
        const uint64_t per_row = ceil_div(op->depth, 128);
        auto* const q = reinterpret_cast<uint8_t*>(op->workspace);
        auto* const scale = reinterpret_cast<float*>(q + op->x_rows * per_row * 128);
        const int err = go_rows8(a.x, op->x_stride, op->x_rows, op->depth, x_dtype, q, (int64_t)per_row * 128, scale, 1, (int64_t)op->x_rows, a.arrived,
                                 (uint32_t)room.clears, stream);
        if (err != MINT_OK) return err;
        a.x = q;
        a.x_stride = (int64_t)per_row * 128;
        a.sx = scale;
        a.sx_row = 1;
        a.sx_block = (int64_t)op->x_rows;
    }
    if (room.rounded) x_dtype = MINT_BYTES;
    if (along) {
        switch (op->dtype) {
            case MINT_F16: return go_product<DT_F16, true, true>(a, matrices, s);
            case MINT_BF16: return go_product<DT_BF16, true, true>(a, matrices, s);
            default: return go_product<DT_F32, true, true>(a, matrices, s);
        }
    }
    switch (op->dtype) {
        case MINT_F16: return go_rows<DT_F16>(a, x_dtype, matrices, s);
        case MINT_BF16: return go_rows<DT_BF16>(a, x_dtype, matrices, s);
        default: return go_rows<DT_F32>(a, x_dtype, matrices, s);
    }
}
