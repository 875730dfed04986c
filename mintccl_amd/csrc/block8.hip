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
// one's power of two before they are added in 32 bits (all their forms; measured: 1.4e-5 of a sum of 128
// normal numbers' products, 1.5e-5 of the magnitudes' sum at most).  That is far below what a result loses that is rounded to 16 bits, so those results
// take them; a 32-bit result has its 8-bit numbers widened to 16-bit floats, exactly, and takes the 16-bit
// instructions, which keep every bit (9e-9) at half the rate.
#include "operators.hpp"

namespace mint {
namespace {

constexpr float kLargest8 = 448.0f, kLeastBlock = 0x1p-96f;

__device__ __forceinline__ uint32_t pack8(float a, float b, float c, float d) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}
// max |v| of numbers of which one may be a NaN, which then it is
__device__ __forceinline__ float larger(float a, float b) { return a > b || a != a ? a : b; }

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
// The expert of tile `t`.  `rest`: the rows that are no expert's follow as those of an expert with number
// g.experts.  Every wavefront looks for itself, 64 experts at a time.
__device__ __forceinline__ Tile find_tile(const Groups& g, uint32_t t, uint32_t tile_rows, bool rest) {
    Tile r = {0, 0, 0, g.rows, true};
    if (!g.offsets) return r;
    uint32_t base = 0;
    for (uint32_t e0 = 0; e0 < g.experts + rest; e0 += 64) {
        const uint32_t e = e0 + lane_id();
        uint32_t begin = 0, end = 0;
        if (e < g.experts + rest) {
            begin = row_bound(g, e);
            end = e < g.experts ? row_bound(g, e + 1) : g.rows;
            end = max(begin, end);
        }
        const uint32_t tiles = (end - begin + tile_rows - 1) / tile_rows;
        uint32_t sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t other = (uint32_t)__shfl_up((int)sum, d);
            sum += lane_id() >= d ? other : 0u;
        }
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
    r.found = false;
    return r;
}

// ---- rounding to 8 bits ------------------------------------------------------------
struct RowsArgs {
    const void* x;
    uint8_t* q;
    float* scale;
    int64_t x_stride, q_stride, s_row, s_block;
    uint32_t rows, depth, blocks, whole;     // blocks of a row
};
// 16 lanes have a block of 128 numbers of a row.  The last block is filled up with zeros.
template <int DT>
__global__ void __launch_bounds__(256) rows8_kernel(RowsArgs a) {
    using T = typename Elem<DT>::type;
    const uint64_t unit = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const uint32_t row = (uint32_t)(unit / a.blocks), block = (uint32_t)(unit % a.blocks), at = block * 128 + (threadIdx.x & 15u) * 8;
    if (row >= a.rows) return;
    float v[8];
    load_elements<DT, 8>(static_cast<const T*>(a.x) + row * a.x_stride + at, a.whole && at + 8 <= a.depth, (int64_t)a.depth - at, v);
    float m = kLeastBlock;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = larger(fabsf(v[i]), m);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = larger(__shfl_xor(m, d), m);
    const float r = kLargest8 / m;
    const u32x2 w = {pack8(v[0] * r, v[1] * r, v[2] * r, v[3] * r), pack8(v[4] * r, v[5] * r, v[6] * r, v[7] * r)};
    *(MINT_GLOBAL u32x2*)as_global(a.q + row * a.q_stride + at) = w;
    if ((threadIdx.x & 15u) == 0) a.scale[row * a.s_row + block * a.s_block] = m / kLargest8;
}

struct ColumnsArgs {
    const void* x;
    const int32_t* tokens;       // 0, or the row of x that is row i
    uint8_t* q;                  // (width, q_stride): a column of x is a row of it
    float* scale;                // (blocks, width)
    int64_t x_stride, q_stride;
    Groups groups;
    uint32_t x_rows, width, whole;
};
// A thread block has 64 columns of 128 rows of an expert (fewer where it has no more: zeros follow). They turn in LDS.
template <int DT>
__global__ void __launch_bounds__(256) columns8_kernel(ColumnsArgs a) {
    using T = typename Elem<DT>::type;
    __shared__ __attribute__((aligned(16))) uint8_t turned[64][128 + 16];
    __shared__ float most[4][64];
    const uint32_t block = blockIdx.x, c0 = blockIdx.y * 64;
    const Tile t = find_tile(a.groups, block, 128, false);
    if (!t.found) return;
    const uint32_t r0 = t.begin + (block - t.first) * 128;
    const uint32_t vec = threadIdx.x & 7u, first = threadIdx.x >> 3, col = c0 + vec * 8;      // rows first + 32 i
    float v[4][8];
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = kLeastBlock;
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
            load_elements<DT, 8>(static_cast<const T*>(a.x) + row * a.x_stride + col, a.whole && col + 8 <= a.width, (int64_t)a.width - col, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = larger(fabsf(v[i][j]), m[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int d = 8; d < 64; d <<= 1) m[j] = larger(__shfl_xor(m[j], d), m[j]);
        if (lane_id() < 8) most[wave_in_block()][vec * 8 + j] = m[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t c = vec * 8 + j;
        const float all = larger(larger(most[0][c], most[1][c]), larger(most[2][c], most[3][c]));
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
    uint32_t rows, depth, blocks, whole;     // blocks of a row
};
// A thread block has a square of 128 x 128: 16 lanes to a row, eight rows to a thread.
template <int DT>
__global__ void __launch_bounds__(256) squares8_kernel(SquaresArgs a) {
    using T = typename Elem<DT>::type;
    __shared__ float most[4];
    const uint32_t square = blockIdx.x, matrix = blockIdx.y, r0 = square / a.blocks * 128 + threadIdx.x / 16, at = square % a.blocks * 128 + (threadIdx.x & 15u) * 8;
    const T* const w = static_cast<const T*>(a.w) + matrix * a.w_matrix;
    float v[8][8], m = kLeastBlock;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t row = r0 + 16 * i;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row < a.rows)
            load_elements<DT, 8>(w + row * a.w_stride + at, a.whole && at + 8 <= a.depth, (int64_t)a.depth - at, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = larger(fabsf(v[i][j]), m);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = larger(__shfl_xor(m, d), m);
    if (lane_id() == 0) most[wave_in_block()] = m;
    __syncthreads();
    m = larger(larger(most[0], most[1]), larger(most[2], most[3]));
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
    const int32_t* tokens;       // 0, or the row of x that row i of the result is made from
    Groups groups;               // experts' rows (or, `along_depth`, experts' blocks of the depth)
    int64_t x_stride, w_stride, w_matrix, out_stride, out_matrix;
    int64_t sx_row, sx_block, sw_matrix, sw_row, sw_block;
    uint32_t x_rows, rows, cols, depth, col_tiles, row_tiles, out_whole;
};

// Where a row's 16-byte piece lies in its 128 bytes of LDS: turned by the row's number so that the lanes of a
// wavefront that read the same piece of different rows (16 consecutive ones of x, four times four of the weights) fall on different banks.
__device__ __forceinline__ uint32_t turn(uint32_t row) { return ((row >> 1) ^ ((row >> 4) << 1)) & 7u; }

__device__ __forceinline__ void to_lds16(const uint8_t* from, uint32_t lds) {
    __builtin_amdgcn_global_load_lds((MINT_GLOBAL const void*)as_global(from), (MINT_LDS void*)(uintptr_t)lds, 16, 0, 0);
}
__device__ __forceinline__ void to_lds4(const float* from, uint32_t lds) {
    __builtin_amdgcn_global_load_lds((MINT_GLOBAL const void*)as_global(from), (MINT_LDS void*)(uintptr_t)lds, 4, 0, 0);
}
__device__ __forceinline__ u32x4 lds16(uint32_t at) { return *(MINT_LDS const u32x4*)(uintptr_t)at; }
__device__ __forceinline__ float lds_float(uint32_t at) { return *(MINT_LDS const float*)(uintptr_t)at; }
__device__ __forceinline__ i32x8 piece(uint32_t row_at, uint32_t turned, uint32_t part) {
    const u32x4 a = lds16(row_at + ((2 * part) ^ turned) * 16), b = lds16(row_at + ((2 * part + 1) ^ turned) * 16);
    return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f16x8 widened(int a, int b) {
    const f16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), v1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const f16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), v3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return f16x8{v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
}
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

// A thread block has BM rows and BN columns of the result, a wavefront 64 columns and BM / WM rows.
// The depth goes by in blocks of 128: while one is multiplied the next one's bytes are on their way into the other half of LDS.
// The weights are the matrix instruction's first operand, so a lane has four consecutive columns of one row for each,
// and 16 with the four of a wavefront's columns dealt to the instructions in fours.
template <int OUT, int BM, int BN, int WM, bool ROWS_W, bool ALONG>
__global__ void __launch_bounds__(64 * WM * (BN / 64)) product_kernel(ProductArgs a) {
    using Op = Operand<OUT == DT_F32>;
    constexpr int WN = BN / 64, WAVES = WM * WN, MT = BM / WM / 16, NT = 4;
    constexpr uint32_t kX = BM * 128, kW = BN * 128, kSx = BM * 4, kSw = ROWS_W ? BN * 4 : 0, kStage = kX + kW + kSx + kSw;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
    const uint32_t base = (uint32_t)(uintptr_t)(MINT_LDS uint8_t*)lds;
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_in_block());
    const uint32_t row_tile = blockIdx.x / a.col_tiles, n0 = blockIdx.x % a.col_tiles * BN;

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
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) before += (uint32_t)__shfl_xor((int)before, d);
            const uint32_t b = row_bound(a.groups, expert), n = row_bound(a.groups, expert + 1);
            depth0 = __builtin_amdgcn_readfirstlane(before) * 128;
            depth = n > b ? (n - b + 127) / 128 * 128 : 0u;
        }
    } else {
        const Tile t = find_tile(a.groups, row_tile, BM, true);
        if (!t.found) return;
        expert = t.expert;
        m0 = t.begin + (row_tile - t.first) * BM;
        m_end = t.end;
        if (a.groups.offsets && expert == a.groups.experts) depth = 0;
    }
    const uint32_t full = depth / 128, steps = (depth + 127) / 128;

    // A wavefront brings 8 rows of 128 bytes with an instruction: the rows it has of x, then of w.
    constexpr int XI = BM / 8 / WAVES, WI = BN / 8 / WAVES;
    const uint8_t *from_x[XI], *from_w[WI];
    const uint32_t sub = lane >> 3, slot = lane & 7u;
    const auto x_row = [&](uint32_t r) MINT_INLINE_LAMBDA {
        uint32_t row = min(m0 + r, m_end ? m_end - 1 : 0u);
        if (!ALONG && a.tokens) row = (uint32_t)a.tokens[row];
        return min(row, a.x_rows - 1);
    };
    const uint8_t* const w0 = a.w + (ALONG ? 0 : (int64_t)expert * a.w_matrix);
    if (steps) {
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const uint32_t r = (wave * XI + i) * 8 + sub;
            from_x[i] = a.x + (int64_t)x_row(r) * a.x_stride + depth0 + ((slot ^ turn(r)) * 16);
        }
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const uint32_t r = (wave * WI + i) * 8 + sub;
            from_w[i] = w0 + (int64_t)min(n0 + r, a.cols - 1) * a.w_stride + depth0 + ((slot ^ turn(r)) * 16);
        }
    }
    const float *from_sx = nullptr, *from_sw = nullptr;
    if (steps) {
        if (wave < BM / 64) from_sx = a.sx + (int64_t)x_row(wave * 64 + lane) * a.sx_row + (int64_t)(depth0 / 128) * a.sx_block;
        if (ROWS_W && wave < BN / 64)
            from_sw = a.sw + (int64_t)min(n0 + wave * 64 + lane, a.cols - 1) * a.sw_row + (int64_t)(depth0 / 128) * a.sw_block;
    }
    const float* sw_block = a.sw + (ALONG ? 0 : (int64_t)expert * a.sw_matrix);      // one number for 128 columns
    const uint32_t wm = wave / WN, wn = wave % WN;
    if (!ROWS_W) sw_block += (int64_t)((n0 + wn * 64) / 128) * a.sw_row;

    static_assert(BM / 64 <= WAVES && BN / 64 <= WAVES, "a wavefront for each 64 scales");
    const auto bring_scales = [&](uint32_t at) MINT_INLINE_LAMBDA {
        if (wave < BM / 64) {
            to_lds4(from_sx, at + kX + kW + wave * 256);
            from_sx += a.sx_block;
        }
        if (ROWS_W && wave < BN / 64) {
            to_lds4(from_sw, at + kX + kW + kSx + wave * 256);
            from_sw += a.sw_block;
        }
    };
    const auto bring = [&](uint32_t at) MINT_INLINE_LAMBDA {
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            to_lds16(from_x[i], at + (wave * XI + i) * 1024);
            from_x[i] += 128;
        }
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            to_lds16(from_w[i], at + kX + (wave * WI + i) * 1024);
            from_w[i] += 128;
        }
        bring_scales(at);
    };
    // the last block of a depth that is no multiple of 128: nothing is read behind a row's end
    const auto bring_tail = [&](uint32_t at) MINT_INLINE_LAMBDA {
        const auto guarded = [&](const uint8_t* from, uint32_t r, uint32_t to) MINT_INLINE_LAMBDA {
            const int32_t left = (int32_t)(depth - full * 128) - (int32_t)((slot ^ turn(r)) * 16);
            u32x4 v = {0, 0, 0, 0};
            if (left >= 16) {
                v = *(MINT_GLOBAL const u32x4*)as_global(from);
            } else if (left > 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i < left) v[i / 4] |= (uint32_t)*as_global(from + i) << (i % 4 * 8);
            }
            *(MINT_LDS u32x4*)(uintptr_t)(to + lane * 16) = v;
        };
#pragma unroll
        for (int i = 0; i < XI; ++i) guarded(from_x[i], (wave * XI + i) * 8 + sub, at + (wave * XI + i) * 1024);
#pragma unroll
        for (int i = 0; i < WI; ++i) guarded(from_w[i], (wave * WI + i) * 8 + sub, at + kX + (wave * WI + i) * 1024);
        bring_scales(at);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    const uint32_t r16 = lane & 15u, part = lane >> 4;
    const uint32_t xr = wm * (BM / WM) + r16, wr = wn * 64 + (r16 >> 2) * 16 + (r16 & 3u);
    const auto multiply = [&](uint32_t at, float sw) MINT_INLINE_LAMBDA {
        f32x4 sw4[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (ROWS_W) sw4[j] = *(MINT_LDS const f32x4*)(uintptr_t)(at + kX + kW + kSx + (wn * 64 + part * 16 + j * 4) * 4);
        const auto w_piece = [&](int j) MINT_INLINE_LAMBDA { return Op(piece(at + kX + (wr + j * 4) * 128, turn(wr + j * 4), part)); };
        const Op w[NT] = {w_piece(0), w_piece(1), w_piece(2), w_piece(3)};
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t r = xr + i * 16;
            const Op x(piece(at + r * 128, turn(r), part));
            const float s = lds_float(at + kX + kW + r * 4) * sw;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const f32x4 d = Op::multiply(w[j], x);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[i][j][k] = fmaf(d[k], ROWS_W ? s * sw4[j][k] : s, acc[i][j][k]);
            }
        }
    };

    if (steps) {
        if (full) bring(base);
        else bring_tail(base);
        for (uint32_t b = 0; b < steps; ++b) {
            const uint32_t at = base + (b & 1u) * kStage, other = base + ((b + 1) & 1u) * kStage;
            const float sw = ROWS_W ? 1.0f : sw_block[(int64_t)b * a.sw_block];
            __syncthreads();             // (waits for the loads into LDS too)
            if (b + 1 < full) bring(other);
            else if (b + 1 < steps) bring_tail(other);
            multiply(at, sw);
        }
    }

    using T = typename Elem<OUT>::type;
    T* const out = static_cast<T*>(a.out) + (ALONG ? (int64_t)expert * a.out_matrix : 0);
    const uint32_t col = n0 + wn * 64 + part * 16;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const uint32_t row = m0 + xr + i * 16;
        if (row >= m_end || col >= a.cols) continue;
        T* const to = out + (int64_t)row * a.out_stride + col;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = acc[i][h * 2 + k / 4][k % 4];
            if (col + h * 8 < a.cols) store_elements<OUT, 8>(to + h * 8, a.out_whole && col + h * 8 + 8 <= a.cols, (int64_t)a.cols - (col + h * 8), v);
        }
    }
}

template <int OUT, bool ROWS_W, bool ALONG>
int go_product(ProductArgs a, uint32_t matrices, hipStream_t stream) {
    constexpr int BM = 128, BN = 128, WM = 2;
    a.col_tiles = (uint32_t)ceil_div(a.cols, BN);
    a.row_tiles = (uint32_t)ceil_div(a.rows, BM);
    const uint64_t tiles = ALONG ? (uint64_t)a.row_tiles * matrices : a.groups.offsets ? (uint64_t)a.row_tiles + a.groups.experts + 1 : a.row_tiles;
    const uint64_t blocks = tiles * a.col_tiles;
    if (blocks > 0x7FFFFFFFull / (64 * WM * (BN / 64))) return MINT_ERR_TOO_LARGE;
    if (!blocks) return MINT_OK;
    return Launch<&product_kernel<OUT, BM, BN, WM, ROWS_W, ALONG>>::go((uint32_t)blocks, 64 * WM * (BN / 64), 0, stream, a);
}

bool known(int dtype) { return dtype == MINT_F16 || dtype == MINT_BF16 || dtype == MINT_F32; }
// eight elements as one vector
bool vectors(const void* p, int64_t stride, int dtype) { return aligned_to(p, 8 * element_bytes(dtype)) && stride % 8 == 0; }
constexpr uint64_t kMostRows = 0x7FFFFFFF - 128;

}  // namespace
}  // namespace mint

using namespace mint;

extern "C" int mint_rows8(const void* x, int64_t x_stride, uint64_t rows, uint64_t depth, int dtype, void* q, int64_t q_stride,
                          void* scale, int64_t s_row, int64_t s_block, void* stream) {
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
                        (uint32_t)depth, (uint32_t)per_row, vectors(x, x_stride, dtype)};
    const auto s = static_cast<hipStream_t>(stream);
    switch (dtype) {
        case MINT_F16: return Launch<&rows8_kernel<DT_F16>>::go((uint32_t)blocks, 256, 0, s, a);
        case MINT_BF16: return Launch<&rows8_kernel<DT_BF16>>::go((uint32_t)blocks, 256, 0, s, a);
        default: return Launch<&rows8_kernel<DT_F32>>::go((uint32_t)blocks, 256, 0, s, a);
    }
}

extern "C" size_t mint_columns8_blocks(uint64_t rows, uint32_t experts) { return ceil_div(rows, 128) + experts; }

extern "C" int mint_columns8(const void* x, int64_t x_stride, uint64_t x_rows, uint64_t width, int dtype, const void* tokens, uint64_t rows,
                             const void* offsets, uint32_t experts, void* q, int64_t q_stride, void* scale, void* stream) {
    if (!known(dtype) || (!offsets && experts)) return MINT_ERR_ARG;
    if (rows > kMostRows || x_rows > kMostRows || width > 65535ull * 64) return MINT_ERR_TOO_LARGE;
    if (rows == 0 || width == 0) return MINT_OK;
    if (!x || !q || !scale || (!tokens && x_rows < rows)) return MINT_ERR_ARG;
    const uint64_t blocks = mint_columns8_blocks(rows, experts);
    if (!aligned_to(q, 16) || q_stride % 16) return MINT_ERR_ALIGN;
    if (q_stride < (int64_t)(blocks * 128)) return MINT_ERR_GEOMETRY;
    if (blocks > 0x7FFFFFFFull / 256) return MINT_ERR_TOO_LARGE;
    const ColumnsArgs a = {x, static_cast<const int32_t*>(tokens), static_cast<uint8_t*>(q), static_cast<float*>(scale), x_stride, q_stride,
                           {static_cast<const int32_t*>(offsets), experts, (uint32_t)rows}, (uint32_t)x_rows, (uint32_t)width,
                           vectors(x, x_stride, dtype)};
    const auto s = static_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)blocks, (uint32_t)ceil_div(width, 64));
    switch (dtype) {
        case MINT_F16: return Launch<&columns8_kernel<DT_F16>>::go(grid, 256, 0, s, a);
        case MINT_BF16: return Launch<&columns8_kernel<DT_BF16>>::go(grid, 256, 0, s, a);
        default: return Launch<&columns8_kernel<DT_F32>>::go(grid, 256, 0, s, a);
    }
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
                           (uint32_t)depth, (uint32_t)per_row, vectors(w, w_stride, dtype) && w_matrix % 8 == 0};
    const auto s = static_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)blocks, matrices);
    switch (dtype) {
        case MINT_F16: return Launch<&squares8_kernel<DT_F16>>::go(grid, 256, 0, s, a);
        case MINT_BF16: return Launch<&squares8_kernel<DT_BF16>>::go(grid, 256, 0, s, a);
        default: return Launch<&squares8_kernel<DT_F32>>::go(grid, 256, 0, s, a);
    }
}

extern "C" int mint_product8(const mint_product_op* op, void* stream) {
    if (!op || !known(op->dtype) || (op->kind != MINT_PRODUCT_ROWS && op->kind != MINT_PRODUCT_GRADIENT)) return MINT_ERR_ARG;
    if (op->rows > kMostRows || op->cols > kMostRows || op->depth > kMostRows || op->x_rows > kMostRows || op->experts > 65535)
        return MINT_ERR_TOO_LARGE;
    const bool along = op->kind == MINT_PRODUCT_GRADIENT;
    if (op->rows == 0 || op->cols == 0) return MINT_OK;
    if (!op->out || (!op->offsets && op->experts)) return MINT_ERR_ARG;
    // (nothing to multiply: the result is zeros, and neither operand is read)
    const bool some = op->depth != 0;
    if (some && (!op->x || !op->w || !op->sx || !op->sw || op->x_rows == 0)) return MINT_ERR_ARG;
    if (some && !along && !op->tokens && op->x_rows < op->rows) return MINT_ERR_ARG;
    if (some && (!aligned_to(reinterpret_cast<void*>(op->x), 16) || !aligned_to(reinterpret_cast<void*>(op->w), 16) || op->x_stride % 16 ||
                 op->w_stride % 16 || op->w_matrix % 16))
        return MINT_ERR_ALIGN;
    if (along && op->depth % 128) return MINT_ERR_GEOMETRY;
    const bool whole = vectors(reinterpret_cast<void*>(op->out), op->out_stride, op->dtype) && op->out_matrix % 8 == 0;
    const ProductArgs a = {reinterpret_cast<const uint8_t*>(op->x), reinterpret_cast<const uint8_t*>(op->w),
                           reinterpret_cast<const float*>(op->sx), reinterpret_cast<const float*>(op->sw), reinterpret_cast<void*>(op->out),
                           reinterpret_cast<const int32_t*>(op->tokens),
                           {reinterpret_cast<const int32_t*>(op->offsets), op->experts, (uint32_t)(along ? op->group_rows : op->rows)},
                           op->x_stride, op->w_stride, op->w_matrix, op->out_stride, op->out_matrix, op->sx_row, op->sx_block, op->sw_matrix,
                           op->sw_row, op->sw_block, (uint32_t)op->x_rows, (uint32_t)op->rows, (uint32_t)op->cols, (uint32_t)op->depth, 0, 0, whole};
    const auto s = static_cast<hipStream_t>(stream);
    const uint32_t matrices = op->offsets ? op->experts : 1;
    if (along) {
        switch (op->dtype) {
            case MINT_F16: return go_product<DT_F16, true, true>(a, matrices, s);
            case MINT_BF16: return go_product<DT_BF16, true, true>(a, matrices, s);
            default: return go_product<DT_F32, true, true>(a, matrices, s);
        }
    }
    switch (op->dtype) {
        case MINT_F16: return go_product<DT_F16, false, false>(a, matrices, s);
        case MINT_BF16: return go_product<DT_BF16, false, false>(a, matrices, s);
        default: return go_product<DT_F32, false, false>(a, matrices, s);
    }
}
