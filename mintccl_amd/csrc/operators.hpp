// What the kernels of the expert layer (routing.hip, block8.hip, combine.hip) and of the block around
// it (norms.hpp, dense.hip, balance.hip) share: the element types, and reductions over a wavefront.  No counterpart in the reference.
#pragma once
#include "ring_launch.hpp"

namespace mint {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// ---- element types -------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<DT_F32> {
    using type = float;
    static __device__ __forceinline__ float load(type v) { return v; }
    static __device__ __forceinline__ type round(float v) { return v; }
};
template <> struct Elem<DT_F16> {
    using type = _Float16;
    static __device__ __forceinline__ float load(type v) { return (float)v; }
    static __device__ __forceinline__ type round(float v) { return (_Float16)v; }
};
template <> struct Elem<DT_BF16> {
    using type = __bf16;
    static __device__ __forceinline__ float load(type v) { return (float)v; }
    static __device__ __forceinline__ type round(float v) { return (__bf16)v; }
};

// N consecutive elements as 32-bit numbers, of which the first `left` are there (zeros for the others): one vector, at any
// address, where all are.  (Vectors that are not aligned to their size take the same instructions.)
template <int DT, int N>
__device__ __forceinline__ void load_elements(const typename Elem<DT>::type* p, int64_t left, float (&v)[N]) {
    using T = typename Elem<DT>::type;
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (left >= N) {
        const vec w = *(MINT_GLOBAL const vec*)as_global(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = Elem<DT>::load(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < left ? Elem<DT>::load(*as_global(p + i)) : 0.0f;
    }
}
template <int DT, int N>
__device__ __forceinline__ void store_elements(typename Elem<DT>::type* p, int64_t left, const float (&v)[N]) {
    using T = typename Elem<DT>::type;
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    if (left >= N) {
        vec w;
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = Elem<DT>::round(v[i]);
        *(MINT_GLOBAL vec*)as_global(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) *as_global(p + i) = Elem<DT>::round(v[i]);
    }
}

// ---- reductions over the 64 lanes: the four lanes of a quad, the quads of a row of 16 and
// the four rows are joined by cross-lane operands of the additions themselves; the result is read
// from lane 63.  The order is fixed, so a sum has the same bits every time.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v, uint32_t absent) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)absent, (int)v, CTRL, ROWS, 0xf, false);
}
template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, uint32_t absent, const F& join) {
    v = join(v, dpp<0xB1, 0xf>(v, absent));     // quad_perm [1,0,3,2]
    v = join(v, dpp<0x4E, 0xf>(v, absent));     // quad_perm [2,3,0,1]
    v = join(v, dpp<0x141, 0xf>(v, absent));    // row_half_mirror
    v = join(v, dpp<0x140, 0xf>(v, absent));    // row_mirror
    v = join(v, dpp<0x142, 0xa>(v, absent));    // row_bcast:15 into rows 1 and 3
    v = join(v, dpp<0x143, 0xc>(v, absent));    // row_bcast:31 into rows 2 and 3
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    return wave_fold(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(wave_fold(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
// the largest of numbers of which none is a NaN
__device__ __forceinline__ float wave_max(float v) {
    return __uint_as_float(wave_fold(__float_as_uint(v), 0xFF800000u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}

__device__ __forceinline__ uint32_t sum_below(uint32_t v) {       // of the lanes up to this one
    v += dpp<0x111, 0xf>(v, 0u);        // row_shr:1, 2, 4, 8
    v += dpp<0x112, 0xf>(v, 0u);
    v += dpp<0x114, 0xf>(v, 0u);
    v += dpp<0x118, 0xf>(v, 0u);
    v += dpp<0x142, 0xa>(v, 0u);        // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xc>(v, 0u);        // row_bcast:31 into rows 2 and 3
    return v;
}
// the largest of the 16 lanes of a row
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, dpp<0xB1, 0xf>(v, 0u));
    v = max(v, dpp<0x4E, 0xf>(v, 0u));
    v = max(v, dpp<0x141, 0xf>(v, 0u));
    return max(v, dpp<0x140, 0xf>(v, 0u));
}

inline bool aligned_to(const void* p, uint64_t bytes) { return reinterpret_cast<uint64_t>(p) % bytes == 0; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Thread blocks of up to 1024 threads, more of them than a grid's first dimension takes (fewer than 2^32 threads): those beyond `blocks` have nothing to do.
inline dim3 wide_grid(uint64_t blocks) {
    const uint64_t x = blocks < (1u << 20) ? blocks : 1u << 20;
    return dim3((uint32_t)x, (uint32_t)ceil_div(blocks, x));
}
__device__ __forceinline__ uint32_t block_in_grid() { return blockIdx.y * gridDim.x + blockIdx.x; }

}  // namespace mint
