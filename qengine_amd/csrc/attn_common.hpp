// Shared parts of the attention kernels (attn_prompt.hip, attn_tree.hip).
//
// Both hold scores transposed, S^T = K Q^T: the accumulator lane of an MFMA then owns one query column and several keys,
// which is the layout that the second product, O^T = V^T P^T, wants of its B operand (one query column, 8 keys a lane).
// So probabilities go from the first product's registers to the second's without LDS. The keys that a lane holds are not
// consecutive, but the sum over keys does not care in which order it runs as long as V^T's lanes use the same one.
#pragma once
#include "qe_common.hpp"

typedef short s16x4_v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();

constexpr float kLazy = 8.f;  // the running maximum follows a row's scores once they pass it by this much (2^8 in the sums)
constexpr float kFar = 1048576.f;  // maxima beyond which an exponent is not one FMA (below)

// A product that the compiler does not join with a subtraction behind it. The largest score's exponent is score * scale - maximum
// with the maximum that product rounded: an FMA gives the rounding error in its place, up to half a step of the maximum. It is
// the same factor in a row's sums and cancels while weights stay in range: up to a maximum of 2^20 it is below 2^-4. From 2^28
// on fp16 weights, from 2^31 on fp32 ones, left their type.
__device__ __forceinline__ float mul_rounded(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

enum AttnType : int { kAttnBF16 = 0, kAttnF16 = 1 };

template <int DT>
struct AttnT;
template <>
struct AttnT<kAttnBF16> {
    static __device__ __forceinline__ f32x4_v mfma16(u32x4_v a, u32x4_v b, f32x4_v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_v mfma32(u32x4_v a, u32x4_v b, f32x16_v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
    static constexpr uint32_t kExpMask = 0x7f80u, kInf = 0x7f80u, kOne = 0x3f80u;
    static constexpr float kRoom = 40.f;
};
template <>
struct AttnT<kAttnF16> {
    static __device__ __forceinline__ f32x4_v mfma16(u32x4_v a, u32x4_v b, f32x4_v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_v mfma32(u32x4_v a, u32x4_v b, f32x16_v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
    static constexpr uint32_t kExpMask = 0x7c00u, kInf = 0x7c00u, kOne = 0x3c00u;
    static constexpr float kRoom = 0.f;
};

// x of the lane 32 (16) places away, combined: every lane gets op over the pair
__device__ __forceinline__ float max_over_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_over_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_over_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_over_quarters(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return sum_over_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// ---- values that are not finite in keys that some rows of a tile must not see
// A masked key has weight 0, but 0 times an infinity or a NaN in the matrix product is NaN. Kernels whose sums come out not
// finite, or so large that they soon would, therefore run again, first over the finite values alone (pass 1: zeros in the
// others' place), then once for each kind of the others with ones in their place and weight 1 where a row sees a key: where
// such a sum is positive the row sees a +inf (pass 2), a -inf (3) or a NaN (4) in that column.
// Sums of bf16 values can pass fp32 although the result, their mean, does not (weights reach 2^8, and there are many): pass 1
// holds the maximum kRoom higher than the scores, so that weights are 2^-40 of what they were. bf16 probabilities lose nothing
// by it; columns with values below 2^-86 do, beside others above 2^100, and maxima beyond 2^29 have no digits for it. fp16
// values are too small to get there.
constexpr int kKinds = 4;
// NaN where a sum is not finite or past 2^108 (parts that are below it stay finite when they are added), else x
__device__ __forceinline__ float if_bad(float sum, float x) { return __builtin_fmaf(sum * 0x1p20f, 0.f, x); }
// A part's sums join the others times the power of two that its maximum is below theirs. Sums that are not finite must not meet
// a 0 there (a row that is not split gets an infinity of a key under any weight that is not masked), so that of a part with
// keys stays above it.
__device__ __forceinline__ float above_zero(float f) { return fmaxf(f, 0x1p-149f); }
template <int DT>
__device__ __forceinline__ uint32_t keep_half(uint32_t h, int pass) {
    constexpr uint32_t E = AttnT<DT>::kExpMask, I = AttnT<DT>::kInf;
    if (pass == 1) return (h & E) == E ? 0u : h;
    const bool is = pass == 2 ? h == I : pass == 3 ? h == (I | 0x8000u) : (h & 0x7fffu) > I;
    return is ? AttnT<DT>::kOne : 0u;
}
template <int DT>
__device__ __forceinline__ uint32_t keep_two(uint32_t w, int pass) {
    return keep_half<DT>(w & 0xffffu, pass) | keep_half<DT>(w >> 16, pass) << 16;
}
template <int DT>
__device__ __forceinline__ void keep_tile(char* tile, int bytes, int pass, int tid, int threads) {
    for (int i = tid * 4; i < bytes; i += threads * 4) {
        uint32_t* w = reinterpret_cast<uint32_t*>(tile + i);
        *w = keep_two<DT>(*w, pass);
    }
}
// an output (in the type's bits) where the row sees a value of the pass's kind; the order of the passes makes +inf - inf NaN
template <int DT>
__device__ __forceinline__ uint16_t add_kind(uint16_t o, int pass) {
    constexpr uint32_t I = AttnT<DT>::kInf, N = I | 0x40u;
    const bool nan = (o & 0x7fffu) > I;
    if (pass == 2) return nan ? N : I;
    if (pass == 3) return nan || o == I ? N : (I | 0x8000u);
    return N;
}
