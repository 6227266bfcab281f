// Shared parts of the attention kernels (attn_prompt.hip, attn_tree.hip).
//
// Both hold scores transposed, S^T = K Q^T: the accumulator lane of an MFMA then owns one query column and several keys,
// which is the layout that the second product, O^T = V^T P^T, wants of its B operand (one query column, 8 keys a lane).
// So probabilities go from the first product's registers to the second's without LDS. The keys that a lane holds are not
// consecutive, but the sum over keys does not care in which order it runs as long as V^T's lanes use the same one.
#pragma once
#include "qe_common.hpp"

typedef short s16x4_v __attribute__((ext_vector_type(4)));
typedef short s16x8_v __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();

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
// A masked key has weight 0, but 0 times an infinity or a NaN in the matrix product is NaN. Tiles with a mask therefore
// look for such values (a vote; there are none in ordinary data), put zeros in their place, and add to each row what the
// keys that it does see contribute: products of indicators on the matrix cores, which say whether a row sees a +inf, a
// -inf or a NaN in a column.
template <int DT>
__device__ __forceinline__ bool half_not_finite(uint32_t two) {  // either 16-bit value of the pair
    constexpr uint32_t E = AttnT<DT>::kExpMask;
    return (two & E) == E || ((two >> 16) & E) == E;
}
template <int DT>
__device__ __forceinline__ bool any_not_finite(u32x4_v v) {
    return half_not_finite<DT>(v[0]) || half_not_finite<DT>(v[1]) || half_not_finite<DT>(v[2]) || half_not_finite<DT>(v[3]);
}
enum class Keep { kFinite, kPosInf, kNegInf, kNan };
// the finite values with zeros elsewhere, or ones (in the type's own bits) where a value is of the asked kind
template <int DT, Keep K>
__device__ __forceinline__ uint32_t keep_half(uint32_t h) {
    constexpr uint32_t E = AttnT<DT>::kExpMask;
    if constexpr (K == Keep::kFinite) return (h & E) == E ? 0u : h;
    bool is = false;
    if constexpr (K == Keep::kPosInf) is = h == AttnT<DT>::kInf;
    if constexpr (K == Keep::kNegInf) is = h == (AttnT<DT>::kInf | 0x8000u);
    if constexpr (K == Keep::kNan) is = (h & 0x7fffu) > AttnT<DT>::kInf;
    return is ? AttnT<DT>::kOne : 0u;
}
template <int DT, Keep K>
__device__ __forceinline__ uint32_t keep_two(uint32_t w) {
    return keep_half<DT, K>(w & 0xffffu) | keep_half<DT, K>(w >> 16) << 16;
}
template <int DT, Keep K>
__device__ __forceinline__ u32x4_v keep(u32x4_v v) {
    u32x4_v r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = keep_two<DT, K>(v[i]);
    return r;
}
// the same for 32 columns x 16 keys
template <int DT>
__device__ __forceinline__ void add_kinds32(f32x16_v& o, u32x4_v v, u32x4_v on) {
    f32x16_v zero;
#pragma unroll
    for (int e = 0; e < 16; e++) zero[e] = 0.f;
    f32x16_v n = AttnT<DT>::mfma32(keep<DT, Keep::kPosInf>(v), on, zero);
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (n[e] > 0.f) o[e] += __builtin_huge_valf();
    n = AttnT<DT>::mfma32(keep<DT, Keep::kNegInf>(v), on, zero);
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (n[e] > 0.f) o[e] -= __builtin_huge_valf();
    n = AttnT<DT>::mfma32(keep<DT, Keep::kNan>(v), on, zero);
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (n[e] > 0.f) o[e] = __builtin_nanf("");
}
// v: 16 columns x 32 keys of V^T (A operand), on: 1 where a row sees a key (B operand); o: the rows' sums of those columns
template <int DT>
__device__ __forceinline__ void add_kinds(f32x4_v& o, u32x4_v v, u32x4_v on) {
    const f32x4_v zero = {0.f, 0.f, 0.f, 0.f};
    const f32x4_v pos = AttnT<DT>::mfma16(keep<DT, Keep::kPosInf>(v), on, zero);
    const f32x4_v neg = AttnT<DT>::mfma16(keep<DT, Keep::kNegInf>(v), on, zero);
    const f32x4_v nan = AttnT<DT>::mfma16(keep<DT, Keep::kNan>(v), on, zero);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float y = o[e];
        if (pos[e] > 0.f) y += __builtin_huge_valf();
        if (neg[e] > 0.f) y -= __builtin_huge_valf();
        o[e] = nan[e] > 0.f ? __builtin_nanf("") : y;
    }
}
