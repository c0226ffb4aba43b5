// v_mfma_f32_32x32x16 in f16 and bf16, and the pieces that attention builds on
// its lane layout (lane l, half h = l / 32, c = l % 32):
//   A (32 x 16): row c, k = 8 h .. 8 h + 7;  B (16 x 32): column c, the same k;
//   D (32 x 32): column c, register 4 j + r (j, r < 4) is row 8 j + 4 h + r.
// With keys as A's rows and queries as B's columns, a lane of S^T = K . Q^T holds
// 16 of 32 keys' scores of one query: a softmax row is one lane pair, and
// registers 8 i .. 8 i + 7 are already the B operand of O^T = V^T . P^T for the
// keys {16 i + 8 (e / 4) + 4 h + e % 4}, e < 8.
#pragma once

#include <algorithm>

#include "kernels.hpp"

namespace tlh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) void lds_void;

template <bool BF> __device__ __forceinline__ f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A softmax's numerators in f16 have their reference 7 (of an exponent of 2) below the
// maximum that set it, so that maximum's own is 2^7, and none is above 2^15, half of f16's
// range, as the reference lags by no more than 8. What f16 rounds to 0, or to a multiple of
// its smallest number 2^-24, is then off by at most 2^-32 of the largest a key: 2^-15 over
// 131072 keys, not the 2^-8 of numerators that begin at 1.
constexpr float F16_LIFT = 7.0f;
// ... in scores (finite where the scale nearly vanishes and no numerator does)
inline float f16_lift(float cs) { return std::min(F16_LIFT / cs, 1e30f); }

// eight f32 rounded to nearest even
template <bool BF> __device__ __forceinline__ uint4 pack8(const float (&p)[8]) {
    if constexpr (BF) {
        const bf16x8 v = {(__bf16)p[0], (__bf16)p[1], (__bf16)p[2], (__bf16)p[3],
                          (__bf16)p[4], (__bf16)p[5], (__bf16)p[6], (__bf16)p[7]};
        return __builtin_bit_cast(uint4, v);
    } else {
        const f16x8 v = {(_Float16)p[0], (_Float16)p[1], (_Float16)p[2], (_Float16)p[3],
                         (_Float16)p[4], (_Float16)p[5], (_Float16)p[6], (_Float16)p[7]};
        return __builtin_bit_cast(uint4, v);
    }
}
template <bool BF> __device__ __forceinline__ float unpack16(uint32_t h) {
    return BF ? bf16_to_f32((uint16_t)h) : h2f((uint16_t)h);
}
__device__ __forceinline__ uint32_t word4(const uint4 &v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }

// 16 bytes a lane from global memory straight to LDS: lane l's land at lds + 16 l
__device__ __forceinline__ void to_lds(const void *g, void *lds) {
    __builtin_amdgcn_global_load_lds(g, (lds_void *)lds, 16, 0, 0);
}

// a lane's value and its partner's (l ^ 32)
__device__ __forceinline__ float max_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

}  // namespace tlh
