// Reductions over the lanes of a wave by butterflies, within the vector unit where it can
// (a step through LDS waits some hundred cycles).
#pragma once

#include "common.hpp"

namespace tlh {

// A lane's value and its partner's at distance STEP = 1, 2, 4, .. (4 and 8 mirror groups
// whose lanes already agree, which is as good)
template <int STEP> __device__ __forceinline__ uint32_t wave_other(uint32_t v) {
    if constexpr (STEP == 1) return __builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true);
    else if constexpr (STEP == 2) return __builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true);
    else if constexpr (STEP == 4) return __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true);
    else if constexpr (STEP == 8) return __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true);
    else return __shfl_xor(v, STEP, 64);
}
template <int STEP, typename T> __device__ __forceinline__ T wave_swap(T v) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, wave_other<STEP>(__builtin_bit_cast(uint32_t, v)));
    else {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)wave_other<STEP>((uint32_t)(b >> 32)) << 32 | wave_other<STEP>((uint32_t)b));
    }
}
// f over the values of every `lanes` consecutive lanes (a power of two), in each of them
template <typename T, typename F> __device__ __forceinline__ T wave_all(T v, int lanes, F f) {
    if (lanes > 1) v = f(v, wave_swap<1>(v));
    if (lanes > 2) v = f(v, wave_swap<2>(v));
    if (lanes > 4) v = f(v, wave_swap<4>(v));
    if (lanes > 8) v = f(v, wave_swap<8>(v));
    if (lanes > 16) v = f(v, wave_swap<16>(v));
    if (lanes > 32) v = f(v, wave_swap<32>(v));
    return v;
}

}  // namespace tlh
