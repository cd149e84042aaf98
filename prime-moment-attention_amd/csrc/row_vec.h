// 16 bytes of a row of F32, BF16 or F16, wherever it starts, and its elements in fp32.
#pragma once

#include "prime_common.h"

namespace prime {

struct __attribute__((packed, aligned(2))) Raw {
    u32x4 v;
};

template <int DT>
constexpr int kVec = DT == PRIME_F32 ? 4 : 8;  // elements of 16 bytes

template <int DT>
__device__ __forceinline__ void widen(const u32x4 &v, float (&x)[kVec<DT>]) {
#pragma unroll
    for (int j = 0; j < kVec<DT>; ++j) {
        if constexpr (DT == PRIME_F32) x[j] = __uint_as_float(v[j]);
        else if constexpr (DT == PRIME_BF16) x[j] = __uint_as_float(j & 1 ? v[j / 2] & 0xFFFF0000u : v[j / 2] << 16);
        else x[j] = h16_bits_to_f32(static_cast<uint16_t>(j & 1 ? v[j / 2] >> 16 : v[j / 2]));
    }
}

// Each element rounded once.
template <int DT>
__device__ __forceinline__ u32x4 narrow(const float (&x)[kVec<DT>]) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < kVec<DT>; j += DT == PRIME_F32 ? 1 : 2) {
        if constexpr (DT == PRIME_F32) v[j] = __float_as_uint(x[j]);
        else if constexpr (DT == PRIME_BF16) v[j / 2] = f32_to_bf16_bits(x[j]) | static_cast<uint32_t>(f32_to_bf16_bits(x[j + 1])) << 16;
        else v[j / 2] = f32_to_h16_bits(x[j]) | static_cast<uint32_t>(f32_to_h16_bits(x[j + 1])) << 16;
    }
    return v;
}

}  // namespace prime
