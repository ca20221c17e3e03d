// sq8_text_quant.h — e4m3 codes of 128 values and their scale, sixteen lanes to a group, eight values a lane.
#pragma once

#include <type_traits>

#include "sq8_device.h"
#include "sq8_text.h"

namespace sq8 {

// Runs at any address: global loads and stores take them as they are, in one instruction. 8192 rows of 4095, normed, take
// 84 µs so and took 159 value by value (of 4096 46); their quantization 29 and 56 (23); an append to heads of 120 38 and
// 106.
typedef u32x4 __attribute__((aligned(1))) u32x4_any;
typedef u32x2 __attribute__((aligned(1))) u32x2_any;
typedef uint32_t __attribute__((aligned(1))) u32_any;

__device__ __forceinline__ float max8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    return m;
}

// The largest of 16 consecutive lanes (a group of 128 columns, eight a lane): four row rotations.
__device__ __forceinline__ float max_of_16(float m) {
    auto turn = [](float f, auto by) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(f), 0x120 + decltype(by)::value, 0xF, 0xF, true));
    };
    m = fmaxf(m, turn(m, std::integral_constant<int, 8>{}));
    m = fmaxf(m, turn(m, std::integral_constant<int, 4>{}));
    m = fmaxf(m, turn(m, std::integral_constant<int, 2>{}));
    return fmaxf(m, turn(m, std::integral_constant<int, 1>{}));
}

__device__ __forceinline__ float group_scale(float m) {
    const float q = m * (1.0f / 448.0f);
    return q > 1e-30f ? q : 1e-30f;
}

__device__ __forceinline__ void e4m3_codes(const float (&y)[8], float scale, uint32_t &lo, uint32_t &hi) {
    const Quotient by(scale);
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = by.of(y[e]);
    lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    lo = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], (int)lo, true);
    hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    hi = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], (int)hi, true);
}

}  // namespace sq8
