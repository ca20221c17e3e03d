// sq8_text_device.h — what the kernels of a text decoder's heads share: runs of a head's values in and out, e4m3 codes as
// bf16, a wave's running sums, tiles shared out over workgroups.
#pragma once

#include <type_traits>

#include "sq8_device.h"
#include "sq8_text.h"
#include "sq8_text_quant.h"

namespace sq8 {

__device__ __forceinline__ float bf16_f32(uint32_t bits) { return __uint_as_float(bits << 16); }

template <int W>
__device__ __forceinline__ void load_run(const uint16_t *src, float (&v)[W]) {
    if constexpr (W == 1) {
        v[0] = bf16_f32(src[0]);
    } else {
        typename std::conditional<W == 8, u32x4, u32x2>::type d;
        if constexpr (W == 8) d = *reinterpret_cast<const u32x4_any *>(src);
        else d = *reinterpret_cast<const u32x2_any *>(src);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) {
            v[2 * e] = bf16_f32(d[e] & 0xFFFFu);
            v[2 * e + 1] = __uint_as_float(d[e] & 0xFFFF0000u);
        }
    }
}

template <int W>
__device__ __forceinline__ void load_angles(const float *src, float (&v)[W]) {
    if constexpr (W == 1) {
        v[0] = src[0];
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const u32x4 d = reinterpret_cast<const u32x4_any *>(src)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * i + e] = __uint_as_float(d[e]);
        }
    }
}

template <int W>
__device__ __forceinline__ void store_bf16(uint16_t *dst, const float (&v)[W]) {
    if constexpr (W == 8)
        *reinterpret_cast<u32x4_any *>(dst) = u32x4{pack_bf16_rne(v[0], v[1]), pack_bf16_rne(v[2], v[3]), pack_bf16_rne(v[4], v[5]),
                                                    pack_bf16_rne(v[6], v[7])};
    else if constexpr (W == 4)
        *reinterpret_cast<u32x2_any *>(dst) = u32x2{pack_bf16_rne(v[0], v[1]), pack_bf16_rne(v[2], v[3])};
    else
        dst[0] = (uint16_t)(pack_bf16_rne(v[0], v[0]) & 0xFFFFu);
}

template <int W>
__device__ __forceinline__ void store_e4m3(uint8_t *dst, const float (&v)[W], const Quotient &by) {
    float q[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
        const float near = v[e] * by.r;
        const float t = fabsf(near) < INFINITY ? by.of(v[e]) : near;
        q[e] = t != t ? t : fminf(fmaxf(t, -448.0f), 448.0f);
    }
    if constexpr (W > 1) {
        auto four = [&](int e) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[e], q[e + 1], 0, false);
            return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[e + 2], q[e + 3], lo, true);
        };
        if constexpr (W == 8) *reinterpret_cast<u32x2_any *>(dst) = u32x2{four(0), four(4)};
        else *reinterpret_cast<u32_any *>(dst) = four(0);
    } else {
        dst[0] = (uint8_t)((uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[0], 0, false) & 0xFFu);
    }
}

// How a batch's tiles are shared out: the first `more` of `groups` workgroups take each + 1, the others `each`, in
// order. (Fewer workgroups of four tiles or more where there are not enough for all: slower, 20 µs against 12 at one
// sequence of 777.)
struct Share {
    int groups, each, more;
    __device__ __forceinline__ Share() {}
    __device__ __forceinline__ Share(int total, int most) {
        groups = min(most, total);
        each = groups > 0 ? total / groups : 0;
        more = groups > 0 ? total - each * groups : 0;
    }
    __device__ __forceinline__ int first(int g) const { return g * each + min(g, more); }
    __device__ __forceinline__ int of(int tile) const {
        return tile < more * (each + 1) ? tile / (each + 1) : more + (tile - more * (each + 1)) / each;
    }
};

// The sum of v over this lane and those before it.
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// The larger (the sum) of a value over the four lanes of a column (16 apart): the swaps leave each row's neighbour's, and
// each half's other's, in the second of the pair.
template <bool SUM>
__device__ __forceinline__ float over_rows(float v) {
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    auto both = [](u32x2_t r) {
        const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
        return SUM ? a + b : fmaxf(a, b);
    };
    v = both(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return both(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}

template <int N>
struct Raw {
    uint32_t d[N];
};

template <int N>
__device__ __forceinline__ Raw<N> load_raw(const uint8_t *src) {
    Raw<N> r;
    if constexpr (N == 1) {
        r.d[0] = *reinterpret_cast<const uint32_t *>(src);
    } else if constexpr (N == 2) {
        const u32x2 v = *reinterpret_cast<const u32x2 *>(src);
        r.d[0] = v[0]; r.d[1] = v[1];
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4 v = reinterpret_cast<const u32x4 *>(src)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) r.d[4 * i + e] = v[e];
        }
    }
    return r;
}

// Two e4m3 codes (bytes 2W, 2W + 1) as a bf16 pair, exactly.
template <int W>
__device__ __forceinline__ uint32_t bf16_of_e4m3(uint32_t d) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, 1.0f, W != 0));
}

// 1 / l, or 0 where nothing was added (a NaN stays one).
__device__ __forceinline__ float inverse(float l) { return l > 0.0f ? __fdiv_rn(1.0f, l) : l == 0.0f ? 0.0f : l; }

}  // namespace sq8
