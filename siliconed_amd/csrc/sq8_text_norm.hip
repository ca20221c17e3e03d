// sq8_text_norm.hip — the passes that write a product's 8-bit operand in a text decoder: the RMS norm of the
// residual stream's new sum, and the quantization alone.
//
//   s' = r + x,  y = (s' · 1/sqrt(mean(s'²) + eps)) · w
//   e4m3: per 128 columns s = max(max|y| · fl(1/448), 1e-30), code = e4m3(y / s), nearest even
//   int8: per row s = max(max|y| / 127, 1e-30), code = clamp(rint(y / s), −128, 127)
//
// The sums, the norm and the scales are fp32; s' is rounded to the stream's type only where it is stored, so the
// norm sees the sum before that rounding. y/s is correctly rounded: an ulp of it decides a code where it lies
// halfway between two, and among bf16 values that is common (448 = 7 · 64: y = 3·2^j · max|y| is such a
// tie). It is under 449, which rounds to the largest code: none overflows to NaN.
//
// What is not finite: a NaN y is a NaN e4m3 code, and the other codes of its group are as without it; int8 has no code
// for one, so a row with a NaN y has a NaN scale, which makes its products NaN. An infinite y makes the scale of its
// group (e4m3) or row (int8) infinite, and the finite values' codes 0. A NaN s' makes every y of its row NaN, an infinite
// one itself NaN and the others 0 (1/sqrt is 0 there).
#include <hip/hip_runtime.h>

#include "sq8_device.h"
#include "sq8_quant.h"
#include "sq8_text.h"
#include "sq8_text_quant.h"

namespace sq8 {
namespace {

// Eight consecutive values from element `at` of a bf16 or fp32 array: as they lie, so that every load of a row is under
// way before the first is waited for, then as fp32; element e of the row is real when col + e < cols (WHOLE: rows are
// whole runs of eight).
struct Raw8 {
    u32x4 a, b;  // bf16: a
};

template <bool WHOLE>
__device__ __forceinline__ Raw8 load8(const void *base, bool bf16, int64_t at, int col, int cols) {
    Raw8 v = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
    if (col >= cols) return v;
    const uint8_t *const src = static_cast<const uint8_t *>(base) + at * (bf16 ? 2 : 4);
    if (WHOLE || col + 8 <= cols) {
        v.a = *reinterpret_cast<const u32x4_any *>(src);
        if (!bf16) v.b = *reinterpret_cast<const u32x4_any *>(src + 16);
    } else if (bf16) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (col + e < cols) v.a[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(src)[e] << (16 * (e & 1));
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (col + e < cols) (e < 4 ? v.a : v.b)[e & 3] = reinterpret_cast<const uint32_t *>(src)[e];
    }
    return v;
}

__device__ __forceinline__ void widen8(const Raw8 &x, bool bf16, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = __uint_as_float(bf16 ? (e & 1 ? x.a[e >> 1] & 0xFFFF0000u : x.a[e >> 1] << 16) : x.a[e]);
        v[4 + e] = __uint_as_float(bf16 ? (e & 1 ? x.a[2 + (e >> 1)] & 0xFFFF0000u : x.a[2 + (e >> 1)] << 16) : x.b[e]);
    }
}

template <bool WHOLE>
__device__ __forceinline__ void store8(void *base, bool bf16, int64_t at, int col, int cols, const float (&v)[8]) {
    uint8_t *const dst = static_cast<uint8_t *>(base) + at * (bf16 ? 2 : 4);
    if (WHOLE || col + 8 <= cols) {
        if (bf16) {
            *reinterpret_cast<u32x4_any *>(dst) =
                u32x4{pack_bf16_rne(v[0], v[1]), pack_bf16_rne(v[2], v[3]), pack_bf16_rne(v[4], v[5]), pack_bf16_rne(v[6], v[7])};
        } else {
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<u32x4_any *>(dst + 4 * e) = u32x4{__float_as_uint(v[e]), __float_as_uint(v[e + 1]),
                                                                    __float_as_uint(v[e + 2]), __float_as_uint(v[e + 3])};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (col + e < cols) {
                if (bf16) reinterpret_cast<uint16_t *>(dst)[e] = (uint16_t)round_bf16(v[e]);
                else reinterpret_cast<float *>(dst)[e] = v[e];
            }
    }
}

template <bool WHOLE>
__device__ __forceinline__ void store_codes8(uint8_t *dst, int col, int cols, uint32_t lo, uint32_t hi) {
    if (WHOLE || col + 8 <= cols) {
        *reinterpret_cast<u32x2_any *>(dst) = u32x2{lo, hi};
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (col + e < cols) dst[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
}

// clamp(rint(y / s)) from the reciprocal's product where that surely rounds alike (quant::store_codes).
__device__ __forceinline__ void int8_codes(const float (&y)[8], float scale, uint32_t &lo, uint32_t &hi) {
    const float recip = __fdiv_rn(1.0f, scale);
    float c[8];
    bool hard = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = y[e] * recip;
        c[e] = rintf(q);
        hard |= fabsf(q - c[e]) > 0.5f - 0x1p-14f;
    }
    if (hard) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = rintf(__fdiv_rn(y[e], scale));
    }
    lo = hi = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        lo |= (uint32_t)(uint8_t)(int8_t)(int)fminf(fmaxf(c[e], -128.0f), 127.0f) << (8 * e);
        hi |= (uint32_t)(uint8_t)(int8_t)(int)fminf(fmaxf(c[4 + e], -128.0f), 127.0f) << (8 * e);
    }
}

// The larger of the two, a NaN if either is one (fmaxf would drop it).
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Rows in turn over the grid, T threads a row, each holding IT runs of 8 columns 8·T apart in registers: one read
// of x and r, w once a workgroup.
//
// Memory bounds long ones: 8192 rows of 4096 on a bf16 stream (236 MB) take 42 to 45 µs, 5.2 to 5.6 TB/s where a large copy
// runs at 5.0; on an fp32 stream (370 MB) 75. One row takes 3.0 µs, 2.3 of them the launch; the loads of x and r under
// way together are 0.3 µs of that.
template <bool INT8, int T, int IT, bool WHOLE>
__global__ void __launch_bounds__(T) add_norm_kernel(const AddNormArgs p) {
    constexpr int WAVES = T / 64;
    __shared__ float sums[2][WAVES], tops[2][WAVES];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    float w[IT][8];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int col = 8 * (tid + T * i);
        widen8(load8<WHOLE>(p.w, false, col, col, p.cols), false, w[i]);
    }
    int turn = 0;
    for (unsigned row = blockIdx.x; row < (unsigned)p.rows; row += gridDim.x, turn ^= 1) {
        float v[IT][8];
        // All of a row's loads at once, or a thousand threads of 128 registers each, half.
        constexpr int AT_ONCE = T * IT > 2048 ? IT / 2 : IT;
#pragma unroll
        for (int i0 = 0; i0 < IT; i0 += AT_ONCE) {
            Raw8 x[AT_ONCE], r[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int col = 8 * (tid + T * (i0 + i));
                x[i] = load8<WHOLE>(p.x, p.x_bf16, (int64_t)row * p.ldx + col, col, p.cols);
                if (p.r) r[i] = load8<WHOLE>(p.r, p.r_bf16, (int64_t)row * p.ldr + col, col, p.cols);
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int col = 8 * (tid + T * (i0 + i));
                float (&y)[8] = v[i0 + i];
                widen8(x[i], p.x_bf16, y);
                if (p.r) {
                    float old[8];
                    widen8(r[i], p.r_bf16, old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = old[e] + y[e];
                    if (p.ro && col < p.cols) store8<WHOLE>(p.ro, p.r_bf16, (int64_t)row * p.ldro + col, col, p.cols, y);
                }
            }
            if constexpr (AT_ONCE < IT) __builtin_amdgcn_sched_barrier(0);
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[i][e], v[i][e], ss);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
        if constexpr (WAVES > 1) {
            // One barrier a row: a wave is at most one row ahead, and writes the other half of `sums` there.
            if (lane == 0) sums[turn][wave] = ss;
            __syncthreads();
            ss = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) ss += sums[turn][i];
        }
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)p.cols) + p.eps));
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = (v[i][e] * r) * w[i][e];
            if constexpr (INT8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max_or_nan(top, fabsf(v[i][e]));
            }
        }
        if constexpr (INT8) {
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) top = max_or_nan(top, __shfl_xor(top, o, 64));
            if constexpr (WAVES > 1) {
                if (lane == 0) tops[turn][wave] = top;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < WAVES; ++i) top = max_or_nan(top, tops[turn][i]);
            }
            const float scale = top != top ? top : quant::row_scale(top);
            if (tid == 0) p.scales[row] = scale;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int col = 8 * (tid + T * i);
                if (col >= p.cols) break;
                uint32_t lo, hi;
                int8_codes(v[i], scale, lo, hi);
                store_codes8<WHOLE>(p.codes + (int64_t)row * p.ldq + col, col, p.cols, lo, hi);
            }
        } else {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int col = 8 * (tid + T * i);
                const float scale = group_scale(max_of_16(max8(v[i])));  // in every lane: the 16 agree
                if (col >= p.cols) continue;
                uint32_t lo, hi;
                e4m3_codes(v[i], scale, lo, hi);
                store_codes8<WHOLE>(p.codes + (int64_t)row * p.ldq + col, col, p.cols, lo, hi);
                if ((tid & 15) == 0) p.scales[(int64_t)row * p.lds + col / F8_GROUP] = scale;
            }
        }
    }
}

// Sixteen lanes a group of 128 columns, groups in order over the grid: memory bounds it, 8192 rows of 12288 (305 MB) in
// 61.7 µs, 4.9 TB/s; 48 rows of 4096 take 2.4 µs, a launch.
template <bool WHOLE>
__global__ void __launch_bounds__(256) quantize_groups_kernel(const void *x, bool x_bf16, int64_t ldx, unsigned total,
                                                              unsigned groups, int cols, uint8_t *codes, int64_t ldq,
                                                              float *scales, int64_t lds) {
    const unsigned sub = threadIdx.x & 15;
    for (unsigned g = blockIdx.x * 16 + (threadIdx.x >> 4); g < total; g += gridDim.x * 16) {
        const unsigned row = g / groups, group = g - row * groups;
        const int col = (int)(group * F8_GROUP + sub * 8);
        float v[8];
        widen8(load8<WHOLE>(x, x_bf16, (int64_t)row * ldx + col, col, cols), x_bf16, v);
        const float scale = group_scale(max_of_16(max8(v)));
        if (col < cols) {
            uint32_t lo, hi;
            e4m3_codes(v, scale, lo, hi);
            store_codes8<WHOLE>(codes + (int64_t)row * ldq + col, col, cols, lo, hi);
        }
        if (sub == 0) scales[(int64_t)row * lds + group] = scale;
    }
}

// A thread 16 bytes of the destination.
__global__ void __launch_bounds__(256) pad_bytes_kernel(const uint8_t *src, int64_t lds, uint8_t *dst, int64_t ldd,
                                                        int64_t runs, unsigned row_runs, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < runs; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / row_runs;
        const int64_t at = (i - row * row_runs) * 16;
        u32x4 run = {0, 0, 0, 0};
        if (at + 16 <= n) {
            run = *reinterpret_cast<const u32x4_any *>(src + row * lds + at);
        } else {
#pragma unroll
            for (int e = 0; e < 15; ++e)
                if (at + e < n) run[e >> 2] |= (uint32_t)src[row * lds + at + e] << (8 * (e & 3));
        }
        *reinterpret_cast<u32x4 *>(dst + row * ldd + at) = run;
    }
}

}  // namespace

hipError_t launch_add_norm(const AddNormArgs &p, bool int8, int cus, hipStream_t stream) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    const bool whole = p.cols % 8 == 0;
#define SQ8_ADD_NORM(T, IT)                                                                                          \
    do {                                                                                                             \
        const int most = cus * (2048 / T), grid = p.rows < most ? p.rows : most;                                      \
        if (int8 && whole) hipLaunchKernelGGL((add_norm_kernel<true, T, IT, true>), dim3(grid), dim3(T), 0, stream, p); \
        else if (int8) hipLaunchKernelGGL((add_norm_kernel<true, T, IT, false>), dim3(grid), dim3(T), 0, stream, p);  \
        else if (whole) hipLaunchKernelGGL((add_norm_kernel<false, T, IT, true>), dim3(grid), dim3(T), 0, stream, p);   \
        else hipLaunchKernelGGL((add_norm_kernel<false, T, IT, false>), dim3(grid), dim3(T), 0, stream, p);           \
        return hipGetLastError();                                                                                    \
    } while (0)
    if (p.cols <= 512) SQ8_ADD_NORM(64, 1);
    if (p.cols <= 1024) SQ8_ADD_NORM(64, 2);
    if (p.cols <= 4096) SQ8_ADD_NORM(256, 2);
    if (p.cols <= 8192) SQ8_ADD_NORM(256, 4);
    if (p.cols <= 16384) SQ8_ADD_NORM(1024, 2);
    if (p.cols <= kAddNormCols) SQ8_ADD_NORM(1024, 4);
#undef SQ8_ADD_NORM
    return hipErrorInvalidValue;
}

hipError_t launch_quantize_groups(const void *x, bool x_bf16, int64_t ldx, int rows, int cols, uint8_t *codes, int64_t ldq,
                                  float *scales, int64_t lds, hipStream_t stream) {
    if (rows == 0 || cols == 0) return hipSuccess;
    const int64_t groups = (cols + F8_GROUP - 1) / F8_GROUP, total = rows * groups;
    if (total > INT32_MAX - 65536 * 16) return hipErrorInvalidValue;
    const int64_t want = (total + 15) / 16;
    const dim3 grid((unsigned)(want < 65536 ? want : 65536));
    if (cols % 8 == 0)
        hipLaunchKernelGGL(quantize_groups_kernel<true>, grid, dim3(256), 0, stream, x, x_bf16, ldx, (unsigned)total,
                           (unsigned)groups, cols, codes, ldq, scales, lds);
    else
        hipLaunchKernelGGL(quantize_groups_kernel<false>, grid, dim3(256), 0, stream, x, x_bf16, ldx, (unsigned)total,
                           (unsigned)groups, cols, codes, ldq, scales, lds);
    return hipGetLastError();
}

hipError_t launch_pad_bytes(const void *src, int64_t lds, void *dst, int64_t ldd, int64_t rows, int64_t n,
                            hipStream_t stream) {
    if (rows == 0 || ldd == 0) return hipSuccess;
    const int64_t runs = rows * (ldd / 16), want = (runs + 255) / 256;
    hipLaunchKernelGGL(pad_bytes_kernel, dim3((unsigned)(want < 65536 ? want : 65536)), dim3(256), 0, stream,
                       static_cast<const uint8_t *>(src), lds, static_cast<uint8_t *>(dst), ldd, runs, (unsigned)(ldd / 16), n);
    return hipGetLastError();
}

}  // namespace sq8
