// sq8_f8_gemm.hip — products of e4m3 codes by e4m3 codes, a scale per 128 of K of an activation row and per
// 128 × 128 block of the weight:
//
//   C[i, j] = act( Σ_b sx[i, b] · sw[j / 128, b] · (Σ_{k in b} A[i, k] · W[j, k]) + bias[j] )
//
// A bf16 C is computed on v_mfma_f32_16x16x128_f8f6f4, whose K is one block: each instruction's sum is one block's,
// added into the fp32 accumulator with one multiply-add by the two scales' rounded product. That instruction sums in
// fp32 but for one thing, measured here: within each 8 consecutive K it aligns the products to the largest and drops
// what is under 2^-13 of that one's power of two. On normal operands that is 1.4e-5 of a result's size, a hundredth of
// what the rounding to bf16 then costs, and it runs at twice the bf16 rate. (v_mfma_f32_16x16x32_fp8_fp8 does the
// same.) An fp32 C is for callers who want the sums as they are: its codes are widened to bf16, exactly, for
// v_mfma_f32_16x16x32_bf16, whose products and sums are fp32.
//
// The weight is the first operand, so a lane ends with four consecutive outputs of one row; K is laid out alike for
// both operands (lane group h of four holds bytes 16h and 64 + 16h on), any such order giving the same products.
//
// A GLU's gate and up halves ([0, H) and [H, 2H) of the weight's rows) are blocked each by itself: the up half's
// scales start at row ⌈H/128⌉.
//
// K ends anywhere on a multiple of 16 (the host pads what does not): 16-byte runs past it are zeros. Rows past M
// and weight rows past the last read the last one; their results are not stored.
#include <hip/hip_runtime.h>

#include "sq8_device.h"
#include "sq8_text.h"

namespace sq8 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// A lane's codes 8·J .. 8·J + 7 of a block as bf16, exactly.
template <int J>
__device__ __forceinline__ bf16x8 widen_f8(const i32x8 &x) {
    uint32_t d0, d1, d2, d3;
    widen4<(int)W_FP8>((uint32_t)x[2 * J], d0, d1);
    widen4<(int)W_FP8>((uint32_t)x[2 * J + 1], d2, d3);
    return __builtin_bit_cast(bf16x8, u32x4{d0, d1, d2, d3});
}

// One block's sums of 16 weight rows by 16 activation rows.
template <bool F32>
__device__ __forceinline__ f32x4 block_sums(const i32x8 &w, const i32x8 &a) {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (F32) {
        static_for<0, 4>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen_f8<j>(w), widen_f8<j>(a), sum, 0, 0, 0);
        });
    } else {
        sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, sum, 0, 0, 0, 0, 0, 0);
    }
    return sum;
}

// One operand of block kb: the lane's 2 × 16 bytes of its row (`row` points at K = 0), zeros past K.
__device__ __forceinline__ i32x8 load_f8(const uint8_t *row, int kb, int h, int K) {
    const int at = kb * F8_GROUP + 16 * h;
    u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (at < K) lo = *reinterpret_cast<const u32x4 *>(row + at);
    if (at + 64 < K) hi = *reinterpret_cast<const u32x4 *>(row + at + 64);
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// Four consecutive outputs from column `col` of row `row`: bias, activation, store.
template <bool GLU, bool F32>
__device__ __forceinline__ void store4(const F8Args &p, int row, int col, f32x4 x, f32x4 u) {
    if (row >= p.M || col >= p.H) return;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = min(col + e, p.H - 1);
        float v = x[e];
        if (p.bias) v += p.bias[n];
        if constexpr (GLU) {
            float w = u[e];
            if (p.bias) w += p.bias[p.H + n];
            v = silu_glu(v, w);
        }
        y[e] = v;
    }
    const int64_t at = (int64_t)row * p.ldc + col;
    if (p.c_vec && col + 4 <= p.H) {
        if constexpr (F32) *reinterpret_cast<f32x4 *>(static_cast<float *>(p.c) + at) = f32x4{y[0], y[1], y[2], y[3]};
        else *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.c) + at) = u32x2{pack_bf16_rne(y[0], y[1]), pack_bf16_rne(y[2], y[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.H) {
                if constexpr (F32) static_cast<float *>(p.c)[at + e] = y[e];
                else static_cast<uint16_t *>(p.c)[at + e] = (uint16_t)(pack_bf16_rne(y[e], y[e]) & 0xFFFFu);
            }
    }
}

// Few rows: a workgroup of NW waves takes 16 output columns (GLU: of both halves) and TM tiles of 16 rows; the
// waves take the K blocks in turn, both operands straight from memory, and add up through LDS.
template <int TM, int NW, bool GLU, bool F32>
__global__ void __launch_bounds__(64 * NW) f8_short_kernel(const F8Args p) {
    constexpr int NT = GLU ? 2 : 1;
    __shared__ __attribute__((aligned(16))) f32x4 sums[NW][TM * NT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * (16 * TM);
    const uint8_t *wrow[NT];
    const float *sw[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        wrow[j] = p.w + ((int64_t)min(n0 + c, p.H - 1) + (int64_t)j * p.H) * p.ldw;
        sw[j] = p.sw + (int64_t)(n0 / F8_GROUP + j * p.up_block) * p.ldsw;
    }
    const uint8_t *arow[TM];
    const float *sx[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t row = min(m0 + 16 * i + c, p.M - 1);
        arow[i] = p.a + row * p.lda;
        sx[i] = p.sx + row * p.ldsx;
    }
    f32x4 acc[TM][NT];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int kb = wave; kb < p.KB; kb += NW) {
        i32x8 w[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j] = load_f8(wrow[j], kb, h, p.K);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const i32x8 a = load_f8(arow[i], kb, h, p.K);
            const float s = sx[i][kb];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const f32x4 part = block_sums<F32>(w[j], a);
                const float both = s * sw[j][kb];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[e], both, acc[i][j][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int i = wave; i < TM; i += NW) {
        f32x4 x[2] = {};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            f32x4 v = sums[0][i * NT + j][lane];
#pragma unroll
            for (int g = 1; g < NW; ++g) v += sums[g][i * NT + j][lane];
            x[j] = v;
        }
        store4<GLU, F32>(p, m0 + 16 * i + c, n0 + 4 * h, x[0], x[1]);
    }
}

template <int TM, bool GLU, bool F32>
hipError_t launch_short(const F8Args &p, hipStream_t stream) {
    constexpr int NW = 8;
    const dim3 grid((unsigned)((p.H + 15) / 16), (unsigned)((p.M + 16 * TM - 1) / (16 * TM)));
    hipLaunchKernelGGL((f8_short_kernel<TM, NW, GLU, F32>), grid, dim3(64 * NW), 0, stream, p);
    return hipGetLastError();
}

template <bool GLU, bool F32>
hipError_t launch(const F8Args &p, int cus, hipStream_t stream) {
    if (p.M <= 16) return launch_short<1, GLU, F32>(p, stream);
    if (p.M <= 32) return launch_short<2, GLU, F32>(p, stream);
    return launch_short<4, GLU, F32>(p, stream);
}

}  // namespace

hipError_t launch_f8_product(const F8Args &p, bool glu, bool out_f32, int cus, hipStream_t stream) {
    if (p.M == 0 || p.H == 0) return hipSuccess;
    if (glu) return out_f32 ? launch<true, true>(p, cus, stream) : launch<true, false>(p, cus, stream);
    return out_f32 ? launch<false, true>(p, cus, stream) : launch<false, false>(p, cus, stream);
}

}  // namespace sq8
