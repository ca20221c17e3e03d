// sq8_f8_gemm.hip — products of e4m3 codes by e4m3 codes, a scale per 128 of K of an activation row and per
// 128 × 128 block of the weight:
//
//   C[i, j] = act( Σ_b sx[i, b] · sw[j / 128, b] · (Σ_{k in b} A[i, k] · W[j, k]) + bias[j] )
//
// A bf16 C is computed on v_mfma_f32_16x16x128_f8f6f4, whose K is one block: each instruction's sum is one block's,
// added into the fp32 accumulator with one multiply-add by the two scales' rounded product. That instruction sums in
// fp32 but for one thing, measured here: within each 8 consecutive K it aligns the products to the largest and drops
// what is under 2^-13 of that one's power of two. On normal operands that is 1.4e-5 of a result's size, a hundredth of
// what the rounding to bf16 then costs; at worst it is 7 · 2^-13 of the largest product of each eight, where e4m3's own
// rounding of a factor may have put that product off by 2^-4. It runs at twice the bf16 rate, and without the widening:
// one row by K = 4096, N = 24576 (GLU) takes 21.6 µs so and 25.4 on the bf16 instructions. (v_mfma_f32_16x16x32_fp8_fp8
// drops the same.) An fp32 C is for callers who want the sums as they are: its codes are widened to bf16, exactly, for
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
#include "sq8_text_quant.h"
#include "sq8_wdirect_kernel.h"

namespace sq8 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// A lane's codes 8·J .. 8·J + 7 of a block as bf16, exactly (the conversion's scale is 1): two codes an instruction.
template <int J>
__device__ __forceinline__ bf16x8 widen_f8(const i32x8 &x) {
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)x[2 * J + i], 1.0f, false));
        y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)x[2 * J + i], 1.0f, true));
    }
    return __builtin_bit_cast(bf16x8, y);
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

// N consecutive outputs, the first `real` of them, from element `at` of C.
template <int N, bool F32>
__device__ __forceinline__ void store_run(void *c, int64_t at, int real, int vec, const float (&y)[N]) {
    if (vec && real == N) {
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < N; e += 4)
                *reinterpret_cast<f32x4 *>(static_cast<float *>(c) + at + e) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        } else {
            uint16_t *to = static_cast<uint16_t *>(c) + at;
            if (N == 4 || vec < 8) {
#pragma unroll
                for (int e = 0; e < N; e += 4)
                    *reinterpret_cast<u32x2 *>(to + e) = u32x2{pack_bf16_rne(y[e], y[e + 1]), pack_bf16_rne(y[e + 2], y[e + 3])};
            } else {
#pragma unroll
                for (int e = 0; e + 8 <= N; e += 8)
                    *reinterpret_cast<u32x4 *>(to + e) = u32x4{pack_bf16_rne(y[e], y[e + 1]), pack_bf16_rne(y[e + 2], y[e + 3]),
                                                               pack_bf16_rne(y[e + 4], y[e + 5]), pack_bf16_rne(y[e + 6], y[e + 7])};
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < real) {
                if constexpr (F32) static_cast<float *>(c)[at + e] = y[e];
                else static_cast<uint16_t *>(c)[at + e] = (uint16_t)(pack_bf16_rne(y[e], y[e]) & 0xFFFFu);
            }
    }
}

// Four consecutive outputs from column `col` of row `row`: bias, activation, store.
template <bool GLU, bool F32>
__device__ __forceinline__ void store4(const F8Args &p, int row, int col, f32x4 x, f32x4 u) {
    if (row >= p.M || col >= p.H) return;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = min(col + e, p.H - 1);
        y[e] = x[e];
        if (p.bias) y[e] += p.bias[n];
        if constexpr (GLU) y[e] = silu_glu(y[e], p.bias ? u[e] + p.bias[p.H + n] : u[e]);
    }
    store_run<4, F32>(p.c, (int64_t)row * p.ldc + col, p.H - col < 4 ? p.H - col : 4, p.c_vec, y);
}

// The waves' sums, in their order, and the outputs of TM tiles of 16 rows by NO × 16 columns.
template <int TM, int NO, int NW, bool GLU, bool F32>
__device__ __forceinline__ void add_waves(const F8Args &p, f32x4 (*sums)[TM * (GLU ? 2 * NO : NO)][64],
                                          const f32x4 (&acc)[TM][GLU ? 2 * NO : NO], int m0, int n0, int wave, int lane) {
    constexpr int NT = GLU ? 2 * NO : NO;
    const int c = lane & 15, h = lane >> 4;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int q = wave; q < TM * NO; q += NW) {
        const int i = q / NO, j = q - i * NO;
        f32x4 x[2] = {};
#pragma unroll
        for (int half = 0; half < NT / NO; ++half) {
            f32x4 v = sums[0][i * NT + half * NO + j][lane];
#pragma unroll
            for (int g = 1; g < NW; ++g) v += sums[g][i * NT + half * NO + j][lane];
            x[half] = v;
        }
        store4<GLU, F32>(p, m0 + 16 * i + c, n0 + 16 * j + 4 * h, x[0], x[1]);
    }
}

// Few rows: a workgroup of NW waves takes NO × 16 output columns (GLU: of both halves) and TM tiles of 16 rows; the
// waves take the K blocks in turn, both operands straight from memory, U blocks' loads in flight, and add up through
// LDS.
//
// The weight's bytes bound it: one row by K = 4096, N = 6144 (25 MB) takes 7.1 µs, 3.5 TB/s with 2.5 of them the launch,
// and a gate and up product of N = 24576 (101 MB) 20 to 22, 4.6 to 5 TB/s. Fragments that lanes load from 16 rows at
// once come in at 34 KB/µs a CU (whole rows of 128 bytes: 115), which is above a CU's share of the memory's rate but
// not by much: past 16 rows, whose loads then outweigh the weight's, the tile kernel's way through LDS is the faster.
template <int TM, int NO, int NW, int U, bool GLU, bool F32>
__global__ void __launch_bounds__(64 * NW) f8_short_kernel(const F8Args p) {
    constexpr int NT = GLU ? 2 * NO : NO;
    __shared__ __attribute__((aligned(16))) f32x4 sums[NW][TM * NT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int n0 = blockIdx.x * (16 * NO), m0 = blockIdx.y * (16 * TM);
    const uint8_t *wrow[NT];
    const float *sw[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int half = j / NO, at = n0 + 16 * (j - half * NO);
        wrow[j] = p.w + ((int64_t)min(at + c, p.H - 1) + (int64_t)half * p.H) * p.ldw;
        sw[j] = p.sw + (int64_t)(min(at, p.H - 1) / F8_GROUP + half * p.up_block) * p.ldsw;
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
    for (int k0 = wave; k0 < p.KB; k0 += U * NW) {
        i32x8 w[U][NT], a[U][TM];
        float s_x[U][TM], s_w[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = min(k0 + u * NW, p.KB - 1);  // past the last: read, not used
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                w[u][j] = load_f8(wrow[j], kb, h, p.K);
                s_w[u][j] = sw[j][kb];
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                a[u][i] = load_f8(arow[i], kb, h, p.K);
                s_x[u][i] = sx[i][kb];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u * NW >= p.KB) break;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const f32x4 part = block_sums<F32>(w[u][j], a[u][i]);
                    const float both = s_x[u][i] * s_w[u][j];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[e], both, acc[i][j][e]);
                }
        }
    }
    add_waves<TM, NO, NW, GLU, F32>(p, sums, acc, m0, n0, wave, lane);
}

// A few rows of values that are still to be quantized: as the short kernel, but the workgroup first makes its rows' codes
// and scales, GROUPS groups of 128 at most, in LDS, so that no other kernel runs before (a launch is 2.4 µs, among
// other kernels nearly 5). The rows' loads go first, the weight's next: the codes are made while those are on their way.
// Then U blocks of the weight are always under way, each asked for when its predecessor is used.
template <int NO, int U, int GROUPS, bool F32>
__global__ void __launch_bounds__(512) f8_staged_kernel(const F8Args p) {
    constexpr int NW = 8, IT = GROUPS / 32;
    __shared__ __attribute__((aligned(16))) uint8_t staged[GROUPS * F8_GROUP];
    __shared__ float scales[GROUPS];
    __shared__ __attribute__((aligned(16))) f32x4 sums[NW][NO][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int n0 = blockIdx.x * (16 * NO);

    // ---- the rows' loads: sixteen threads a group, eight values each ----
    const int groups = p.M * p.KB, sub = threadIdx.x & 15;
    u32x4 raw[IT];
    int to[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int g = 32 * i + (int)(threadIdx.x >> 4);
        raw[i] = u32x4{0, 0, 0, 0};
        to[i] = 0;
        if (32 * i >= groups) continue;
        const int row = g / p.KB, kb = g - row * p.KB, col = kb * F8_GROUP + 8 * sub;
        to[i] = g * F8_GROUP + (((sub >> 1) ^ (row & 7)) << 4) + 8 * (sub & 1);  // 16-byte runs permuted: rows on other banks
        if (g < groups && col < p.K) raw[i] = *reinterpret_cast<const u32x4 *>(p.x + row * p.ldx + col);
    }

    // ---- the weight's ----
    const uint8_t *wrow[NO];
    const float *sw[NO];
#pragma unroll
    for (int j = 0; j < NO; ++j) {
        wrow[j] = p.w + (int64_t)min(n0 + 16 * j + c, p.H - 1) * p.ldw;
        sw[j] = p.sw + (int64_t)(min(n0 + 16 * j, p.H - 1) / F8_GROUP) * p.ldsw;
    }
    const int mine = p.KB > wave ? (p.KB - wave + NW - 1) / NW : 0;  // this wave's blocks
    i32x8 w[U][NO];
    float s_w[U][NO];
    auto load = [&](auto uc, int n) {
        constexpr int u = decltype(uc)::value;
        const int kb = min(wave + n * NW, p.KB - 1);
#pragma unroll
        for (int j = 0; j < NO; ++j) {
            w[u][j] = load_f8(wrow[j], kb, h, p.K);
            s_w[u][j] = sw[j][kb];
        }
    };
    if (mine > 0) static_for<0, U>([&](auto uc) { load(uc, min((int)decltype(uc)::value, mine - 1)); });

    // ---- the rows' codes ----
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        if (32 * i >= groups) continue;
        const int g = 32 * i + (int)(threadIdx.x >> 4);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(e & 1 ? raw[i][e >> 1] & 0xFFFF0000u : raw[i][e >> 1] << 16);
        const float scale = group_scale(max_of_16(max8(v)));
        uint32_t lo, hi;
        e4m3_codes(v, scale, lo, hi);
        if (g < groups) {
            *reinterpret_cast<u32x2 *>(staged + to[i]) = u32x2{lo, hi};
            if (sub == 0) scales[g] = scale;
        }
    }
    __syncthreads();

    f32x4 acc[1][NO];
#pragma unroll
    for (int j = 0; j < NO; ++j) acc[0][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int row = min(c, p.M - 1), runs[2] = {(h ^ (row & 7)) << 4, ((4 + h) ^ (row & 7)) << 4};
    auto use = [&](auto uc, int n) {
        constexpr int u = decltype(uc)::value;
        const int g = row * p.KB + wave + n * NW;
        const u32x4 lo = *reinterpret_cast<const u32x4 *>(staged + g * F8_GROUP + runs[0]);
        const u32x4 hi = *reinterpret_cast<const u32x4 *>(staged + g * F8_GROUP + runs[1]);
        const i32x8 a = {(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
        const float s_x = scales[g];
#pragma unroll
        for (int j = 0; j < NO; ++j) {
            const f32x4 part = block_sums<F32>(w[u][j], a);
            const float both = s_x * s_w[u][j];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[0][j][e] = __builtin_fmaf(part[e], both, acc[0][j][e]);
        }
    };
    int n = 0;
    for (; n + 2 * U <= mine; n += U)
        static_for<0, U>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            use(uc, n + u);
            load(uc, n + U + u);
        });
    static_for<0, U>([&](auto uc) {
        if (n + (int)decltype(uc)::value < mine) use(uc, n + decltype(uc)::value);
    });
    n += U;
    if (n < mine) {
        static_for<0, U>([&](auto uc) { load(uc, min(n + (int)decltype(uc)::value, mine - 1)); });
        static_for<0, U>([&](auto uc) {
            if (n + (int)decltype(uc)::value < mine) use(uc, n + decltype(uc)::value);
        });
    }
    add_waves<1, NO, NW, false, F32>(p, sums, acc, 0, n0, wave, lane);
}

// Many rows: tiles of BM rows by BN weight rows (GLU: half of them of each half), WM × WN waves.
//
// Both operands go to LDS by direct loads, a block (128 bytes) of each row a step, in NS stages. 16-byte runs of a
// row are permuted within it (by key_a, key_w) so that the eight rows a fragment read touches at once lie on different
// banks. The rows' scales go to LDS too, four blocks at a time where they can be read so (a load of one block's scales
// a step, a line for each row, cost the small tiles a tenth).
//
// Each wave multiplies (BM/WM) × (BN/WN) in 16 × 16 parts, a row of TN parts at a time, the weight's fragments held for
// the step and the rows' read two parts ahead; the multiply-adds that scale one row of parts go between the matrix
// instructions of the next. The step's one barrier stands before its last two rows of parts, whose fragments are in
// registers by then: the stage is free for the loads of NS steps on, which go between the last matrix instructions (in
// one burst behind the barrier they held up the small tiles' steps by a seventh), the next step's loads have landed,
// and its first fragments are read under those instructions too.
//
// What bounds it: at M = 8192, K = 4096, N = 24576 (GLU) the 256 × 256 tile runs at the card's power limit, 703 to 785 µs
// or 2.10 to 2.35 PFLOP/s on normal operands and 578 on zeros, its matrix instructions busy for 55 % of the cycles (a
// library's product of such codes with one scale a tensor, no GLU: 650). A 64-row tile's step is a chain of a barrier, reads, four
// to eight matrix instructions a wave and their scaling, 0.36 µs where the instructions alone are 0.06, so few rows want
// many workgroups: N = 24576 (GLU) has 192 of 64 × 128, 27.6 µs at M = 48 (100 MB, 3.7 TB/s), and N = 4096 takes its K in
// four parts, 10.1 µs at M = 64, K = 4096, and 17.7 at K = 12288. (More waves a tile, sets of waves on K parts of one
// workgroup, deeper stages and fragments read a whole block ahead took as long or longer.)
//
// The weight row an instruction's row stands for is chosen so that a lane ends with consecutive outputs: lane group
// h, register r of part j is output 4·NTO·h + 4j + r of the wave's (NTO parts wide).
template <int BM, int BN, int WM, int WN, int NS, bool GLU, bool F32>
struct TileShape {
    static constexpr int THREADS = 64 * WM * WN;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;  // parts of a wave
    static constexpr int NTO = GLU ? TN / 2 : TN;               // and those of one half
    static constexpr int OUT = GLU ? BN / 2 : BN;               // outputs of a tile
    static constexpr int STAGE = (BM + BN) * F8_GROUP;
    static constexpr int SCALES = BM * 16;                      // four blocks' scales of the rows
    static constexpr int LDS = NS * STAGE + 2 * SCALES;
    static constexpr bool SPLIT = BM == 64;                       // K may be split
    static_assert(NS <= 4, "two buffers of scales hold the blocks under way");
    static_assert(TM * 16 * WM == BM && TN * 16 * WN == BN && (!GLU || TN % 2 == 0), "whole parts");
    static_assert(NTO == 1 || NTO == 2 || NTO == 4, "a lane's outputs");
};

__device__ __forceinline__ int key_a(int row) { return row & 7; }
// Rows 4·NTO·(c / 4) + 4j + c mod 4 of eight consecutive c: different keys.
template <int NTO>
__device__ __forceinline__ int key_w(int row) {
    constexpr int SHIFT = NTO == 4 ? 4 : NTO == 2 ? 3 : 2;
    return (row & 3) | ((row >> SHIFT) & 1) << 2;
}

template <int BM, int BN, int WM, int WN, int NS, bool GLU, bool F32>
__global__ void __attribute__((amdgpu_flat_work_group_size(64 * WM * WN, 64 * WM * WN), amdgpu_waves_per_eu(2, 2)))
f8_tile_kernel(const F8Args p, int tiles_m, int tiles_n) {
    using S = TileShape<BM, BN, WM, WN, NS, GLU, F32>;
    constexpr int TM = S::TM, TN = S::TN, NTO = S::NTO, WAVES = WM * WN;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[S::LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    int tm, tn;
    kern::tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    // This workgroup's blocks of K: all, or one of gridDim.y parts.
    const int t0 = (int)((int64_t)p.KB * blockIdx.y / gridDim.y), t1 = (int)((int64_t)p.KB * (blockIdx.y + 1) / gridDim.y);
    const int m0 = tm * BM, n0 = tn * S::OUT;
    const int wm = wave % WM, wn = wave / WM;

    // ---- loads: a wave instruction fills 8 rows; lane → row lane / 8, run (lane mod 8) ^ key ----
    constexpr int A_LOADS = BM / 8 / WAVES, W_LOADS = BN / 8 / WAVES;
    static_assert(A_LOADS * 8 * WAVES == BM && W_LOADS * 8 * WAVES == BN, "loads spread evenly");
    const wd::i32x4 a_rsrc = wd::buffer_rsrc(p.a + (int64_t)m0 * p.lda), w_rsrc = wd::buffer_rsrc(p.w + (int64_t)n0 * p.ldw);
    uint32_t a_off[A_LOADS], w_off[W_LOADS];
    const int a_run = ((lane & 7) ^ key_a(lane >> 3)) * 16;
    auto w_run = [&](int i) { return ((lane & 7) ^ key_w<NTO>((wave * W_LOADS + i) * 8 + (lane >> 3))) * 16; };
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i)
        a_off[i] = (uint32_t)(min((wave * A_LOADS + i) * 8 + (lane >> 3), p.M - 1 - m0) * p.lda) + a_run;
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i) {
        const int row = (wave * W_LOADS + i) * 8 + (lane >> 3);
        const int half = GLU && row >= BN / 2 ? 1 : 0;
        const int64_t n = min(row - half * (BN / 2), p.H - 1 - n0) + (int64_t)half * p.H;
        w_off[i] = (uint32_t)(n * p.ldw) + w_run(i);
    }
    const int left = p.K & (F8_GROUP - 1);  // of a last block that K ends inside
    uint8_t *const scales = lds + NS * S::STAGE;
    const wd::i32x4 sx_rsrc = wd::buffer_rsrc(p.sx + (int64_t)m0 * p.ldsx);
    constexpr int LOADS = A_LOADS + W_LOADS;  // a wave's of one block, besides those of scales
    // Block t's loads into a stage: first `ahead`, then each of LOADS. Past t1 the buffers have no bytes: nothing is
    // read, but the loads under way stay as many.
    wd::i32x4 a_from = a_rsrc, w_from = w_rsrc;
    auto ahead = [&](int t) {
        int under = t - t1;
        asm volatile("" : "+s"(under));  // (a comparison's result would go through vector registers)
        a_from[2] = w_from[2] = under >> 31;
        if (t >= t1) return;
        if (left != 0 && t == p.KB - 1) {
            // Runs past K are read from the block's first: it is the last that these offsets are for.
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) a_off[i] -= a_run >= left ? a_run : 0;
#pragma unroll
            for (int i = 0; i < W_LOADS; ++i) w_off[i] -= w_run(i) >= left ? w_run(i) : 0;
        }
        if (!p.sx_vec || (t & 3) == 0 || t == t0) {
            // A lane a row; sx_vec: blocks t .. t + 3 as [row][4], else one block as [4][row].
            uint8_t *const s = scales + ((t >> 2) & 1) * S::SCALES;
            int last_row = p.M - 1 - m0;
            asm volatile("" : "+s"(last_row));
            for (int r = wave * 64; r < BM; r += 64 * WAVES) {
                const int from = (int)(min(r + lane, last_row) * (uint32_t)p.ldsx * 4);
                if (p.sx_vec) wd::raw_buffer_load_lds(sx_rsrc, (wd::lds_u32)(s + r * 16), 16, from, (t & ~3) * 4, 0, 0);
                else wd::raw_buffer_load_lds(sx_rsrc, (wd::lds_u32)(s + ((t & 3) * BM + r) * 4), 4, from, t * 4, 0, 0);
            }
        }
    };
    auto load = [&](auto nc, int t, int stage) {
        constexpr int n = decltype(nc)::value, i = n < A_LOADS ? n : n - A_LOADS;
        uint8_t *const to = lds + stage;
        if constexpr (n < A_LOADS)
            wd::raw_buffer_load_lds(a_from, (wd::lds_u32)(to + (wave * A_LOADS + i) * 1024), 16, (int)a_off[i], t * F8_GROUP, 0, 0);
        else
            wd::raw_buffer_load_lds(w_from, (wd::lds_u32)(to + BM * F8_GROUP + (wave * W_LOADS + i) * 1024), 16, (int)w_off[i], t * F8_GROUP, 0, 0);
    };
    // Block t's loads are done, this wave's and then all; those of NS − 2 later ones may be under way. The activation's
    // runs past K become zeros in between.
    auto landed = [&](int t, int stage) {
        wd::wait_vmcnt<(NS - 2) * LOADS>();
        if (left != 0 && t == p.KB - 1 && a_run >= left) {
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i)
                *reinterpret_cast<u32x4 *>(lds + stage + (wave * A_LOADS + i) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        }
        // No fence: one would wait for the later blocks' loads too. What LDS this wave still reads has come.
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    const int scale_row = p.sx_vec ? 16 : 4, scale_block = p.sx_vec ? 4 : BM * 4;

    // ---- fragment addresses: neither key depends on the part, whose rows lie at fixed distances ----
    int a_at[2], w_at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int ra = wm * (BM / WM) + c, rw = wn * (16 * NTO) + 4 * NTO * (c >> 2) + (c & 3);
        a_at[u] = ra * F8_GROUP + (((4 * u + h) ^ key_a(ra)) << 4);
        w_at[u] = BM * F8_GROUP + rw * F8_GROUP + (((4 * u + h) ^ key_w<NTO>(rw)) << 4);
    }
    const int sx_at = NS * S::STAGE + (wm * (BM / WM) + c) * scale_row;
    // A wave's outputs of one half lie in one block of 128 columns (past the last: none are stored). Lane l keeps the
    // scale of block l of each 64.
    const float *const sw0 = p.sw + (int64_t)min((n0 + wn * 16 * NTO) / F8_GROUP, p.up_block - 1) * p.ldsw;
    float sw_of[2];
    auto load_sw = [&](int t) {
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); ++g) sw_of[g] = sw0[(int64_t)g * p.up_block * p.ldsw + min(t + lane, t1 - 1)];
        wd::wait_vmcnt<0>();
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    i32x8 w[TN], a[2];
    float s_x[2], both[2][2];
    f32x4 part[TN];
    auto fragment = [&](int lo, int hi) {
        const u32x4 x = *reinterpret_cast<const u32x4 *>(lds + lo), y = *reinterpret_cast<const u32x4 *>(lds + hi);
        return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    };
    int stage = 0;  // the offset in LDS of the stage whose fragments are read, and of its scales
    auto scales_of = [&](int t) { return sx_at + (t & 3) * scale_block + ((t >> 2) & 1) * S::SCALES; };
    int sx_now = scales_of(t0);
    auto read_a = [&](auto ic) {
        constexpr int i = decltype(ic)::value;
        a[i & 1] = fragment(a_at[0] + stage + i * 16 * F8_GROUP, a_at[1] + stage + i * 16 * F8_GROUP);
        s_x[i & 1] = *reinterpret_cast<const float *>(lds + sx_now + i * 16 * scale_row);
    };
    auto read_w = [&](auto jc) {
        constexpr int j = decltype(jc)::value, from = ((j / NTO) * (BN / 2) + 4 * (j % NTO)) * F8_GROUP;
        w[j] = fragment(w_at[0] + stage + from, w_at[1] + stage + from);
    };
    auto add = [&](auto ic, auto jc) {
        constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(part[j][e], both[i & 1][j / NTO & 1], acc[i][j][e]);
        // Kept where it stands: moved down past the step's branches it would hold on to its part's registers.
        asm volatile("" : "+v"(acc[i][j][0]), "+v"(acc[i][j][1]), "+v"(acc[i][j][2]), "+v"(acc[i][j][3]));
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using Last = std::integral_constant<int, TM - 1>;
    static_assert(TM >= 2 && TM % 2 == 0, "fragments of two rows of parts in turn");

    if (t0 < t1) {
        load_sw(t0);
        static_for<0, NS>([&](auto sc) {
            constexpr int s = decltype(sc)::value;
            ahead(t0 + s);
            static_for<0, LOADS>([&](auto nc) { load(nc, t0 + s, s * S::STAGE); });
            if constexpr (s == NS - 2) landed(t0, 0);
        });
        static_for<0, TN>([&](auto jc) { read_w(jc); });
        read_a(I0{});
        read_a(I1{});
#pragma unroll
        for (int j = 0; j < TN; ++j) part[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        both[1][0] = both[1][1] = 0.0f;
    }
#pragma clang loop unroll(disable)
    for (int t = t0; t < t1; ++t) {
        float s_w[2];
        int from = 0;  // the stage that is free after this step's barrier
        if (t != t0 && ((t - t0) & 63) == 0) load_sw(t);
#pragma unroll
        for (int g = 0; g < (GLU ? 2 : 1); ++g) s_w[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sw_of[g]), (t - t0) & 63));
        static_for<0, TM>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            using Before = std::integral_constant<int, (i + TM - 1) % TM>;
            if constexpr (i == TM - 2) {
                // Every fragment of this stage is in registers (or on its way there: the barrier waits for those).
                from = stage;
                stage = stage == (NS - 1) * S::STAGE ? 0 : stage + S::STAGE;
                landed(t + 1, stage);
                ahead(t + NS);
                sx_now = scales_of(t + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < (GLU ? 2 : 1); ++g) both[i & 1][g] = s_x[i & 1] * s_w[g];
            static_for<0, TN>([&](auto jc) {
                constexpr int j = decltype(jc)::value;
                add(Before{}, jc);
                part[j] = block_sums<F32>(w[j], a[i & 1]);
                if constexpr (i >= TM - 2) {
                    constexpr int SLOT = (i - (TM - 2)) * TN + j, SLOTS = 2 * TN;
                    static_for<LOADS * SLOT / SLOTS, LOADS * (SLOT + 1) / SLOTS>([&](auto nc) { load(nc, t + NS, from); });
                }
                if constexpr (i == TM - 1) read_w(jc);
            });
            read_a(std::integral_constant<int, (i + 2) % TM>{});
            if constexpr (!F32) {
                // The multiply-adds of a part of the row before, the matrix instruction that takes its place, its reads.
                static_for<0, TN>([&](auto jc) {
                    constexpr int SLOT = (i - (TM - 2)) * TN + decltype(jc)::value, SLOTS = 2 * TN;
                    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if constexpr (SLOT >= 0) __builtin_amdgcn_sched_group_barrier(0x010, LOADS * (SLOT + 1) / SLOTS - LOADS * SLOT / SLOTS, 0);
                    if constexpr (i == TM - 1) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                });
                __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    }
    if (t0 < t1) static_for<0, TN>([&](auto jc) { add(Last{}, jc); });
    wd::wait_vmcnt<0>();  // a load's write to LDS may not outlive the workgroup

    // ---- outputs: N consecutive ones of each of TM rows ----
    constexpr int N = 4 * NTO;
    const int col = n0 + wn * 16 * NTO + N * h;
    const int real = min(N, p.H - col);  // of them
    const int row0 = m0 + wm * (BM / WM) + c;
    if constexpr (S::SPLIT) {
        if (gridDim.y > 1) {
            // One part of K. Its sums go to its slot, past the caches that workgroups do not share, and the workgroup
            // that a tile's counter finds last adds the slots up, in their order.
            const int splits = gridDim.y, mine = blockIdx.y;
            float *const slots = p.part + (int64_t)blockIdx.x * splits * (BM * BN) + 2 * threadIdx.x;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
                        put(slots + (int64_t)mine * (BM * BN) + ((i * TN + j) * 4 + e) * S::THREADS, Pair{acc[i][j][e], acc[i][j][e + 1]});
            wd::wait_vmcnt<0>();
            __syncthreads();
            int *const joins = reinterpret_cast<int *>(lds);
            if (threadIdx.x == 0) {
                int *const mark = p.marks + (int64_t)blockIdx.x * MARK;
                const bool last = __hip_atomic_fetch_add(mark, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == splits - 1;
                if (last) __hip_atomic_store(mark, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                *joins = last;
            }
            __syncthreads();
            if (!*joins) return;
            f32x4 total[TM][TN];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) total[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int k = 0; k < splits; ++k) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const Pair x = get(slots + (int64_t)k * (BM * BN) + ((i * TN + j) * 4 + e) * S::THREADS);
                            total[i][j][e] += x.a;
                            total[i][j][e + 1] += x.b;
                        }
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = total[i][j];
        }
    }
    float bias[GLU ? 2 : 1][N];
    if (p.bias) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            bias[0][e] = p.bias[min(col + e, p.H - 1)];
            if constexpr (GLU) bias[1][e] = p.bias[min(col + e, p.H - 1) + p.H];
        }
    }
    static_for<0, TM>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        float y[N];
        static_for<0, N>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            float x = acc[i][e / 4][e % 4];
            if (p.bias) x += bias[0][e];
            if constexpr (GLU) {
                float u = acc[i][NTO + e / 4][e % 4];
                if (p.bias) u += bias[1][e];
                x = silu_glu(x, u);
            }
            y[e] = x;
        });
        if (row0 + 16 * i < p.M) store_run<N, F32>(p.c, (int64_t)(row0 + 16 * i) * p.ldc + col, real, p.c_vec, y);
        __builtin_amdgcn_sched_barrier(0);
    });
}

template <int BM, int BN, int WM, int WN, int NS, bool GLU, bool F32>
hipError_t launch_tile(const F8Args &p, int splits, hipStream_t stream) {
    using S = TileShape<BM, BN, WM, WN, NS, GLU, F32>;
    const int64_t tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.H + S::OUT - 1) / S::OUT;
    if (tiles_m * tiles_n > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((f8_tile_kernel<BM, BN, WM, WN, NS, GLU, F32>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)splits),
                       dim3(S::THREADS), 0, stream, p, (int)tiles_m, (int)tiles_n);
    return hipGetLastError();
}

template <int TM, int NO, int NW, int U, bool GLU, bool F32>
hipError_t launch_short(const F8Args &p, hipStream_t stream) {
    const dim3 grid((unsigned)((p.H + 16 * NO - 1) / (16 * NO)), (unsigned)((p.M + 16 * TM - 1) / (16 * TM)));
    hipLaunchKernelGGL((f8_short_kernel<TM, NO, NW, U, GLU, F32>), grid, dim3(64 * NW), 0, stream, p);
    return hipGetLastError();
}

template <int NO, bool F32>
hipError_t launch_staged(const F8Args &p, hipStream_t stream) {
    hipLaunchKernelGGL((f8_staged_kernel<NO, 4, F8_STAGED_GROUPS, F32>), dim3((unsigned)((p.H + 16 * NO - 1) / (16 * NO))), dim3(512), 0, stream, p);
    return hipGetLastError();
}

template <bool GLU, bool F32>
hipError_t launch(const F8Args &p, const F8Plan &plan, hipStream_t stream) {
    switch (plan.kernel) {
        case F8_256: return launch_tile<256, 256, 2, 4, 2, GLU, false>(p, plan.splits, stream);
        case F8_128: return launch_tile<128, 128, 2, 2, 2, GLU, F32>(p, plan.splits, stream);
        case F8_128_ONE: return launch_tile<128, 128, 2, 4, 4, GLU, F32>(p, 1, stream);
        case F8_64x128: return launch_tile<64, 128, 2, 2, 3, GLU, F32>(p, plan.splits, stream);
        case F8_64: return launch_tile<64, 64, 2, 2, 4, GLU, F32>(p, plan.splits, stream);
        case F8_SHORT: return launch_short<1, 1, 8, 4, GLU, F32>(p, stream);
        case F8_SHORT_WIDE: return launch_short<1, 2, 8, 4, GLU, F32>(p, stream);
        default: break;  // F8_FAR
    }
    if constexpr (!GLU) {
        if (plan.kernel == F8_STAGED) return launch_staged<1, F32>(p, stream);
        if (plan.kernel == F8_STAGED_WIDE) return launch_staged<2, F32>(p, stream);
    }
    return launch_short<4, 1, 8, 2, GLU, F32>(p, stream);
}

}  // namespace

hipError_t launch_f8_product(const F8Args &p, const F8Plan &plan, bool glu, bool out_f32, hipStream_t stream) {
    if (p.M == 0 || p.H == 0) return hipSuccess;
    if (glu) return out_f32 ? launch<true, true>(p, plan, stream) : launch<true, false>(p, plan, stream);
    return out_f32 ? launch<false, true>(p, plan, stream) : launch<false, false>(p, plan, stream);
}

}  // namespace sq8
