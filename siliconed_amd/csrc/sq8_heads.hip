// sq8_heads.hip — the norm of every query and key head and the position rotation in one pass, into a paged cache or beside
// the heads (include/siliconed_q8.h: sq8_norm_append_kv, sq8_norm_rotate).
//
//   y = x / sqrt(mean x² + eps) · w over a head's values (none where w is null), then pairs (a, b) of its first `rot` values
//   turned: (a·cos − b·sin, b·cos + a·sin); one rounding, of the turned value (e4m3: of it over the head's scale).
//
// All in fp32. A head's units of two runs of W values (the halves of W pairs) lie in as many consecutive lanes, a power of
// two of them, so the sum of squares crosses lanes by a few exchanges and everything is read and written once.
//
// Bound by memory: 8192 tokens of 32 and 8 heads of 128 into an e4m3 cache (189 MB with v) take 36.4 µs alone and 44 in turns
// with other tensors (5.2 and 4.3 TB/s; a copy runs at 4.9); 4608 tokens of 24 and 24 beside the heads (116 MB) 26 and 31. One
// token 2.9 to 3.5 µs, a launch.
#include <hip/hip_runtime.h>

#include "sq8_device.h"
#include "sq8_text.h"
#include "sq8_text_device.h"

namespace sq8 {
namespace {

enum { BESIDE = 0, CACHE_BF16, CACHE_E4M3 };

// The sum over 2^log consecutive lanes.
__device__ __forceinline__ float sum_of_lanes(float v, int log) {
    for (int i = 0; i < log; ++i) v += __shfl_xor(v, 1 << i, 64);
    return v;
}

template <int W, int DEST>
__global__ void __launch_bounds__(256) norm_heads_kernel(const HeadsArgs p) {
    constexpr int U = W == 1 ? 4 : 1;  // units of a lane: heads of up to 512
    const int units = p.dim / (2 * W), mask = (1 << p.lanes_log) - 1;
    const int per_group = 256 >> p.lanes_log;  // heads of a workgroup
    const int heads = p.q_heads + (DEST == BESIDE ? 1 : 2) * p.kv_heads;
    const int64_t first = (int64_t)blockIdx.x * per_group;  // of this workgroup's heads over all tokens
    const int64_t token0 = first / heads;
    const unsigned local = (unsigned)(first - token0 * heads) + (threadIdx.x >> p.lanes_log);
    const int64_t token = token0 + local / (unsigned)heads;
    if (token >= p.tokens) return;
    int head = (int)(local % (unsigned)heads);
    const int kind = head < p.q_heads ? 0 : head < p.q_heads + p.kv_heads ? 1 : 2;  // q, k, v
    head -= kind == 0 ? 0 : kind == 1 ? p.q_heads : p.q_heads + p.kv_heads;
    int64_t slot = 0;
    if (DEST != BESIDE && kind != 0) {
        slot = p.slots[token];
        if (slot < 0 || slot >= p.slot_count) return;  // (all of a head's lanes)
    }
    const uint16_t *const src = kind == 0   ? p.q + token * p.q_tok + head * p.q_head
                                : kind == 1 ? p.k + token * p.k_tok + head * p.k_head
                                            : p.v + token * p.v_tok + head * p.v_head;
    const int turned = kind == 2 ? 0 : p.rot / (2 * W);  // units of a head that are turned
    float a[U][W], b[U][W];
    int at0[U], at1[U];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = (threadIdx.x & mask) + (i << p.lanes_log);
        const bool halves = u < turned && !p.interleaved;
        at0[i] = u >= units ? -1 : halves ? W * u : 2 * W * u;
        at1[i] = halves ? at0[i] + p.rot / 2 : at0[i] + W;
        if (at0[i] < 0) continue;
        load_run<W>(src + at0[i], a[i]);
        load_run<W>(src + at1[i], b[i]);
#pragma unroll
        for (int e = 0; e < W; ++e) ss += a[i][e] * a[i][e] + b[i][e] * b[i][e];
    }
    const float *const w = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
    if (w) {
        ss = sum_of_lanes(ss, p.lanes_log);
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)p.dim) + p.eps));
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (at0[i] < 0) continue;
            float x[W], y[W];
            load_angles<W>(w + at0[i], x);
            load_angles<W>(w + at1[i], y);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                a[i][e] = a[i][e] * r * x[e];
                b[i][e] = b[i][e] * r * y[e];
            }
        }
    }
    if (turned > 0) {
        int position = p.positions[token];
        position = position < 0 || position >= p.max_position ? p.max_position - 1 : position;
        const float *const row = p.table + (int64_t)position * p.table_row;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = (threadIdx.x & mask) + (i << p.lanes_log);
            if (u >= turned) continue;
            float cs[W], sn[W];
            load_angles<W>(row + W * u, cs);
            load_angles<W>(row + W * u + p.rot / 2, sn);
            if (p.interleaved && W > 1) {
                // Pair j of the unit's 2W values is values 2j and 2j + 1: both in `a` or both in `b`.
#pragma unroll
                for (int j = 0; j < W / 2; ++j) {
                    const float x = a[i][2 * j], y = a[i][2 * j + 1], z = b[i][2 * j], t = b[i][2 * j + 1];
                    a[i][2 * j] = x * cs[j] - y * sn[j];
                    a[i][2 * j + 1] = y * cs[j] + x * sn[j];
                    b[i][2 * j] = z * cs[W / 2 + j] - t * sn[W / 2 + j];
                    b[i][2 * j + 1] = t * cs[W / 2 + j] + z * sn[W / 2 + j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float x = a[i][j], y = b[i][j];
                    a[i][j] = x * cs[j] - y * sn[j];
                    b[i][j] = y * cs[j] + x * sn[j];
                }
            }
        }
    }
    if (kind == 0 || DEST == BESIDE) {
        uint16_t *const dst = kind == 0 ? p.q_out + token * p.qo_tok + head * p.qo_head : p.k_out + token * p.ko_tok + head * p.ko_head;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (at0[i] < 0) continue;
            store_bf16<W>(dst + at0[i], a[i]);
            store_bf16<W>(dst + at1[i], b[i]);
        }
        return;
    }
    const int64_t page = slot / p.page, in = slot - page * p.page;
    const int64_t to = kind == 1 ? page * p.kc_page + in * p.kc_tok + head * p.kc_head : page * p.vc_page + in * p.vc_tok + head * p.vc_head;
    void *const pool = kind == 1 ? p.kc : p.vc;
    const float *const scales = kind == 1 ? p.k_scale : p.v_scale;
    const Quotient by(DEST == CACHE_E4M3 && scales ? scales[head] : 1.0f);
#pragma unroll
    for (int i = 0; i < U; ++i) {
        if (at0[i] < 0) continue;
        if constexpr (DEST == CACHE_E4M3) {
            uint8_t *const dst = static_cast<uint8_t *>(pool) + to;
            store_e4m3<W>(dst + at0[i], a[i], by);
            store_e4m3<W>(dst + at1[i], b[i], by);
        } else {
            uint16_t *const dst = static_cast<uint16_t *>(pool) + to;
            store_bf16<W>(dst + at0[i], a[i]);
            store_bf16<W>(dst + at1[i], b[i]);
        }
    }
}

template <int W>
hipError_t launch_heads(const HeadsArgs &p, int dest, unsigned blocks, hipStream_t stream) {
    const dim3 grid(blocks), block(256);
    if (dest == BESIDE) hipLaunchKernelGGL((norm_heads_kernel<W, BESIDE>), grid, block, 0, stream, p);
    else if (dest == CACHE_BF16) hipLaunchKernelGGL((norm_heads_kernel<W, CACHE_BF16>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((norm_heads_kernel<W, CACHE_E4M3>), grid, block, 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_norm_heads(HeadsArgs p, bool e4m3, hipStream_t stream) {
    if (p.tokens == 0) return hipSuccess;
    const int run = (p.dim | p.rot) % 16 == 0 ? 8 : (p.dim | p.rot) % 8 == 0 ? 4 : 1;
    p.lanes_log = 0;
    while (p.lanes_log < 6 && (1 << p.lanes_log) < p.dim / (2 * run)) ++p.lanes_log;
    const int64_t each = (int64_t)p.q_heads + (int64_t)(p.kc ? 2 : 1) * p.kv_heads;
    if (each > INT32_MAX) return hipErrorInvalidValue;  // a token's heads are counted in 32 bits
    const int64_t heads = each * p.tokens, per_group = 256 >> p.lanes_log;
    const int64_t blocks = (heads + per_group - 1) / per_group;
    if (blocks > kMostThreads / 256) return hipErrorInvalidValue;
    const int dest = !p.kc ? BESIDE : e4m3 ? CACHE_E4M3 : CACHE_BF16;
    return run == 8   ? launch_heads<8>(p, dest, (unsigned)blocks, stream)
           : run == 4 ? launch_heads<4>(p, dest, (unsigned)blocks, stream)
                      : launch_heads<1>(p, dest, (unsigned)blocks, stream);
}

}  // namespace sq8
