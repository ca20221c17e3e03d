// sq8_paged.hip — a paged key-value cache: appending new keys and values with the position rotation applied, and
// attention of one new token per sequence over it.
//
// A cache is two pools [pages, page, kv_heads, dim] of bf16 or e4m3 (times a scale per head), any strides with the
// values of a head contiguous. Offsets into them are 64-bit. No index read from device memory is trusted: a slot
// outside the pools is not written, a position outside the table reads its last row, a page outside the pools
// counts as masked, a length past the page table's end is cut to it.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sq8_device.h"
#include "sq8_text.h"
#include "sq8_text_quant.h"

namespace sq8 {
namespace {

__device__ __forceinline__ float bf16_f32(uint32_t bits) { return __uint_as_float(bits << 16); }

// ---- append ------------------------------------------------------------------------------------------------------
//
// q' = rot(q), k' = rot(k): with (cos, sin) of the token's position, pair i of the first `rot` values of a head,
// (a, b) → (a·cos − b·sin, b·cos + a·sin); pairs (i, i + rot/2), or (2i, 2i + 1) when interleaved. Products and sums
// in fp32, one rounding. e4m3: code = e4m3(v / scale), saturated at ±448 (a NaN stays one).
//
// Bound by memory: every value is read once and written once. A thread takes one unit of a token: two runs of W
// values, the two halves of W pairs (or W values of one run and the next where there is nothing to turn), so a wave
// reads whole 16-byte runs on both sides (W = 8, wherever the rows lie; W = 4 where heads or their turned part are no
// multiple of 16, W = 1 where not of 8). 8192 tokens of 32 query and
// 8 key heads of 128 into a bf16 cache (206 MB) take 42.5 µs, 4.8 TB/s where a large copy runs at 5.0; 48 tokens
// into an e4m3 one 3.2 µs, 2.3 of them the launch.
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

template <int W, bool E4M3>
__global__ void __launch_bounds__(256) append_kv_kernel(const AppendArgs p) {
    const unsigned per_head = (unsigned)p.dim / (2 * W);
    const unsigned units = (unsigned)(p.q_heads + 2 * p.kv_heads) * per_head;
    const int64_t first = (int64_t)blockIdx.x * 256;  // of this workgroup's units over all tokens
    const int64_t token0 = first / units;
    const unsigned local = (unsigned)(first - token0 * units) + threadIdx.x;
    const int64_t token = token0 + local / units;
    if (token >= p.tokens) return;
    const unsigned unit = local % units;
    int head = (int)(unit / per_head);
    const int u = (int)(unit % per_head);
    const int32_t slot = p.slots[token];
    const int kind = head < p.q_heads ? 0 : head < p.q_heads + p.kv_heads ? 1 : 2;  // q, k, v
    head -= kind == 0 ? 0 : kind == 1 ? p.q_heads : p.q_heads + p.kv_heads;
    const bool live = slot >= 0 && slot < p.slot_count;
    if (kind != 0 && !live) return;
    const uint16_t *src = kind == 0   ? p.q + token * p.q_tok + head * p.q_head
                          : kind == 1 ? p.k + token * p.k_tok + head * p.k_head
                                      : p.v + token * p.v_tok + head * p.v_head;
    const int turned = p.rot / (2 * W);  // units of a head that are turned
    const bool turns = kind != 2 && u < turned;
    const int at0 = turns && !p.interleaved ? W * u : 2 * W * u;
    const int at1 = turns && !p.interleaved ? at0 + p.rot / 2 : at0 + W;
    float a[W], b[W];
    load_run<W>(src + at0, a);
    load_run<W>(src + at1, b);
    if (turns) {
        int position = p.positions[token];
        position = position < 0 || position >= p.max_position ? p.max_position - 1 : position;
        float cs[W], sn[W];
        const float *row = p.table + (int64_t)position * p.table_row + W * u;
        load_angles<W>(row, cs);
        load_angles<W>(row + p.rot / 2, sn);
        if (p.interleaved && W > 1) {
            // Pair i of the unit's 2W values is values 2i and 2i + 1: both in `a` or both in `b`.
#pragma unroll
            for (int i = 0; i < W / 2; ++i) {
                const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], t = b[2 * i + 1];
                a[2 * i] = x * cs[i] - y * sn[i];
                a[2 * i + 1] = y * cs[i] + x * sn[i];
                b[2 * i] = z * cs[W / 2 + i] - t * sn[W / 2 + i];
                b[2 * i + 1] = t * cs[W / 2 + i] + z * sn[W / 2 + i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float x = a[i], y = b[i];
                a[i] = x * cs[i] - y * sn[i];
                b[i] = y * cs[i] + x * sn[i];
            }
        }
    }
    if (kind == 0) {
        uint16_t *dst = p.q_out + token * p.qo_tok + head * p.qo_head;
        store_bf16<W>(dst + at0, a);
        store_bf16<W>(dst + at1, b);
        return;
    }
    const int64_t page = slot / p.page, in = slot - page * p.page;
    const int64_t to = kind == 1 ? page * p.kc_page + in * p.kc_tok + head * p.kc_head
                                 : page * p.vc_page + in * p.vc_tok + head * p.vc_head;
    void *pool = kind == 1 ? p.kc : p.vc;
    if constexpr (E4M3) {
        const float *scales = kind == 1 ? p.k_scale : p.v_scale;
        const Quotient by(scales ? scales[head] : 1.0f);
        uint8_t *dst = static_cast<uint8_t *>(pool) + to;
        store_e4m3<W>(dst + at0, a, by);
        store_e4m3<W>(dst + at1, b, by);
    } else {
        uint16_t *dst = static_cast<uint16_t *>(pool) + to;
        store_bf16<W>(dst + at0, a);
        store_bf16<W>(dst + at1, b);
    }
}

// ---- attention of one new token ------------------------------------------------------------------------------------
//
//   o[b, h] = Σ_t softmax_t(s_t) · v_t,  s_t = cap(scale · q·k_t),  t in [max(0, len − window), len)
//
// One pass over the cache with the running maximum and sum of the softmax, both fp32. The maximum is moved only when a
// score passes it by 8 powers of two, so a probability may be up to 2^8 of what it will be divided by: the same bits
// of it, and the sums rescaled hardly ever. For their product with v the probabilities are split into two bf16 numbers each,
// 2^-17 of one at most left out: rounded to one they would cost the output as much as its own rounding to bf16.
//
// Bound by the cache's bytes. The query heads of one kv head (up to 16; more take several passes) are the columns of
// both products, on v_mfma_f32_16x16x32_bf16:
//   S[token, head] = K · Qᵀ   (first operand: 16 tokens × 32 values)
//   O[value, head] += Vᵀ · P  (first operand: 16 values × 32 tokens)
// A lane (c = lane mod 16, h = lane / 16) ends with S of tokens 4h..4h+3 of each 16-token tile for head c, and the
// second product takes its 32 tokens in the order (4h + r of the first tile, 4h + r of the second), so a lane's eight
// probabilities are its operand as they lie: nothing crosses lanes between the products. Its V operand is those eight
// tokens' rows at values DV·c .. DV·c + DV − 1 (DV = dim / 16): one contiguous load a token, transposed within the
// lane, value DV·c + i going to instruction i. So both pools go from memory to registers in whole rows, without LDS.
//
// Work is split over tiles of 128 tokens (a wave takes 32) of every (sequence, kv head, 16 query heads), numbered in
// that order and shared out evenly (Share), whatever sequences they belong to, so ragged lengths load the card evenly and
// the host needs no lengths. A sequence's head whose tiles lie in several workgroups leaves its maximum, sum and
// unnormalised output in each one's slot, and the workgroup that finishes last, as a counter tells it, joins them in
// tile order: the result does not depend on which one that is. It also sets the counter back to zero, as every call
// finds it.
//
// With 32 query heads on 8 of 128: two sequences of 131 072 tokens in bf16 (1074 MB) take 207 to 213 µs, 5.0 to 5.2 TB/s; 48
// ragged ones of up to 8192 in e4m3 (414 MB) 96 to 97, 4.3 TB/s, of which some ten are the start (the launch, the lengths,
// the first pages and rows) and the join, and the rest runs at what 128-byte pieces a kilobyte apart come in at; one of 777
// tokens 8.9, a chain of those latencies (6.5 without a join), one of 4096 12.7 and of 16 384 25. The arithmetic is not
// felt: without it the loads alone take as long. Neither are more workgroups a CU, or the heads of a sequence going through
// the same pages at the same time. What the join costs is its slots' lines and its counters: with the values of a head's
// lanes side by side (not by the 16 columns of the products), pairs to a load and a line for each counter the
// sequence of 4096 went from 15.8 µs to 12.8, the ragged ones from 100 to 96.
//
// Pages that 16-token tiles do not fill are looked up row by row, by vector loads, which wait for the rows' loads under way:
// the 48 sequences take 101 µs in pages of 24 or 8 tokens and 105 of one (in bf16 175, where pages of 16 and 64 take 165),
// the two long ones 226 to 229.

constexpr int TILE = PAGED_TILE;
constexpr int WAVES = 4;

// Token / tokens a page, by a multiplication (page_divisor).
__device__ __forceinline__ int page_of(const PagedArgs &p, int token) {
    return (int)(((uint64_t)(uint32_t)token * p.page_mul) >> p.page_shift);
}

struct Span {
    int first, last;  // tokens [first, last), from the window's first
    int base;         // `first` rounded down to 32
    int tiles;
};

__device__ __forceinline__ Span span_of(const PagedArgs &p, int length) {
    const int64_t most = (int64_t)p.max_pages * p.page;
    Span s;
    s.last = (int)(length < 0 ? 0 : length > most ? most : length);
    s.first = p.window > 0 && s.last > p.window ? s.last - p.window : 0;
    s.base = s.first & ~31;
    s.tiles = (s.last - s.base + TILE - 1) / TILE;
    return s;
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

// The batch's tiles of one head, by 64 sequences at a time in every wave.
__device__ __forceinline__ int batch_tiles(const PagedArgs &p, int lane) {
    int total = 0;
    for (int b = 0; b < p.batch; b += 64) {
        int v = b + lane < p.batch ? span_of(p, p.lengths[b + lane]).tiles : 0;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
        total += v;
    }
    return total;
}

// The sequence that holds per-head tile number `at`, and the tiles of the sequences before it.
__device__ __forceinline__ int sequence_of(const PagedArgs &p, int at, int lane, int &before) {
    int base = 0;
    for (int b = 0; b < p.batch; b += 64) {
        const int v = b + lane < p.batch ? span_of(p, p.lengths[b + lane]).tiles : 0;
        const int upto = wave_scan(v, lane);
        const uint64_t past = __ballot(base + upto > at);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            before = base + (l > 0 ? __shfl(upto, l - 1, 64) : 0);
            return b + l;
        }
        base += __shfl(upto, 63, 64);
    }
    before = base;
    return 0;  // not reached: `at` is under the batch's tiles
}

// The larger (the sum) of a value over the four lanes of a head (16 apart): the swaps leave each row's neighbour's, and
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

// The results of workgroups g0 .. g1 over one sequence's head, in that order: the first's in slot `slot0`, the others' in
// 2g (where a workgroup's tiles begin with that sequence's). A thread takes two values of a query head, side by side in
// every slot as its neighbours' are; its loads of up to 16 slots are under way at once.
template <int DP>
__device__ __forceinline__ void join_slots(const PagedArgs &p, int slot0, int g0, int g1, int live, float v_scale, uint16_t *out) {
    constexpr int DV = DP / 16, ROUND = 16;
    auto slot_of = [&](int g) { return p.part + (int64_t)(g == g0 ? slot0 : 2 * g) * paged_part_floats(DP); };
    // An item a thread: head c, row h of the lanes and register r, values d and d + 1.
    for (int i = threadIdx.x; i < live * 8 * DV; i += 64 * WAVES) {
        const int rest = i / live, c = i - rest * live;
        const int h = rest & 3, r = rest >> 2 & 3, d = 2 * (rest >> 4), at = DV * (4 * h + r) + d;
        if (at >= p.dim) continue;
        float top = -INFINITY, l = 0.0f, x = 0.0f, y = 0.0f;
        for (int g = g0; g <= g1; g += ROUND) {
            Pair s[ROUND], v[ROUND];
            float most = top;
            static_for<0, ROUND / 8>([&](auto qc) {
                constexpr int q = 8 * decltype(qc)::value;
                if (g + q > g1) return;
#pragma unroll
                for (int e = q; e < q + 8; ++e) {
                    const float *slot = slot_of(min(g + e, g1));
                    s[e] = get(slot + 2 * c);
                    v[e] = get(slot + 32 + 2 * i);
                }
            });
            static_for<0, ROUND / 8>([&](auto qc) {
                constexpr int q = 8 * decltype(qc)::value;
                if (g + q > g1) return;
#pragma unroll
                for (int e = q; e < q + 8; ++e) most = fmaxf(most, s[e].a);
            });
            const float from = most == -INFINITY ? 0.0f : most;
            const float keep = __builtin_amdgcn_exp2f(top - from);
            top = most;
            l *= keep;
            x *= keep;
            y *= keep;
            static_for<0, ROUND>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                if (g + e > g1) return;
                const float weight = __builtin_amdgcn_exp2f(s[e].a - from);
                l = __builtin_fmaf(s[e].b, weight, l);
                x = __builtin_fmaf(v[e].a, weight, x);
                y = __builtin_fmaf(v[e].b, weight, y);
            });
        }
        const float scale = inverse(l) * v_scale;
        *reinterpret_cast<uint32_t *>(out + c * p.o_head + at) = pack_bf16_rne(x * scale, y * scale);
    }
}

template <int DP, bool E4M3, bool PAGE16>
__global__ void __launch_bounds__(64 * WAVES, paged_held(DP)) paged_attention_kernel(const PagedArgs p) {
    constexpr int ES = E4M3 ? 1 : 2;
    constexpr int STEPS = DP / 32;                // MFMAs of a 16-token tile's scores
    constexpr int KRUNS = DP * ES / 64;           // 16-byte runs of a key a lane reads
    constexpr int DV = DP / 16;                   // values of a token a lane reads: MFMAs of the second product
    constexpr int VN = DV * ES / 4;               // and their dwords
    constexpr float LOG2E = 1.4426950408889634f;
    __shared__ __attribute__((aligned(16))) f32x4 joined[WAVES - 1][DV][64];
    __shared__ float tops[WAVES][16], totals[WAVES][16];
    __shared__ int joins[2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, h = lane >> 4;
    const int group = p.q_heads / p.kv_heads;
    const int passes = (group + 15) / 16;
    const int heads = p.kv_heads * passes;
    const bool full = p.dim == DP;
    const bool capped = p.softcap > 0.0f;
    // The bytes of a row a lane reads (past `dim`, the row's first), and PAGE16: with its row's place from the 16-token
    // tile's first.
    uint32_t k_run[KRUNS], k_lane[KRUNS], v_lane[4];
#pragma unroll
    for (int s = 0; s < KRUNS; ++s) {
        const int d = E4M3 ? 64 * s + 16 * h : 32 * s + 8 * h;
        k_run[s] = d < p.dim ? d * ES : 0;
        k_lane[s] = (uint32_t)(c * p.kc_tok * ES) + k_run[s];
    }
    const uint32_t v_run = DV * c < p.dim ? DV * c * ES : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v_lane[i] = (uint32_t)((4 * h + i) * p.vc_tok * ES) + v_run;

    // This workgroup's tiles, and the sequence they begin in; all uniform. Up to 64 sequences lie in a wave's lanes at once.
    int total, before = 0, b = 0, length;
    Share share;
    int start, end;
    auto mine = [&](int per_head) {
        total = __builtin_amdgcn_readfirstlane(per_head) * heads;
        share = Share(total, gridDim.x);
        start = share.first(min((int)blockIdx.x, share.groups));
        end = share.first(min((int)blockIdx.x + 1, share.groups));
    };
    if (p.batch <= 64) {
        const int n = lane < p.batch ? p.lengths[lane] : 0;
        const int v = span_of(p, n).tiles;
        const int upto = wave_scan(v, lane);
        mine(__builtin_amdgcn_readlane(upto, 63));
        const uint64_t past = __ballot(upto > start / heads);
        b = past ? __ffsll((unsigned long long)past) - 1 : 0;
        before = __builtin_amdgcn_readlane(upto - v, b);
        length = __builtin_amdgcn_readlane(n, b);
    } else {
        mine(batch_tiles(p, lane));
        if (start < end) b = __builtin_amdgcn_readfirstlane(sequence_of(p, start / heads, lane, before));
        length = p.lengths[b];
    }
    // Tiles are numbered sequence by sequence, `heads` runs of a sequence's tiles each.
    Span span = span_of(p, __builtin_amdgcn_readfirstlane(length));
    int seq0 = __builtin_amdgcn_readfirstlane(before) * heads;  // the sequence's first tile

    struct Part {
        int b, head, first, tiles;  // tiles 0: none
    } parts[2] = {};
    for (int pos = start; pos < end;) {
        while (pos >= seq0 + span.tiles * heads) {
            seq0 += span.tiles * heads;
            ++b;
            span = span_of(p, __builtin_amdgcn_readfirstlane(p.lengths[b]));
        }
        const int in_seq = pos - seq0;
        const int head = in_seq / span.tiles;
        const int tile0 = in_seq - head * span.tiles;
        const int run = min(span.tiles - tile0, end - pos);
        const int kvh = head / passes, pass = head - kvh * passes;
        const int q0 = kvh * group + pass * 16;
        const int live = min(16, group - pass * 16);  // query heads of this pass

        // ---- the queries: head c's values in the order the keys' lanes hold them ----
        bf16x8 q[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int d = E4M3 ? 64 * (s >> 1) + 16 * h + 8 * (s & 1) : 32 * s + 8 * h;
            u32x4 v = {0, 0, 0, 0};
            if (c < live && d < p.dim) v = *reinterpret_cast<const u32x4 *>(p.q + b * p.q_tok + (q0 + c) * p.q_head + d);
            q[s] = __builtin_bit_cast(bf16x8, v);
        }
        // Scores in units of log2, or where they are capped, in those of the cap.
        const float score_scale = p.scale * (E4M3 && p.k_scale ? p.k_scale[kvh] : 1.0f) * (capped ? 1.0f / p.softcap : LOG2E);
        const uint8_t *kbase = p.kc + (int64_t)kvh * p.kc_head * ES;
        const uint8_t *vbase = p.vc + (int64_t)kvh * p.vc_head * ES;
        // Read as constant memory: scalar loads, for which the vector loads under way need not be waited for.
        const auto pages = (const __attribute__((address_space(4))) int32_t *)(p.pages + (int64_t)b * p.pages_row);

        // The rows of a subtile's 32 tokens. PAGE16: each 16-token tile lies in one page, whose index is uniform and read
        // one subtile before its use. Else each lane looks up its own rows.
        struct Where {
            int id[2], in[2];                              // PAGE16: the page's index as read, and the first row in it
            int64_t k[PAGE16 ? 1 : 2], v[PAGE16 ? 1 : 8];  // else the rows' offsets in elements
            uint32_t bad;                                  // and tokens on a page outside the pools (in the order of the lane's eight)
        };
        auto locate = [&](int token) {
            Where w;
            w.bad = 0;
            if constexpr (PAGE16) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int at = min(token + 16 * t, (span.last - 1) & ~15);
                    const int page = page_of(p, at);
                    w.in[t] = at - page * p.page;
                    w.id[t] = pages[page];
                }
            } else {
                auto row = [&](int t, int64_t page_stride, int64_t tok_stride, bool &bad) {
                    const int at = min(t, span.last - 1);
                    const int page = page_of(p, at), in = at - page * p.page;
                    int id = pages[page];
                    bad = (unsigned)id >= (unsigned)p.page_count;
                    if (bad) id = 0;
                    return id * page_stride + in * tok_stride;
                };
                bool bad;
#pragma unroll
                for (int t = 0; t < 2; ++t) w.k[t] = row(token + 16 * t + c, p.kc_page, p.kc_tok, bad);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    w.v[i] = row(token + 16 * (i >> 2) + 4 * h + (i & 3), p.vc_page, p.vc_tok, bad);
                    w.bad |= bad ? 1u << i : 0u;
                }
            }
            return w;
        };
        auto inside = [&](int id) { return (unsigned)id < (unsigned)p.page_count; };
        auto bad_of = [&](const Where &w) {
            return PAGE16 ? (inside(w.id[0]) ? 0u : 0x0Fu) | (inside(w.id[1]) ? 0u : 0xF0u) : w.bad;
        };
        Raw<4> k[2][KRUNS];
        auto load_k = [&](const Where &w) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint8_t *row = PAGE16 ? kbase + ((inside(w.id[t]) ? w.id[t] : 0) * p.kc_page + w.in[t] * p.kc_tok) * ES
                                            : kbase + w.k[PAGE16 ? 0 : t] * ES;
#pragma unroll
                for (int s = 0; s < KRUNS; ++s) k[t][s] = load_raw<4>(row + (PAGE16 ? k_lane[s] : k_run[s]));
            }
        };
        Raw<VN> v[8];
        auto load_v = [&](const Where &w) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = i >> 2;
                v[i] = load_raw<VN>(PAGE16 ? vbase + ((inside(w.id[t]) ? w.id[t] : 0) * p.vc_page + w.in[t] * p.vc_tok) * ES + v_lane[i & 3]
                                           : vbase + w.v[PAGE16 ? 0 : i] * ES + v_run);
            }
        };

        float top = -INFINITY, sum = 0.0f;  // of head c, in units of log2: the sum over this lane's tokens
        f32x4 o[DV];
#pragma unroll
        for (int i = 0; i < DV; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

        int token = span.base + tile0 * TILE + wave * 32;
        Where at = locate(token);
        load_k(at);
        load_v(at);
        Where next = locate(token + TILE);
        // One subtile, and the loads of the next: the keys' once the scores are done with this one's, the values' after the
        // second product. A run's last one loads nothing (a copy of its own, so that the waits of the others are for
        // what they use).
        auto subtile = [&](auto last) {
            constexpr bool more = !decltype(last)::value;
            f32x4 s[2] = {};
            if (!full) {
                // Keys past `dim`, which were read from the row's first values, are zeros (such values give no output).
#pragma unroll
                for (int j = 0; j < KRUNS; ++j)
                    if ((E4M3 ? 64 * j + 16 * h : 32 * j + 8 * h) >= p.dim) k[0][j] = k[1][j] = Raw<4>{{0, 0, 0, 0}};
            }
#pragma unroll
            for (int j = 0; j < STEPS; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    bf16x8 kk;
                    if constexpr (E4M3) {
                        const uint32_t d0 = k[t][j >> 1].d[2 * (j & 1)], d1 = k[t][j >> 1].d[2 * (j & 1) + 1];
                        kk = __builtin_bit_cast(bf16x8, u32x4{bf16_of_e4m3<0>(d0), bf16_of_e4m3<1>(d0), bf16_of_e4m3<0>(d1),
                                                              bf16_of_e4m3<1>(d1)});
                    } else {
                        kk = __builtin_bit_cast(bf16x8, k[t][j]);
                    }
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[j], s[t], 0, 0, 0);
                }
            if (more) load_k(next);
            const uint32_t bad = bad_of(at);
            const Where later = more ? locate(token + 2 * TILE) : at;

            // Tokens 16t + 4h + r.
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = s[j >> 2][j & 3] * score_scale;
            if (capped) {
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = p.softcap * LOG2E * tanh_rel(e[j]);
            }
            const bool edge = token < span.first || token + 32 > span.last;
            if (edge || (PAGE16 ? bad != 0 : __any(bad != 0))) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = token + 16 * (j >> 2) + 4 * h + (j & 3);
                    const bool dead = t < span.first || t >= span.last || (bad >> j & 1);
                    e[j] = dead ? -INFINITY : e[j];
                    // A masked row may hold anything, and 0 · NaN is one.
#pragma unroll
                    for (int d = 0; d < VN; ++d) v[j].d[d] = dead ? 0 : v[j].d[d];
                }
            }
            float m = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
            if (__any(m > top + 8.0f)) {
                m = fmaxf(over_rows<false>(m), top);
                const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - m);
                top = m;
                sum *= keep;
#pragma unroll
                for (int d = 0; d < DV; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] *= keep;
            }
            const float from = top == -INFINITY ? 0.0f : top;
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(e[j] - from);
            sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            // Each probability in two bf16 parts: its first 8 bits, and what they leave, rounded, at least 2^-126, so that an
            // infinite value meets no zero and no other sign.
            u32x4 part[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t x = __float_as_uint(w[2 * j]), y = __float_as_uint(w[2 * j + 1]);
                part[0][j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                part[1][j] = pack_bf16_rne(fmaxf(w[2 * j] - __uint_as_float(x & 0xFFFF0000u), 0x1p-126f),
                                           fmaxf(w[2 * j + 1] - __uint_as_float(y & 0xFFFF0000u), 0x1p-126f));
            }
            const bf16x8 prob[2] = {__builtin_bit_cast(bf16x8, part[0]), __builtin_bit_cast(bf16x8, part[1])};
            // Value DV·c + d of the lane's eight tokens, two tokens a dword, two values at a time.
#pragma unroll
            for (int d = 0; d < DV; d += 2) {
                u32x4 t[2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (E4M3) {
                        // bytes (x[d], y[d], x[d + 1], y[d + 1]), then as bf16
                        const uint32_t four = __builtin_amdgcn_perm(v[2 * j + 1].d[d >> 2], v[2 * j].d[d >> 2], d & 2 ? 0x07030602u : 0x05010400u);
                        t[0][j] = bf16_of_e4m3<0>(four);
                        t[1][j] = bf16_of_e4m3<1>(four);
                    } else {
                        const uint32_t x = v[2 * j].d[d >> 1], y = v[2 * j + 1].d[d >> 1];
                        t[0][j] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                        t[1][j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 1; j >= 0; --j)
                        o[d + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t[i]), prob[j], o[d + i], 0, 0, 0);
            }
            if (more) load_v(next);
            at = next;
            next = later;
            token += TILE;
        };
        for (int i = 1; i < run; ++i) subtile(std::false_type{});
        subtile(std::true_type{});

        // ---- the waves' results joined, by the first ----
        sum = over_rows<true>(sum);
        __syncthreads();  // the run before has been read
        if (h == 0) { tops[wave][c] = top; totals[wave][c] = sum; }
        if (wave > 0) {
#pragma unroll
            for (int d = 0; d < DV; ++d) joined[wave - 1][d][lane] = o[d];
        }
        __syncthreads();
        if (wave == 0) {
            float all = top;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) all = fmaxf(all, tops[w][c]);
            const float from = all == -INFINITY ? 0.0f : all;
            float weight = __builtin_amdgcn_exp2f(top - from);
            float l = sum * weight;
#pragma unroll
            for (int d = 0; d < DV; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][r] *= weight;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                weight = __builtin_amdgcn_exp2f(tops[w][c] - from);
                l += totals[w][c] * weight;
#pragma unroll
                for (int d = 0; d < DV; ++d) {
                    const f32x4 t = joined[w - 1][d][lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] = __builtin_fmaf(t[r], weight, o[d][r]);
                }
            }
            if (c < live) {
                if (run == span.tiles) {
                    const float scale = inverse(l) * (E4M3 && p.v_scale ? p.v_scale[kvh] : 1.0f);
                    uint16_t *dst = p.out + b * p.o_tok + (q0 + c) * p.o_head;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at = DV * (4 * h + r);
                        if (at >= p.dim) continue;
#pragma unroll
                        for (int d = 0; d < DV; d += 2)
                            *reinterpret_cast<uint32_t *>(dst + at + d) = pack_bf16_rne(o[d][r] * scale, o[d + 1][r] * scale);
                    }
                } else {
                    float *slot = p.part + (int64_t)(2 * blockIdx.x + (pos == start ? 0 : 1)) * paged_part_floats(DP);
                    if (h == 0) put(slot + 2 * c, Pair{all, l});
#pragma unroll
                    for (int d = 0; d < DV; d += 2)
#pragma unroll
                        for (int r = 0; r < 4; ++r) put(slot + 32 + 2 * (((2 * d + r) * 4 + h) * live + c), Pair{o[d][r], o[d + 1][r]});
                }
            }
        }
        // A part of a sequence's head: at most the first and the last of a workgroup's runs are.
        if (run != span.tiles) {
            Part &part = pos == start ? parts[0] : parts[1];
            part.b = b;
            part.head = head;
            part.first = seq0 + head * span.tiles;
            part.tiles = span.tiles;
        }
        pos += run;
    }

    // Sequences without a token: zeros.
    for (int i = blockIdx.x; i < p.batch; i += gridDim.x) {
        if (span_of(p, p.lengths[i]).tiles != 0) continue;
        for (int j = threadIdx.x; j < p.q_heads * p.dim; j += 64 * WAVES)
            p.out[i * p.o_tok + (j / p.dim) * p.o_head + j % p.dim] = 0;
    }

    // The parts' slots are written (by the first wave) before their counters say so; the last to count joins.
    if (parts[0].tiles == 0 && parts[1].tiles == 0) return;
    if (wave == 0) __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x < 2) {
        const Part part = threadIdx.x == 0 ? parts[0] : parts[1];
        bool last = false;
        if (part.tiles != 0) {
            int *const mark = p.marks + ((int64_t)part.b * heads + part.head) * MARK;
            const int others = share.of(part.first + part.tiles - 1) - share.of(part.first);
            last = __hip_atomic_fetch_add(mark, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == others;
            if (last) __hip_atomic_store(mark, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        joins[threadIdx.x] = last;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!joins[i]) continue;
        const Part part = parts[i];
        const int g0 = share.of(part.first), g1 = share.of(part.first + part.tiles - 1);
        const int kvh = part.head / passes, pass = part.head - kvh * passes;
        join_slots<DP>(p, 2 * g0 + (share.first(g0) < part.first ? 1 : 0), g0, g1, min(16, group - pass * 16),
                       E4M3 && p.v_scale ? p.v_scale[kvh] : 1.0f, p.out + part.b * p.o_tok + (kvh * group + pass * 16) * p.o_head);
    }
}

__global__ void __launch_bounds__(256) zero_marks_kernel(int *marks, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) marks[i] = 0;
}

// Whether 16-token tiles lie in one page each, and a lane's offsets within one in 32 bits.
bool by_pages(const PagedArgs &p) { return p.page % 16 == 0 && 32 * std::max(p.kc_tok, p.vc_tok) <= INT32_MAX; }

template <int DP, bool E4M3>
hipError_t launch_attention(const PagedArgs &p, int groups, hipStream_t stream) {
    if (by_pages(p))
        hipLaunchKernelGGL((paged_attention_kernel<DP, E4M3, true>), dim3(groups), dim3(64 * WAVES), 0, stream, p);
    else
        hipLaunchKernelGGL((paged_attention_kernel<DP, E4M3, false>), dim3(groups), dim3(64 * WAVES), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_append_kv(const AppendArgs &p, bool e4m3, hipStream_t stream) {
    if (p.tokens == 0) return hipSuccess;
    const int run = (p.dim | p.rot) % 16 == 0 ? 8 : (p.dim | p.rot) % 8 == 0 ? 4 : 1;
    const int64_t units = (int64_t)(p.q_heads + 2 * p.kv_heads) * (p.dim / (2 * run)) * p.tokens;
    const int64_t blocks = (units + 255) / 256;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks);
    if (e4m3 && run == 8) hipLaunchKernelGGL((append_kv_kernel<8, true>), grid, dim3(256), 0, stream, p);
    else if (e4m3 && run == 4) hipLaunchKernelGGL((append_kv_kernel<4, true>), grid, dim3(256), 0, stream, p);
    else if (e4m3) hipLaunchKernelGGL((append_kv_kernel<1, true>), grid, dim3(256), 0, stream, p);
    else if (run == 8) hipLaunchKernelGGL((append_kv_kernel<8, false>), grid, dim3(256), 0, stream, p);
    else if (run == 4) hipLaunchKernelGGL((append_kv_kernel<4, false>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((append_kv_kernel<1, false>), grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_zero_marks(int *marks, int64_t count, hipStream_t stream) {
    const int64_t blocks = (count + 255) / 256;
    hipLaunchKernelGGL(zero_marks_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, marks, count);
    return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedArgs &p, bool e4m3, int groups, hipStream_t stream) {
    if (p.batch == 0) return hipSuccess;
    switch (paged_dim(p.dim)) {
        case 64: return e4m3 ? launch_attention<64, true>(p, groups, stream) : launch_attention<64, false>(p, groups, stream);
        case 128: return e4m3 ? launch_attention<128, true>(p, groups, stream) : launch_attention<128, false>(p, groups, stream);
        default: return e4m3 ? launch_attention<256, true>(p, groups, stream) : launch_attention<256, false>(p, groups, stream);
    }
}

}  // namespace sq8
