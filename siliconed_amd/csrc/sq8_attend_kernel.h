// sq8_attend_kernel.h — attention of many tokens of a sequence at once: whole prompts over their own keys and values, or
// chunks of new tokens over a paged cache.
//
//   o[i, h] = Σ_t softmax_t(s_t) · v_t,  s_t = cap(scale · q_i·k_t),  t in [max(0, at_i − window + 1), at_i]
//
// with at_i the token's place in its sequence (without the causal mask: every t). The rows of a tile are (token, query head)
// pairs of one kv head, the head's number running fastest, so the group's heads share each key and value that is read.
//
// One pass over the keys with the running maximum and sum of the softmax, both fp32; the maximum is moved only when a score
// passes it by 8 powers of two. Per 32 rows and 32 tokens, on v_mfma_f32_32x32x16_bf16:
//   S[token, row] = K · Qᵀ        (first operand: 32 tokens × 16 values, from LDS)
//   O[value, row] += Vᵀ · P       (first operand: 32 values × 16 tokens, from LDS, transposed as it is read)
// A lane (column c = lane mod 32, half h = lane / 32) ends with S of one row and half the tokens (8·(r / 4) + 4h + r mod 4 in
// register r), and the second product takes its tokens in that order, so the probabilities are its operand as they lie and a
// row's maximum and sum cross only two lanes.
//
// A workgroup has WM · WT waves: WM sets of 32 rows, and WT waves that share a tile's tokens and are joined at the end. Tiles
// of keys and values go to LDS in two stages, the next tile's loads under way while one is used, in runs of 16 bytes whose
// places are turned by the row's number, so that neither reads nor transposed reads meet in a bank.
#pragma once

#include <hip/hip_runtime.h>

#include "sq8_device.h"
#include "sq8_text.h"
#include "sq8_text_device.h"
#include "sq8_wdirect_kernel.h"

namespace sq8 {
namespace attend {

typedef short i16x4 __attribute__((__vector_size__(8)));
typedef __attribute__((address_space(3))) i16x4 *lds_i16x4;

template <int DP, int WM, int WT, int SRC>
struct Shape {
    static constexpr int WAVES = WM * WT, THREADS = 64 * WAVES;
    static constexpr int M = 32 * WM;                                 // rows of a tile
    static constexpr int TT = attend_tokens(DP, WM, WT);              // tokens of a tile
    static constexpr int SUB = TT / (32 * WT);                        // 32-token parts a wave takes of it
    static constexpr int ROW = 2 * DP;                                // bytes of a token in LDS
    static constexpr int RUNS = DP / 8;                               // and its 16-byte runs
    static constexpr int MATRIX = TT * ROW, STAGE = 2 * MATRIX;
    static constexpr bool F8 = SRC == PAGES16_F8 || SRC == PAGES_F8;
    static constexpr bool PAGED = SRC != ROWS, EACH = SRC == PAGES || SRC == PAGES_F8;  // EACH: rows are looked up one by one
    static constexpr int PER_LOAD = F8 ? 1024 / DP : 1024 / ROW;      // tokens a wave's load instruction fills
    static constexpr int LOADS = TT / PER_LOAD / WAVES;               // a wave's of either matrix
    static constexpr int MINE = TT / WAVES;                           // tokens a wave loads
    static constexpr int LANES = 64 / PER_LOAD;                       // lanes to a token
    static constexpr int IDS = TT / 16;
    static_assert(SUB >= 1 && SUB * 32 * WT == TT && LOADS >= 1 && LOADS * PER_LOAD * WAVES == TT, "whole parts");
    static_assert(MINE <= 16 || MINE % 16 == 0, "a load's tokens lie in one sixteen");
};

__device__ __forceinline__ int key_k(int row) { return row & 7; }
__device__ __forceinline__ int key_v(int row) { return 2 * (row & 3); }

// A value's maximum (sum) over the two lanes of a row.
template <bool SUM>
__device__ __forceinline__ float over_halves(float v) {
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    return SUM ? a + b : fmaxf(a, b);
}

// Whether either bf16 of a pair is an infinity or a NaN.
__device__ __forceinline__ bool unbounded(uint32_t d) {
    return (d & 0x7F80u) == 0x7F80u || (d & 0x7F800000u) == 0x7F800000u;
}

// A sequence's rows of q and the tokens it holds.
struct Sequence {
    int row0, count, held;
};
__device__ __forceinline__ Sequence sequence(const AttendArgs &p, int b) {
    Sequence s;
    if (!p.starts) {
        s.row0 = 0;
        s.count = p.tokens;
    } else {
        const int lo = min(max(p.starts[b], 0), p.tokens), hi = min(max(p.starts[b + 1], lo), p.tokens);
        s.row0 = lo;
        s.count = hi - lo;
    }
    s.held = s.count;
    if (p.lengths) {
        const int64_t most = (int64_t)p.max_pages * p.page;
        const int n = p.lengths[b];
        s.held = (int)(n < 0 ? 0 : n > most ? most : n);
    }
    return s;
}

// Units of a sequence: a tile of rows by a kv head, the head running fastest. Shared out (p.share), each has as many tiles of
// keys as the sequence's longest.
struct Units {
    int tiles;   // of rows
    int run;     // tiles of keys of a unit that are numbered: 1 unless shared
};
template <int M, int TT>
__device__ __forceinline__ Units units_of(const AttendArgs &p, const Sequence &s) {
    Units u;
    u.tiles = (int)(((int64_t)s.count * p.group + M - 1) / M);
    int base = 0;
    if (p.causal && p.window > 0) base = max(0, s.held - s.count - p.window + 1) & ~15;
    u.run = p.share ? max(1, (s.held - base + TT - 1) / TT) : 1;
    return u;
}

template <int DP, int WM, int WT, int SRC, bool PRECISE>
__global__ void __attribute__((amdgpu_flat_work_group_size(64 * WM * WT, 64 * WM * WT), amdgpu_waves_per_eu(attend_waves(DP, WM, WT), attend_waves(DP, WM, WT))))
attend_kernel(const AttendArgs p) {
    using S = Shape<DP, WM, WT, SRC>;
    constexpr int STEPS = DP / 16, DT = DP / 32, SUB = S::SUB, TT = S::TT, M = S::M;
    constexpr float LOG2E = 1.4426950408889634f;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * S::STAGE];
    __shared__ float tops[S::WAVES][32], totals[S::WAVES][32];
    __shared__ int joins[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5;
    const int wm = wave % WM, wt = wave / WM;
    const bool capped = p.softcap > 0.0f;
    const int runs = p.dim / 8;  // 16-byte runs of a token that hold values

    // Runs past `dim` are zeros, written once: no load fills them.
    if (runs < S::RUNS) {
        for (int i = tid; i < 2 * 2 * TT * S::RUNS; i += S::THREADS) {
            const int token = i / S::RUNS % TT, run = i % S::RUNS, matrix = i / (S::RUNS * TT) & 1;
            if ((run ^ (matrix ? key_v(token) : key_k(token))) >= runs) *reinterpret_cast<u32x4 *>(lds + i * 16) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
    }

    // ---- this workgroup's tiles and the sequence they begin in; all uniform ----
    int total = 0, before = 0, b = 0;
    auto size_of = [&](int i) {
        if (i >= p.sequences) return 0;
        const Units u = units_of<M, TT>(p, sequence(p, i));
        return u.tiles * u.run;
    };
    for (int i = 0; i < p.sequences; i += 64) {
        int v = size_of(i + lane);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
        total += v;
    }
    total = __builtin_amdgcn_readfirstlane(total) * p.kv_heads;
    const Share share(total, gridDim.x);
    int start, end;
    if (p.share) {
        start = share.first(min((int)blockIdx.x, share.groups));
        end = share.first(min((int)blockIdx.x + 1, share.groups));
    } else {
        // The last rows of a causal sequence have the most keys: they go first, and every kv head keeps its place (its XCD).
        const int tiles = total / p.kv_heads, tile = (int)blockIdx.x / p.kv_heads;
        start = tile < tiles ? (tiles - 1 - tile) * p.kv_heads + (int)blockIdx.x % p.kv_heads : 0;
        end = tile < tiles ? start + 1 : 0;
    }
    if (start >= end) return;
    for (int i = 0; i < p.sequences; i += 64) {
        const int v = size_of(i + lane), upto = wave_scan(v, lane);
        const uint64_t past = __ballot((before + upto) * p.kv_heads > start);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            before += l > 0 ? __shfl(upto, l - 1, 64) : 0;
            b = i + l;
            break;
        }
        before += __shfl(upto, 63, 64);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    int seq0 = __builtin_amdgcn_readfirstlane(before) * p.kv_heads;
    Sequence seq;
    Units units;
    auto enter = [&]() {
        const Sequence s = sequence(p, b);
        seq.row0 = __builtin_amdgcn_readfirstlane(s.row0);
        seq.count = __builtin_amdgcn_readfirstlane(s.count);
        seq.held = __builtin_amdgcn_readfirstlane(s.held);
        units = units_of<M, TT>(p, seq);
    };
    enter();

    struct Part {
        int first, tiles;      // its numbered tiles (0: none)
        int row0, rows, kvh;   // first row of the tile in its sequence, the sequence's rows; its kv head
        int at;                // the sequence's first row of q
    } parts[2] = {};

    for (int pos = start; pos < end;) {
        while (b + 1 < p.sequences && pos >= seq0 + units.tiles * units.run * p.kv_heads) {
            seq0 += units.tiles * units.run * p.kv_heads;
            ++b;
            enter();
        }
        const int in_seq = pos - seq0;
        const int unit = in_seq / units.run, part0 = in_seq - unit * units.run;
        const int kvh = unit % p.kv_heads, tile = unit / p.kv_heads;
        if (in_seq < 0 || tile >= units.tiles) break;  // starts that do not ascend
        const int numbered = p.share ? min(units.run - part0, end - pos) : 1;
        const int rows = seq.count * p.group;  // of the sequence
        const int row0 = tile * M;
        const int first = seq.held - seq.count;  // the place of the chunk's first token

        // ---- the tokens that these rows see ----
        const int rowN = min(row0 + M, rows) - 1;
        const int tok0 = row0 / p.group, tokN = rowN / p.group;
        const int stop = p.causal ? min(seq.held, first + tokN + 1) : seq.held;                     // past the last
        const bool windowed = p.causal && p.window > 0;
        const int base = (windowed ? max(0, first + tok0 - p.window + 1) : 0) & ~15;
        const int tiles = max(0, (stop - base + TT - 1) / TT);
        // Of the unit's numbered tiles, some may lie past these rows' last: none is read there.
        const int t_from = p.share ? min(part0, tiles) : 0, t_to = p.share ? min(part0 + numbered, tiles) : tiles;

        // ---- the wave's rows ----
        const int r = row0 + wm * 32 + c;
        const int tok = min(r, rows - 1) / p.group, head = kvh * p.group + (min(r, rows - 1) - tok * p.group);
        const bool live = r < rows;
        const int w0 = row0 + wm * 32, wN = min(w0 + 31, rows - 1);
        const bool any = w0 < rows;
        const int hi = p.causal ? min(first + tok, seq.held - 1) : seq.held - 1;   // the last token a row sees
        const int lo = windowed ? first + tok - p.window + 1 : 0;                  // the first
        const int hi_min = __builtin_amdgcn_readfirstlane(p.causal ? first + min(w0, rows - 1) / p.group : seq.held - 1);
        const int hi_max = __builtin_amdgcn_readfirstlane(any ? (p.causal ? first + wN / p.group : seq.held - 1) : -1);
        const int lo_min = windowed ? hi_min - p.window + 1 : 0, lo_max = windowed ? hi_max - p.window + 1 : 0;

        float unit_scale = p.scale * (S::F8 && p.k_scale ? p.k_scale[kvh] : 1.0f);
        const bool minus = unit_scale < 0.0f;  // then Q is taken with the other sign: the largest score is that of S
        unit_scale = fabsf(unit_scale) * (capped ? 1.0f / p.softcap : LOG2E);
        if (unit_scale < 1e-30f) unit_scale = 1e-30f;  // (0 times a masked score would be a NaN)
        bf16x8 q[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            u32x4 v = {0, 0, 0, 0};
            if (live && 2 * s + h < runs)
                v = *reinterpret_cast<const u32x4 *>(p.q + (int64_t)(seq.row0 + tok) * p.q_tok + (int64_t)head * p.q_head + 16 * s + 8 * h);
            if (minus) v ^= u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
            q[s] = __builtin_bit_cast(bf16x8, v);
        }

        // ---- loads ----
        const uint8_t *const kbase = p.kc + ((int64_t)kvh * p.kc_head + (S::PAGED ? 0 : (int64_t)seq.row0 * p.kc_tok)) * (S::F8 ? 1 : 2);
        const uint8_t *const vbase = p.vc + ((int64_t)kvh * p.vc_head + (S::PAGED ? 0 : (int64_t)seq.row0 * p.vc_tok)) * (S::F8 ? 1 : 2);
        const auto pages = (const __attribute__((address_space(4))) int32_t *)(p.pages + (int64_t)b * p.pages_row);
        constexpr int ES = S::F8 ? 1 : 2;
        const int in_load = lane / S::LANES, run = lane % S::LANES;  // a lane's token of a load, and its place in LDS there
        auto page_of = [&](int token) { return (int)(((uint64_t)(uint32_t)token * p.page_mul) >> p.page_shift); };
        // The pages of a tile: PAGES16's, one for each 16 tokens, uniform; EACH: lane l's is that of tokens l and 64 + l.
        struct Where {
            int id[S::EACH ? (TT + 63) / 64 : S::PAGED ? S::IDS : 1];
        };
        auto locate = [&](int token0) {
            Where w;
            if constexpr (S::EACH) {
#pragma unroll
                for (int i = 0; i < (TT + 63) / 64; ++i) w.id[i] = pages[page_of(min(token0 + 64 * i + lane, seq.held - 1))];
            } else if constexpr (S::PAGED) {
#pragma unroll
                for (int i = 0; i < S::IDS; ++i) w.id[i] = pages[page_of(min(token0 + 16 * i, (seq.held - 1) & ~15))];
            }
            return w;
        };
        auto inside = [&](int id) { return (unsigned)id < (unsigned)p.page_count; };
        // The offsets (elements) of load i's tokens, the lane's among them.
        auto offsets = [&](const Where &w, int token0, int i, int64_t &k, int64_t &v) {
            const int local = wave * S::MINE + i * S::PER_LOAD;  // the load's first token in the tile
            if constexpr (S::EACH) {
                const int mine = local + in_load;
                const int t = min(token0 + mine, seq.held - 1);
                int id = w.id[0];
#pragma unroll
                for (int j = 1; j < (TT + 63) / 64; ++j) id = (local >> 6) == j ? w.id[j] : id;
                id = __shfl(id, mine & 63, 64);
                id = inside(id) ? id : 0;
                const int in = t - page_of(t) * p.page;
                k = id * p.kc_page + in * p.kc_tok;
                v = id * p.vc_page + in * p.vc_tok;
            } else if constexpr (S::PAGED) {
                const int t16 = min(token0 + (local & ~15), (seq.held - 1) & ~15);
                int id = 0;
#pragma unroll
                for (int j = 0; j < S::IDS; ++j) id = (local >> 4) == j ? w.id[j] : id;
                id = inside(id) ? id : 0;
                const int in = t16 - page_of(t16) * p.page;
                k = id * p.kc_page + in * p.kc_tok + (int64_t)((local & 15) + in_load) * p.kc_tok;
                v = id * p.vc_page + in * p.vc_tok + (int64_t)((local & 15) + in_load) * p.vc_tok;
            } else {
                const int t = min(token0 + local + in_load, seq.held - 1);
                k = t * p.kc_tok;
                v = t * p.vc_tok;
            }
        };
        auto load = [&](const Where &w, int token0, int stage) {
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                int64_t ko, vo;
                offsets(w, token0, i, ko, vo);
                const int row = wave * S::MINE + i * S::PER_LOAD + in_load;
                const int kr = run ^ key_k(row), vr = run ^ key_v(row);
                uint8_t *const to = lds + stage * S::STAGE + (wave * S::LOADS + i) * 1024;
                if (kr < runs) __builtin_amdgcn_global_load_lds((wd::glb_ptr)(kbase + ko * 2 + kr * 16), (wd::lds_ptr)to, 16, 0, 0);
                if (vr < runs) __builtin_amdgcn_global_load_lds((wd::glb_ptr)(vbase + vo * 2 + vr * 16), (wd::lds_ptr)(to + S::MATRIX), 16, 0, 0);
            }
        };
        // The tile's tokens on a page outside the pools, a bit each of 64.
        struct Bad {
            uint64_t bits[(TT + 63) / 64];
            __device__ __forceinline__ uint64_t from(int token) const {
                uint64_t word = bits[0];
#pragma unroll
                for (int i = 1; i < (TT + 63) / 64; ++i) word = (token >> 6) == i ? bits[i] : word;
                return word >> (token & 63);
            }
            __device__ __forceinline__ bool any() const {
                uint64_t all = bits[0];
#pragma unroll
                for (int i = 1; i < (TT + 63) / 64; ++i) all |= bits[i];
                return all != 0;
            }
        };
        auto bad_of = [&](const Where &w) {
            Bad bad;
#pragma unroll
            for (int i = 0; i < (TT + 63) / 64; ++i) {
                bad.bits[i] = 0;
                if constexpr (S::EACH) {
                    bad.bits[i] = __ballot(!inside(w.id[i]));
                } else if constexpr (S::PAGED) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (4 * i + j < S::IDS && !inside(w.id[4 * i + j])) bad.bits[i] |= 0xFFFFull << (16 * j);
                }
            }
            return bad;
        };
        // Whether no row sees a tile's token, past the sequence's last or on such a page. Its values, which may be anything, are
        // made zeros in LDS: 0 times an infinity or a NaN would not hide them.
        auto gone = [&](int token0, const Bad &bad, int token) { return token0 + token >= seq.held || (S::PAGED && (bad.from(token) & 1)); };
        auto clear = [&](int token0, const Bad &bad, int stage) {
            if (token0 + TT <= seq.held && !bad.any()) return;
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i)
                if (gone(token0, bad, wave * S::MINE + i * S::PER_LOAD + in_load))
                    *reinterpret_cast<u32x4 *>(lds + stage * S::STAGE + S::MATRIX + (wave * S::LOADS + i) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        };

        // e4m3: to registers, and widened into LDS later.
        u32x4 k8[S::F8 ? S::LOADS : 1], v8[S::F8 ? S::LOADS : 1];
        auto fetch = [&](const Where &w, int token0) {
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                int64_t ko, vo;
                offsets(w, token0, i, ko, vo);
                const int at = 16 * run < p.dim ? 16 * run : 0;
                k8[i] = *reinterpret_cast<const u32x4 *>(kbase + ko + at);
                v8[i] = *reinterpret_cast<const u32x4 *>(vbase + vo + at);
            }
        };
        auto widen = [&](int token0, const Bad &bad, int stage) {
            if (16 * run >= p.dim) return;
            const bool some = token0 + TT > seq.held || bad.any();
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const int row = wave * S::MINE + i * S::PER_LOAD + in_load;
                uint8_t *const to = lds + stage * S::STAGE + row * S::ROW;
                if (some && gone(token0, bad, row)) v8[i] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    auto wide = [&](const u32x4 &d) {
                        const uint32_t x = d[2 * half], y = d[2 * half + 1];
                        return u32x4{bf16_of_e4m3<0>(x), bf16_of_e4m3<1>(x), bf16_of_e4m3<0>(y), bf16_of_e4m3<1>(y)};
                    };
                    *reinterpret_cast<u32x4 *>(to + ((2 * run + half) ^ key_k(row)) * 16) = wide(k8[i]);
                    *reinterpret_cast<u32x4 *>(to + S::MATRIX + ((2 * run + half) ^ key_v(row)) * 16) = wide(v8[i]);
                }
            }
        };
        // ---- fragments: the lane's places in a stage ----
        const int wave_token = wt * 32 * SUB;
        int k_at[4];  // run 2s + h of token c, by s mod 4 (further ones 128 bytes on)
#pragma unroll
        for (int s = 0; s < 4; ++s) k_at[s] = (wave_token + c) * S::ROW + (((2 * s + h) ^ key_k(c)) * 16);
        // Transposed: lanes of 16 take 16 values of 4 tokens. Value part d's run is 4d + 2·(lane / 16 mod 2) + ..., turned.
        const int v_token = 4 * h + (lane & 15) / 4;
        const int v_run = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), v_key = key_v(v_token);
        int v_at[2];  // by d mod 2
#pragma unroll
        for (int d = 0; d < 2; ++d) v_at[d] = S::MATRIX + (wave_token + v_token) * S::ROW + (((4 * d + v_run) ^ v_key) * 16) + 8 * (lane & 1);

        float top = -INFINITY, sum = 0.0f;
        f32x16 o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

        Where now, next;
        if (t_from < t_to) {
            now = locate(base + t_from * TT);
            __syncthreads();  // the run before has been read
            if constexpr (S::F8) {
                fetch(now, base + t_from * TT);
                widen(base + t_from * TT, bad_of(now), t_from & 1);
            } else {
                load(now, base + t_from * TT, t_from & 1);
            }
            if (t_from + 1 < t_to) next = locate(base + (t_from + 1) * TT);
        }
#pragma clang loop unroll(disable)
        for (int t = t_from; t < t_to; ++t) {
            const int stage = (t & 1) * S::STAGE, token0 = base + t * TT;
            const bool more = t + 1 < t_to;
            const Bad bad = bad_of(now);
            if constexpr (!S::F8) {
                wd::wait_vmcnt<0>();
                clear(token0, bad, t & 1);
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (more) {
                if constexpr (S::F8) fetch(next, token0 + TT);
                else load(next, token0 + TT, (t + 1) & 1);
                now = next;
                if (t + 2 < t_to) next = locate(token0 + 2 * TT);
            }
            const int mine = token0 + wave_token;  // the wave's first token
            if (mine <= hi_max && mine + 32 * SUB > lo_min) {
                f32x16 s[SUB];
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[u][e] = 0.0f;
#pragma unroll
                for (int j = 0; j < STEPS; ++j)
#pragma unroll
                    for (int u = 0; u < SUB; ++u) {
                        const bf16x8 kk = *reinterpret_cast<const bf16x8 *>(lds + stage + k_at[j & 3] + (j >> 2) * 128 + u * 32 * S::ROW);
                        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kk, q[j], s[u], 0, 0, 0);
                    }
                uint32_t bits[SUB], any_bad = 0;  // the wave's bad tokens
#pragma unroll
                for (int u = 0; u < SUB; ++u) any_bad |= bits[u] = S::PAGED ? (uint32_t)bad.from(wave_token + 32 * u) : 0u;
                const bool edge = mine + 32 * SUB - 1 > hi_min || mine < lo_max || any_bad != 0;
                float scale = unit_scale;
                if (capped) {
                    scale = 1.0f;
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[u][e] = p.softcap * LOG2E * tanh_rel(s[u][e] * unit_scale);
                }
                const int hi_rel = hi - mine - 4 * h, lo_rel = lo - mine - 4 * h;
                auto dead_of = [&](int at, int u) {  // token 32u + at of the lane (4h apart from the wave's)
                    const int j = 32 * u + at;
                    bool dead = j > hi_rel || j < lo_rel;
                    if constexpr (S::PAGED) dead = dead || (bits[u] >> (at + 4 * h) & 1);
                    return dead;
                };
                if (edge) {
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[u][e] = dead_of(8 * (e >> 2) + (e & 3), u) ? -INFINITY : s[u][e];
                }
                float m = s[0][0];
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) m = fmaxf(m, s[u][e]);
                m *= scale;
                if (__any(m > top + 8.0f)) {
                    m = fmaxf(over_halves<false>(m), top);
                    const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - m);
                    top = m;
                    sum *= keep;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] *= keep;
                }
                float from = top == -INFINITY ? 0.0f : top;
                if (__any(fabsf(from) > 0x1p16f)) {
                    // So far out the scaled score's rounding, which a fused multiply-add does not share with `from`, would count.
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[u][e] = s[u][e] * scale - from;
                    scale = 1.0f;
                    from = 0.0f;
                }
                // The probabilities, two a dword in the order of the second product's tokens; what a bf16 leaves of each besides
                // (PRECISE), at least 2^-126 of one that is not 0, so that an infinite value meets no zero and no other sign.
                u32x4 w[SUB][2], rest[PRECISE ? SUB : 1][2];
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e], scale, -from));
                        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e + 1], scale, -from));
                        sum += x + y;
                        if constexpr (PRECISE) {
                            const uint32_t a = __float_as_uint(x), z = __float_as_uint(y);
                            w[u][e >> 3][(e >> 1) & 3] = __builtin_amdgcn_perm(z, a, 0x07060302u);
                            rest[u][e >> 3][(e >> 1) & 3] = pack_bf16_rne(fmaxf(x - __uint_as_float(a & 0xFFFF0000u), fminf(x, 0x1p-126f)),
                                                                         fmaxf(y - __uint_as_float(z & 0xFFFF0000u), fminf(y, 0x1p-126f)));
                        } else {
                            w[u][e >> 3][(e >> 1) & 3] = pack_bf16_rne(x, y);
                        }
                    }
                auto values = [&](int u, int ks, int d) {
                    const uint8_t *const at = lds + stage + v_at[d & 1] + (d >> 1) * 128 + (32 * u + 16 * ks) * S::ROW;
                    const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)at);
                    const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(at + 8 * S::ROW));
                    const u32x2 lo2 = __builtin_bit_cast(u32x2, x), hi2 = __builtin_bit_cast(u32x2, y);
                    return u32x4{lo2[0], lo2[1], hi2[0], hi2[1]};
                };
                bool wild = false;  // a token that some rows do not see may hold an infinity or a NaN
                if (edge) {
                    bool found = false;
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                            for (int d = 0; d < DT; ++d) {
                                const u32x4 v = values(u, ks, d);
                                found = found || unbounded(v[0]) || unbounded(v[1]) || unbounded(v[2]) || unbounded(v[3]);
                            }
                    wild = __any(found);
                }
                if (!wild) {
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                            for (int d = 0; d < DT; ++d) {
                                const bf16x8 v = __builtin_bit_cast(bf16x8, values(u, ks, d));
                                if constexpr (PRECISE) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8, rest[u][ks]), o[d], 0, 0, 0);
                                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8, w[u][ks]), o[d], 0, 0, 0);
                            }
                } else {
                    // Token by token: a row takes the product with one it sees, and keeps what it had where it does not.
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
#pragma unroll 1
                            for (int j = 0; j < 16; ++j) {
                                // Token j of the 16: in half j / 4 mod 2, place 4·(j / 8) + j mod 4 of the lane's eight.
                                const int place = 4 * (j >> 3) + (j & 3), half = (j >> 2) & 1;
                                const int at = 16 * ks + j, rel = 32 * u + at;
                                bool seen = rel <= hi - mine && rel >= lo - mine;
                                if constexpr (S::PAGED) seen = seen && !(bits[u] >> at & 1);
                                u32x4 keep;
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    keep[e] = h == half && (place >> 1) == e ? (place & 1 ? 0xFFFF0000u : 0x0000FFFFu) : 0u;
#pragma unroll
                                for (int d = 0; d < DT; ++d) {
                                    const bf16x8 v = __builtin_bit_cast(bf16x8, values(u, ks, d) & keep);
                                    f32x16 with = o[d];
                                    if constexpr (PRECISE) with = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8, rest[u][ks] & keep), with, 0, 0, 0);
                                    with = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8, w[u][ks] & keep), with, 0, 0, 0);
#pragma unroll
                                    for (int e = 0; e < 16; ++e) o[d][e] = seen ? with[e] : o[d][e];
                                }
                            }
                }
            }
            if constexpr (S::F8) {
                if (more) widen(token0 + TT, bad_of(now), (t + 1) & 1);
            }
        }

        // ---- the waves of a row joined, by the first ----
        sum = over_halves<true>(sum);
        if constexpr (WT > 1) {
            __syncthreads();  // the last tile has been read
            float *const mine = reinterpret_cast<float *>(lds) + ((wt - 1) * WM + wm) * (DT * 16 * 64) + lane;
            if (h == 0) { tops[wave][c] = top; totals[wave][c] = sum; }
            if (wt > 0) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mine[(d * 16 + e) * 64] = o[d][e];
            }
            __syncthreads();
            if (wt == 0) {
                float all = top;
#pragma unroll
                for (int i = 1; i < WT; ++i) all = fmaxf(all, tops[i * WM + wm][c]);
                const float from = all == -INFINITY ? 0.0f : all;
                float weight = __builtin_amdgcn_exp2f(top - from);
                sum *= weight;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= weight;
#pragma unroll
                for (int i = 1; i < WT; ++i) {
                    weight = __builtin_amdgcn_exp2f(tops[i * WM + wm][c] - from);
                    sum = __builtin_fmaf(totals[i * WM + wm][c], weight, sum);
                    const float *const other = reinterpret_cast<const float *>(lds) + ((i - 1) * WM + wm) * (DT * 16 * 64) + lane;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] = __builtin_fmaf(other[(d * 16 + e) * 64], weight, o[d][e]);
                }
                top = all;
            }
        }
        const bool whole = !p.share || numbered == units.run;
        if (wt == 0) {
            if (whole) {
                if (live) {
                    const float by = inverse(sum) * (S::F8 && p.v_scale ? p.v_scale[kvh] : 1.0f);
                    uint16_t *const dst = p.out + (int64_t)(seq.row0 + tok) * p.o_tok + (int64_t)head * p.o_head;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const int at = 32 * d + 2 * e + 4 * h;
                            if (at < p.dim)
                                *reinterpret_cast<u32x2 *>(dst + at) = u32x2{pack_bf16_rne(o[d][e] * by, o[d][e + 1] * by),
                                                                             pack_bf16_rne(o[d][e + 2] * by, o[d][e + 3] * by)};
                        }
                }
            } else {
                float *const slot = p.part + (int64_t)(2 * blockIdx.x + (pos == start ? 0 : 1)) * attend_part_floats(DP, WM);
                if (h == 0) put(slot + 2 * (wm * 32 + c), Pair{top, sum});
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        put(slot + 2 * M + 2 * (((wm * DT + d) * 8 + e / 2) * 64 + lane), Pair{o[d][e], o[d][e + 1]});
            }
        }
        if (!whole) {
            Part &part = pos == start ? parts[0] : parts[1];
            part.first = seq0 + unit * units.run;
            part.tiles = units.run;
            part.row0 = row0;
            part.rows = rows;
            part.kvh = kvh;
            part.at = seq.row0;
        }
        pos += numbered;
    }

    // ---- the parts' slots are written before their counters say so; the last workgroup to count joins ----
    if (!p.share || (parts[0].tiles == 0 && parts[1].tiles == 0)) return;
    wd::wait_vmcnt<0>();
    __syncthreads();
    if (tid < 2) {
        const Part part = tid == 0 ? parts[0] : parts[1];
        bool last = false;
        if (part.tiles != 0) {
            // Of the units that more than one workgroup has, one begins in each: its counter is that workgroup's.
            const int g0 = share.of(part.first), others = share.of(part.first + part.tiles - 1) - g0;
            int *const mark = p.marks + (int64_t)g0 * MARK;
            last = __hip_atomic_fetch_add(mark, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == others;
            if (last) __hip_atomic_store(mark, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        joins[tid] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        if (!joins[i]) continue;
        const Part part = i == 0 ? parts[0] : parts[1];
        const int g0 = share.of(part.first), g1 = share.of(part.first + part.tiles - 1);
        const int slot0 = 2 * g0 + (share.first(g0) < part.first ? 1 : 0);
        const float v_scale = S::F8 && p.v_scale ? p.v_scale[part.kvh] : 1.0f;
        // A thread takes two values, side by side in a row, of every slot.
        for (int item = tid; item < M * DP / 2; item += S::THREADS) {
            const int l = item & 63, e = 2 * (item >> 6 & 7), d = (item >> 9) % DT, set = (item >> 9) / DT;
            const int row = 32 * set + (l & 31), at = 32 * d + 8 * (e >> 2) + 4 * (l >> 5) + (e & 3);
            if (part.row0 + row >= part.rows || at >= p.dim) continue;
            float top = -INFINITY, sum = 0.0f, x = 0.0f, y = 0.0f;
            constexpr int ROUND = 4;  // slots whose loads are under way at once
            for (int g = g0; g <= g1; g += ROUND) {
                Pair s[ROUND], v[ROUND];
#pragma unroll
                for (int k = 0; k < ROUND; ++k) {
                    const int from = min(g + k, g1);
                    const float *const slot = p.part + (int64_t)(from == g0 ? slot0 : 2 * from) * attend_part_floats(DP, WM);
                    s[k] = get(slot + 2 * row);
                    v[k] = get(slot + 2 * M + 2 * item);
                }
                float most = top;
#pragma unroll
                for (int k = 0; k < ROUND; ++k) most = fmaxf(most, s[k].a);
                const float from = most == -INFINITY ? 0.0f : most;
                const float keep = __builtin_amdgcn_exp2f(top - from);
                top = most;
                sum *= keep;
                x *= keep;
                y *= keep;
#pragma unroll
                for (int k = 0; k < ROUND; ++k) {
                    if (g + k > g1) continue;
                    const float weight = __builtin_amdgcn_exp2f(s[k].a - from);
                    sum = __builtin_fmaf(s[k].b, weight, sum);
                    x = __builtin_fmaf(v[k].a, weight, x);
                    y = __builtin_fmaf(v[k].b, weight, y);
                }
            }
            const float by = inverse(sum) * v_scale;
            const int r = part.row0 + row, tok = r / p.group, head = part.kvh * p.group + (r - tok * p.group);
            *reinterpret_cast<uint32_t *>(p.out + (int64_t)(part.at + tok) * p.o_tok + (int64_t)head * p.o_head + at) =
                pack_bf16_rne(x * by, y * by);
        }
    }
}

}  // namespace attend
}  // namespace sq8
