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
// A workgroup has WM · WT waves: WM sets of 32 rows, and WT waves that share a tile's tokens and are joined at the end. Tiles of
// keys and values lie in four slots of LDS each, in runs of 16 bytes whose places are turned by the row's number; half the waves
// load keys, half values, without registers, and bf16 tiles are asked for three and four barriers before their use (e4m3 codes
// go through registers, widened on the way). One barrier a tile. Beside the softmax of a tile run the scores of the next, beside
// its outputs the search of the next one's maximum and the addresses of what is asked for next; the loop is written out in that
// order for each slot. What it took, of 8192 causal tokens with 32 heads on 8 of 128: keys a tile ahead of the values and no
// spilled register (a reload waits for all loads under way) from 1.2 ms to 636 µs; the compiler's own waits out of the way (its
// LDS loads made transposed reads of other slots wait for them) and maxima and conversions kept between the matrix instructions,
// 571; addresses stepped instead of multiplied, 571 to 554 on another card; rows written in whole runs, 563 to 556 on a third.
//
// There it takes 544 to 602 µs, from card to card, 1010 to 910 TFLOP/s of the products that the mask leaves, where a large library
// product of normal values does 1384, both at the power limit (1.8 GHz of 2.4): the matrix pipes are busy 45 % of the cycles, the
// vector ALUs 40 %. Without exponentials it would take 8 % less, without loads 5 %, without three quarters of the second
// product 21 %: no one thing bounds it. Tried
// and not faster: outputs a tile late beside the next tile's softmax (6 % slower), reads six instructions ahead, wave
// priorities, places turned so that no read meets another in a bank (the counted conflicts went from 68 M to none, the time stayed),
// loads between the matrix instructions. 4608 tokens of 24 heads, not causal, take 281 to 306 µs: 432 tiles on 256 CUs, two rounds
// of which the second is two thirds full. 2048 new tokens behind 30 720 in pages of 64, 1.13 to 1.22 ms (950 to 870 TFLOP/s). Capped scores
// take a hyperbolic tangent each: of 30, the two calls take 1120 and 2170 µs (with values looked over in every tile 1275 and 2940).
//
// Tiles of rows (sq8_text_plan.hip): 256, 128 or 64 for prompts, by how many there are for the card's CUs (100 tokens, 32 heads on
// 8: 11.8 µs with 64: the launch, 3 µs of loads one after another, four
// tiles whose instructions are read for the first time, the join of two waves); 256 and 128 for chunks, and for few rows sq8_chunk.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "sq8_attend_device.h"
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
    static constexpr int TT = attend_tokens(WT);                      // tokens of a tile: 32 for each wave that shares it
    static constexpr int STAGES = kAttendStages;
    static constexpr int ROW = 2 * DP;                                // bytes of a token in LDS
    static constexpr int RUNS = DP / 8;                               // and its 16-byte runs
    static constexpr int MATRIX = TT * ROW;
    static constexpr bool F8 = SRC == PAGES16_F8 || SRC == PAGES_F8;
    static constexpr bool PAGED = SRC != ROWS, EACH = SRC == PAGES || SRC == PAGES_F8;  // EACH: rows are looked up one by one
    // Half the waves load keys, half values.
    static constexpr int PER_LOAD = F8 ? 1024 / DP : 1024 / ROW;      // tokens a wave's load instruction fills
    static constexpr int MINE = TT / (WAVES / 2);                     // tokens a wave loads of a tile
    static constexpr int LOADS = MINE / PER_LOAD;
    static constexpr int LANES = 64 / PER_LOAD;                       // lanes to a token
    static constexpr int IDS = EACH ? LOADS : PAGED ? (MINE + 15) / 16 : 1;  // page indices that a wave's loads take
    static_assert(LOADS >= 1 && LOADS * PER_LOAD * (WAVES / 2) == TT, "whole loads");
    static_assert(MINE <= 16 || MINE % 16 == 0, "a load's tokens lie in one sixteen");
};

__device__ __forceinline__ int key_k(int row) { return row & 7; }
__device__ __forceinline__ int key_v(int row) { return 2 * (row & 3); }

// 16 bytes a lane from memory to LDS, to the wave's place and 16 bytes on for each lane. Written out: beside the builtin, the
// compiler waits for all loads under way before it reads anything transposed from LDS. (No register is loaded; whoever reads the
// place waits for it by itself.)
__device__ __forceinline__ void to_lds(const uint8_t *from, uint32_t place) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(place) : "memory", "m0");
}

// A value's maximum (sum) over the two lanes of a row.
template <bool SUM>
__device__ __forceinline__ float over_halves(float v) {
    typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
    const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
    return SUM ? a + b : fmaxf(a, b);
}

template <int DP, int WM, int WT, int SRC, bool SHARE>
__global__ void __attribute__((amdgpu_flat_work_group_size(64 * WM * WT, 64 * WM * WT), amdgpu_waves_per_eu(attend_waves(DP, WT), attend_waves(DP, WT))))
attend_kernel(const AttendArgs p) {
    using S = Shape<DP, WM, WT, SRC>;
    constexpr int STEPS = DP / 16, DT = DP / 32, TT = S::TT, M = S::M;
    constexpr float LOG2E = 1.4426950408889634f;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * S::STAGES * S::MATRIX];  // keys, then values
    __shared__ float tops[S::WAVES][32], totals[S::WAVES][32];
    __shared__ int joins[2], wilds[S::WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5;
    const int wm = wave % WM, wt = wave / WM;
    const bool capped = p.softcap > 0.0f;
    const int runs = p.dim / 8;  // 16-byte runs of a token that hold values

    // Runs past `dim` are zeros, which no load fills: written here, and again where a unit's outputs went by way of LDS.
    auto clear_ends = [&]() {
        if (runs >= S::RUNS) return;
        for (int i = tid; i < 2 * S::STAGES * TT * S::RUNS; i += S::THREADS) {
            const int token = i / S::RUNS % TT, run = i % S::RUNS, matrix = i / (S::RUNS * TT * S::STAGES);
            if ((run ^ (matrix ? key_v(token) : key_k(token))) >= runs) *reinterpret_cast<u32x4 *>(lds + i * 16) = u32x4{0, 0, 0, 0};
        }
    };
    clear_ends();

    // ---- this workgroup's tiles and the sequence they begin in; all uniform ----
    int upto = 0;
    const int total = all_units<M, TT, SHARE>(p, lane, upto) * p.kv_heads;
    const Share share(total, gridDim.x);
    int start, end, b = 0, before = 0;
    if constexpr (SHARE) {
        start = share.first(min((int)blockIdx.x, share.groups));
        end = share.first(min((int)blockIdx.x + 1, share.groups));
    } else {
        // The last rows of a causal sequence have the most keys: they go first, and every kv head keeps its place (its XCD).
        const int tiles = total / p.kv_heads, tile = (int)blockIdx.x / p.kv_heads;
        start = tile < tiles ? (tiles - 1 - tile) * p.kv_heads + (int)blockIdx.x % p.kv_heads : 0;
        end = tile < tiles ? start + 1 : 0;
    }
    if (start >= end) return;
    find_unit<M, TT, SHARE>(p, start, lane, upto, b, before);
    int seq0 = before * p.kv_heads;
    Sequence seq;
    Units units;
    auto enter = [&]() {
        const Sequence s = sequence(p, b);
        seq.row0 = __builtin_amdgcn_readfirstlane(s.row0);
        seq.count = __builtin_amdgcn_readfirstlane(s.count);
        seq.held = __builtin_amdgcn_readfirstlane(s.held);
        units = units_of<M, TT, SHARE>(p, seq);
    };
    enter();

    __shared__ Part parts[2];  // of the workgroup's first unit and of its last
    if (SHARE && tid < 2) parts[tid].tiles = 0;

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
        const int numbered = SHARE ? min(units.run - part0, end - pos) : 1;
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
        const int t_from = SHARE ? min(part0, tiles) : 0, t_to = SHARE ? min(part0 + numbered, tiles) : tiles;

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
        const int lo_max = windowed ? hi_max - p.window + 1 : 0;

        // Uniform, and kept in scalar registers.
        auto scalar = [](float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); };
        float unit_scale = p.scale * (S::F8 && p.k_scale ? p.k_scale[kvh] : 1.0f);
        const bool minus = unit_scale < 0.0f;  // then Q is taken with the other sign: the largest score is that of S
        unit_scale = scalar(fabsf(unit_scale) * (capped ? 1.0f / p.softcap : LOG2E));
        // Scaled before the masked ones become -inf: capped scores, and those by a scale of 0 (or a NaN), which -inf would make NaNs of.
        const bool early = capped || !(unit_scale >= 0x1p-126f);
        bf16x8 q[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            u32x4 v = {0, 0, 0, 0};
            if (live && 2 * s + h < runs)
                v = *reinterpret_cast<const u32x4 *>(p.q + (int64_t)(seq.row0 + tok) * p.q_tok + (int64_t)head * p.q_head + 16 * s + 8 * h);
            q[s] = __builtin_bit_cast(bf16x8, v);
        }

        // ---- loads: the first half of the waves keys, the others values ----
        constexpr int ES = S::F8 ? 1 : 2;
        const bool of_keys = wave < S::WAVES / 2;
        const int slice = wave % (S::WAVES / 2);
        const int64_t tok_bytes = (of_keys ? p.kc_tok : p.vc_tok) * ES, page_bytes = (of_keys ? p.kc_page : p.vc_page) * ES;
        const uint8_t *const pool = (of_keys ? p.kc + (int64_t)kvh * p.kc_head * ES : p.vc + (int64_t)kvh * p.vc_head * ES) +
                                    (S::PAGED ? 0 : (int64_t)seq.row0 * tok_bytes);
        const auto pages = (const __attribute__((address_space(4))) int32_t *)(p.pages + (int64_t)b * p.pages_row);
        const int in_load = lane / S::LANES, run = lane % S::LANES;  // a lane's token of a load, and its place in LDS there
        auto page_of = [&](int token) { return (int)(((uint64_t)(uint32_t)token * p.page_mul) >> p.page_shift); };
        auto inside = [&](int id) { return (unsigned)id < (unsigned)p.page_count; };
        // A lane's run of load i, in the order of LDS (bf16): turned by its token's number.
        auto turned = [&](int i) {
            const int row = i * S::PER_LOAD + in_load;  // (the wave's tokens begin at a multiple of eight)
            return run ^ (of_keys ? key_k(row) : key_v(row));
        };
        // The page indices of a wave's loads of a tile (a uniform one for 16 tokens; EACH: a lane's own for each load).
        struct Ids {
            int id[S::IDS];
        };
        auto look_up = [&](int token0) {
            Ids w;
#pragma unroll
            for (int i = 0; i < S::IDS; ++i) {
                if constexpr (S::EACH) w.id[i] = pages[page_of(min(token0 + slice * S::MINE + i * S::PER_LOAD + in_load, seq.held - 1))];
                else if constexpr (S::PAGED) w.id[i] = pages[page_of(min(token0 + ((slice * S::MINE) & ~15) + 16 * i, (seq.held - 1) & ~15))];
                else w.id[i] = 0;
            }
            return w;
        };
        // Where load i's tokens lie: the lane's address.
        auto address = [&](const Ids &w, int token0, int i) -> const uint8_t * {
            const int local = slice * S::MINE + i * S::PER_LOAD;
            const int64_t in_bytes = in_load * tok_bytes;
            if constexpr (S::EACH) {
                const int t = min(token0 + local + in_load, seq.held - 1);
                const int id = inside(w.id[i]) ? w.id[i] : 0;
                return pool + id * page_bytes + (int64_t)(t - page_of(t) * p.page) * tok_bytes;
            } else if constexpr (S::PAGED) {
                const int t16 = min(token0 + (local & ~15), (seq.held - 1) & ~15);
                const int at = w.id[i * S::PER_LOAD / 16], id = inside(at) ? at : 0;
                return pool + (id * page_bytes + (int64_t)(t16 - page_of(t16) * p.page + (local & 15)) * tok_bytes) + in_bytes;
            } else {
                return pool + min(token0 + local + in_load, seq.held - 1) * tok_bytes;
            }
        };
        const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
        // bf16: straight to LDS. e4m3: to registers, and widened into LDS later.
        u32x4 codes[S::F8 ? S::LOADS : 1];
        const uint8_t *const last_row = pool + (seq.held - 1) * tok_bytes;
        struct Addresses {
            const uint8_t *at[S::LOADS];
        };
        auto addresses = [&](const Ids &w, int token0) {
            Addresses all;
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) all.at[i] = address(w, token0, i);
            return all;
        };
        auto load = [&](const Addresses &from, int slot) {
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const uint8_t *const at = from.at[i];
                if constexpr (S::F8) {
                    codes[i] = *reinterpret_cast<const u32x4 *>(at + (16 * run < p.dim ? 16 * run : 0));
                } else {
                    const int r = turned(i);
                    if (r < runs) to_lds(at + r * 16, lds_at + (of_keys ? 0 : S::STAGES * S::MATRIX) + slice * S::LOADS * 1024 + slot + i * 1024);
                }
            }
        };
        auto widen = [&](int slot) {
            if (16 * run >= p.dim) return;
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const int row = slice * S::MINE + i * S::PER_LOAD + in_load, key = of_keys ? key_k(row) : key_v(row);
                uint8_t *const to = lds + (of_keys ? 0 : S::STAGES * S::MATRIX) + slot + row * S::ROW;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t x = codes[i][2 * half], y = codes[i][2 * half + 1];
                    *reinterpret_cast<u32x4 *>(to + ((2 * run + half) ^ key) * 16) =
                        u32x4{bf16_of_e4m3<0>(x), bf16_of_e4m3<1>(x), bf16_of_e4m3<0>(y), bf16_of_e4m3<1>(y)};
                }
            }
        };
        // A tile's tokens on a page outside the pools, a bit each.
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
        constexpr int BAD = !S::PAGED ? 1 : S::EACH ? (TT + 63) / 64 : TT / 16;
        struct Pages {
            int id[BAD];
        };
        auto pages_of = [&](int token0) {  // a tile's page indices, for its bad tokens
            Pages w;
#pragma unroll
            for (int i = 0; i < BAD; ++i) {
                if constexpr (S::EACH) w.id[i] = pages[page_of(min(token0 + 64 * i + lane, seq.held - 1))];
                else if constexpr (S::PAGED) w.id[i] = pages[page_of(min(token0 + 16 * i, (seq.held - 1) & ~15))];
                else w.id[i] = 0;
            }
            return w;
        };
        auto bad_of = [&](const Pages &w) {
            Bad bad;
#pragma unroll
            for (int i = 0; i < (TT + 63) / 64; ++i) {
                bad.bits[i] = 0;
                if constexpr (S::EACH) {
                    bad.bits[i] = __ballot(64 * i + lane < TT && !inside(w.id[i]));
                } else if constexpr (S::PAGED) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (4 * i + j < BAD && !inside(w.id[4 * i + j < BAD ? 4 * i + j : 0])) bad.bits[i] |= 0xFFFFull << (16 * j);
                }
            }
            return bad;
        };
        // The values of tokens that no row sees, past the sequence's last or on such a page, may be anything: they are made zeros
        // in LDS by the wave that loaded them, as 0 times an infinity or a NaN would not hide them.
        auto clear = [&](int token0, const Bad &bad, int slot) {
            if (of_keys || (token0 + TT <= seq.held && !bad.any())) return;
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const int row = slice * S::MINE + i * S::PER_LOAD + in_load;
                if (token0 + row < seq.held && !(S::PAGED && (bad.from(row) & 1))) continue;
                uint8_t *const at = lds + S::STAGES * S::MATRIX + slot + row * S::ROW;
                constexpr int BYTES = S::ROW / S::LANES;  // a lane's share of a row: one run, or two of widened codes
#pragma unroll
                for (int j = 0; j < BYTES; j += 16) *reinterpret_cast<u32x4 *>(at + run * BYTES + j) = u32x4{0, 0, 0, 0};
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        };

        // ---- fragments: the lane's places in a tile ----
        const int wave_token = wt * 32;
        int k_at[4];  // run 2s + h of token c, by s mod 4 (further ones 128 bytes on)
#pragma unroll
        for (int s = 0; s < 4; ++s) k_at[s] = (wave_token + c) * S::ROW + (((2 * s + h) ^ key_k(c)) * 16);
        // Transposed: lanes of 16 take 16 values of 4 tokens. Value part d's run is 4d + 2·(lane / 16 mod 2) + ..., turned.
        const int v_token = 4 * h + (lane & 15) / 4;
        const int v_run = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), v_key = key_v(v_token);
        int v_at[2];  // by d mod 2
#pragma unroll
        for (int d = 0; d < 2; ++d)
            v_at[d] = S::STAGES * S::MATRIX + (wave_token + v_token) * S::ROW + (((4 * d + v_run) ^ v_key) * 16) + 8 * (lane & 1);
        auto keys = [&](int at, int j) { return *reinterpret_cast<const bf16x8 *>(lds + at + k_at[j & 3] + (j >> 2) * 128); };
        // Four tokens of a lane, from `token` + 4h on.
        auto four = [&](int at, int token, int d) {
            const uint8_t *const from = lds + at + v_at[d & 1] + (d >> 1) * 128 + token * S::ROW;
            return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)from));
        };
        auto values = [&](int at, int ks, int d) {
            const u32x2 x = four(at, 16 * ks, d), y = four(at, 16 * ks + 8, d);
            return u32x4{x[0], x[1], y[0], y[1]};
        };

        float top = -INFINITY, sum = 0.0f;
        f32x16 o[DT], s_now, s_next;
        bool wild = false;  // these rows are to be done again by wild_rows
        bool far = false;  // a maximum is so far from 0 that the scaled scores' rounding counts
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

        // The probabilities, two a dword in the order of the second product's tokens, rounded to bf16: by as much of the output as
        // its own rounding is. A second product for what that leaves out costs a third more time (8192 causal tokens 601 and
        // 806 µs, 12 packed prompts 222 and 279); chunks of few rows, which wait for memory, have it.
        struct Weights {
            u32x4 w[2];
        };
        auto pair = [&](const f32x16 &s, Weights &p2, auto ec, float scale, float from) {
            constexpr int e = decltype(ec)::value;
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e], scale, -from));
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e + 1], scale, -from));
            sum += x + y;
            uint32_t both = pack_bf16_rne(x, y);
            asm volatile("" : "+v"(both));  // here, not where it is used
            p2.w[e >> 2][e & 3] = both;
        };
        // The maximum moved, where a score passes it by 8 powers of two. `far`: a maximum is so far from 0 that the scaled scores'
        // rounding, which a fused multiply-add does not share with it, would count: then the scores are taken as their scaled
        // distance from it here.
        auto raise = [&](float m) {
            const uint64_t move = __ballot(m > top + 8.0f);
            float keep = 1.0f;
            if (move) {
                m = fmaxf(over_halves<false>(m), top);
                keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - m);
                top = m;
                sum *= keep;
                far = __any(fabsf(top) > 0x1p24f && fabsf(top) < INFINITY);
            }
            // In place, and past the compiler, which would keep a copy of every sum for the way that leaves them as they are. (They
            // come from matrix instructions: 18 waits before they are read, and some before the next ones take them.)
            if (move)
#pragma unroll
                for (int d = 0; d < DT; ++d)
                asm volatile("s_nop 15\n\ts_nop 1\n\t"
                             "v_mul_f32 %0, %0, %16\n\tv_mul_f32 %1, %1, %16\n\tv_mul_f32 %2, %2, %16\n\tv_mul_f32 %3, %3, %16\n\t"
                             "v_mul_f32 %4, %4, %16\n\tv_mul_f32 %5, %5, %16\n\tv_mul_f32 %6, %6, %16\n\tv_mul_f32 %7, %7, %16\n\t"
                             "v_mul_f32 %8, %8, %16\n\tv_mul_f32 %9, %9, %16\n\tv_mul_f32 %10, %10, %16\n\tv_mul_f32 %11, %11, %16\n\t"
                             "v_mul_f32 %12, %12, %16\n\tv_mul_f32 %13, %13, %16\n\tv_mul_f32 %14, %14, %16\n\tv_mul_f32 %15, %15, %16\n\t"
                             "s_nop 3"
                             : "+v"(o[d][0]), "+v"(o[d][1]), "+v"(o[d][2]), "+v"(o[d][3]), "+v"(o[d][4]), "+v"(o[d][5]), "+v"(o[d][6]),
                               "+v"(o[d][7]), "+v"(o[d][8]), "+v"(o[d][9]), "+v"(o[d][10]), "+v"(o[d][11]), "+v"(o[d][12]), "+v"(o[d][13]),
                               "+v"(o[d][14]), "+v"(o[d][15])
                             : "v"(keep));
        };
        auto largest = [](const f32x16 &s) {
            float m = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) m = fmaxf(m, s[e]);
            return m;
        };
        // Where some row does not see some token of the wave's, or scores are scaled early: the scores as they count, and the largest.
        auto edge = [&](f32x16 &s, float &most, float &scale, int mine, uint32_t bad, int v_from, bool partly) {
            if (capped) {
                const float cap = scalar(p.softcap * LOG2E);
                scale = 1.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = cap * tanh_rel(s[e] * unit_scale);
            } else if (early) {
                scale = 1.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= unit_scale;
            }
            if (!partly) {
                most = largest(s);
                return;
            }
            const int hi_rel = hi - mine - 4 * h, lo_rel = lo - mine - 4 * h;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 8 * (e >> 2) + (e & 3);  // the token, 4h from the wave's
                const bool dead = j > hi_rel || j < lo_rel || (S::PAGED && (bad >> (j + 4 * h) & 1));
                s[e] = dead ? -INFINITY : s[e];
            }
            most = largest(s);
            // A token that some rows do not see may hold an infinity or a NaN, which 0 times it would not hide: wild_rows. (One that all
            // see belongs in their sums.)
            const int past = hi_min - mine, before = lo_max - mine;
            uint32_t unseen = (past < 0 ? ~0u : past < 31 ? ~1u << past : 0u) | (before > 31 ? ~0u : before > 0 ? (1u << before) - 1 : 0u);
            unseen = unseen >> (4 * h);
            uint32_t found = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n) {  // tokens 8n + 4h on
                u32x2 some = {0, 0};
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const u32x2 v = four(v_from, 8 * n, d);
                    some[0] |= unbounded(v[0]);
                    some[1] |= unbounded(v[1]);
                }
                some = some & u32x2{0x80008000u, 0x80008000u};
                found |= (some[0] >> 15 | some[0] >> 30 | some[1] >> 13 | some[1] >> 28) & unseen >> (8 * n) & 15u;
            }
            wild = wild || __any(found != 0);
        };

        // ---- the tiles: beside tile t's softmax run the scores of t + 1 ----
        // At the barrier of tile t all are done with the scores of t and the outputs of t − 1, so the keys of t + STAGES and the values
        // of t + STAGES − 1 are asked for; the keys of t + 2 and the values of t + 1 have come, and those that were asked for at the
        // STAGES − 3 barriers before may be under way. So the first keys of a step are read before its barrier.
        // A tile's slot goes by its number from the run's first, and the loop below is written out for each: the slots' places are
        // then parts of the instructions, and the two sets of scores need no copies.
        auto slot_of = [](int n) { return (n & (S::STAGES - 1)) * S::MATRIX; };
        const int ahead = of_keys ? S::STAGES : S::STAGES - 1;
        // (What a wave writes to LDS it waits for itself; fragments on their way are of tiles that stay.)
        auto barrier = [] { asm volatile("s_barrier" ::: "memory"); };
        auto written = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
        int t = t_from;
        Ids ids = {};            // of the tile after the one whose
        Addresses asked = {};    // addresses these are: what the next barrier asks for
        Pages tile_pages = {}, next_pages = {};
        constexpr int LEAD = 4, OUTS = 2 * DT;  // reads go this many instructions ahead
        float most = -INFINITY;                 // of the scores at hand
        bf16x8 k[LEAD];
        auto first_keys = [&](auto nc) {  // of the step of slot n
            static_for<0, LEAD>([&](auto jc) { k[decltype(jc)::value] = keys(slot_of(decltype(nc)::value + 1), decltype(jc)::value); });
        };
        static_assert(S::STAGES == 4, "a step for each");
        auto step = [&](auto nc, f32x16 &s, f32x16 &next) {
            constexpr int n = decltype(nc)::value;
            const Bad bad = bad_of(tile_pages);
            tile_pages = next_pages;
            if constexpr (!S::F8) {
                if (t + S::STAGES > t_to) wd::wait_vmcnt<0>();
                else wd::wait_vmcnt<(S::STAGES - 3) * S::LOADS>();
            }
            clear(base + t * TT, bad, slot_of(n));
            if constexpr (S::F8) written();
            barrier();
            if (t + ahead < t_to) load(asked, of_keys ? slot_of(n + S::STAGES) : slot_of(n + S::STAGES - 1));
            const int k_from = slot_of(n + 1), v_from = slot_of(n);
            const int mine = base + t * TT + wave_token;  // the wave's first token
            float scale = unit_scale;
            const bool partly = mine + 31 > hi_min || mine < lo_max || bad.any();
            if (early || partly) edge(s, most, scale, mine, (uint32_t)bad.from(wave_token), v_from, partly);
            raise(most * scale);
            float from = top == -INFINITY ? 0.0f : top;
            if (far) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = s[e] * scale - from;
                scale = 1.0f;
                from = 0.0f;
            }
            // Written out in the order it runs, reads LEAD instructions ahead: between the matrix instructions of the next scores the
            // softmax, two values each; then the outputs, and between them the largest of the next scores and what the next
            // barrier asks for. (The last tile's next one is whatever lies there.)
            Weights p2;
            bf16x8 v[LEAD];
#pragma unroll
            for (int e = 0; e < 16; ++e) next[e] = 0.0f;
            __builtin_amdgcn_sched_barrier(0);
            static_for<0, STEPS>([&](auto jc) {
                constexpr int j = decltype(jc)::value;
                next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[j % LEAD], q[j], next, 0, 0, 0);
                if constexpr (j + LEAD < STEPS) k[j % LEAD] = keys(k_from, j + LEAD);
                else v[j + LEAD - STEPS] = __builtin_bit_cast(bf16x8, values(v_from, (j + LEAD - STEPS) / DT, (j + LEAD - STEPS) % DT));
                static_for<8 * j / STEPS, 8 *(j + 1) / STEPS>([&](auto ec) { pair(s, p2, ec, scale, from); });
                __builtin_amdgcn_sched_barrier(0);
            });
            // (Past the last tile: the last token's.) Rows of a projection lie a tile's bytes on, the last token's at most.
            if constexpr (S::PAGED) asked = addresses(ids, base + (t + 1 + ahead) * TT);
            else
#pragma unroll
                for (int i = 0; i < S::LOADS; ++i) asked.at[i] = std::min(asked.at[i] + TT * tok_bytes, last_row);
            // Here, not where it is used.
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) asm volatile("" : "+v"(asked.at[i]));
            ids = look_up(base + (t + 2 + ahead) * TT);
            next_pages = pages_of(base + (t + 2) * TT);
            static_for<0, OUTS>([&](auto jc) {
                constexpr int i = decltype(jc)::value;
                o[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[i % LEAD], __builtin_bit_cast(bf16x8, p2.w[i / DT]), o[i % DT], 0, 0, 0);
                if constexpr (i + LEAD < OUTS) v[i % LEAD] = __builtin_bit_cast(bf16x8, values(v_from, (i + LEAD) / DT, (i + LEAD) % DT));
                if constexpr (i == 0) most = -INFINITY;
                else static_for<16 * (i - 1) / (OUTS - 1), 16 * i / (OUTS - 1)>([&](auto ec) { most = fmaxf(most, next[decltype(ec)::value]); });
                asm volatile("" : "+v"(most));
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (S::F8) {
                if (t + ahead < t_to) widen(of_keys ? slot_of(n + S::STAGES) : slot_of(n + S::STAGES - 1));
            }
            ++t;
            first_keys(std::integral_constant<int, n + 1>{});
        };
        if (t < t_to) {
            __syncthreads();  // the run before has been read
            if (SHARE && DP <= 128 && pos != start) clear_ends();
            for (int i = t; i < min(t + ahead, t_to); ++i) {
                load(addresses(look_up(base + i * TT), base + i * TT), slot_of(i - t));
                if constexpr (S::F8) widen(slot_of(i - t));
            }
            asked = addresses(look_up(base + (t + ahead) * TT), base + (t + ahead) * TT);
            ids = look_up(base + (t + 1 + ahead) * TT);
            tile_pages = pages_of(base + t * TT);
            next_pages = pages_of(base + (t + 1) * TT);
            if constexpr (!S::F8) wd::wait_vmcnt<0>();
            written();
            barrier();
            first_keys(std::integral_constant<int, 0>{});
            if (minus) {  // (here, where the rows have come)
#pragma unroll
                for (int j = 0; j < STEPS; ++j)
                    q[j] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, q[j]) ^ u32x4{0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u});
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s_now[e] = 0.0f;
#pragma unroll
            for (int j = 0; j < STEPS; ++j) s_now = __builtin_amdgcn_mfma_f32_32x32x16_bf16(keys(slot_of(0), j), q[j], s_now, 0, 0, 0);
            most = largest(s_now);
            for (;;) {
                step(std::integral_constant<int, 0>{}, s_now, s_next);
                if (t >= t_to) break;
                step(std::integral_constant<int, 1>{}, s_next, s_now);
                if (t >= t_to) break;
                step(std::integral_constant<int, 2>{}, s_now, s_next);
                if (t >= t_to) break;
                step(std::integral_constant<int, 3>{}, s_next, s_now);
                if (t >= t_to) break;
            }
        }

        // ---- the waves of a row joined, by the first ----
        sum = over_halves<true>(sum);
        if constexpr (WT > 1) {
            __syncthreads();  // the last tile has been read
            float *const mine = reinterpret_cast<float *>(lds) + ((wt - 1) * WM + wm) * (DT * 16 * 64) + lane;
            if (h == 0) { tops[wave][c] = top; totals[wave][c] = sum; }
            if (lane == 0) wilds[wave] = wild;
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
#pragma unroll
                for (int i = 1; i < WT; ++i) wild = wild || wilds[i * WM + wm] != 0;
            }
        }
        const bool whole = !SHARE || numbered == units.run;
        if (WT == 1 && DP <= 128 && whole) __syncthreads();  // the last tile has been read
        if (wt == 0) {
            if (whole) {
                const float by = inverse(sum) * (S::F8 && p.v_scale ? p.v_scale[kvh] : 1.0f);
                if constexpr (DP > 128) {
                    // As they lie: the way below takes registers that spill (8192 tokens of 16 heads of 256, 976 and 923 µs).
                    if (live) {
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
                    // By way of LDS (a place of the wave's own), so that rows are written in whole runs: written as they lie, 16 bytes a row
                    // and instruction, they took 1.5 µs of a unit.
                    uint8_t *const mine = lds + (WT > 1 ? S::STAGES * S::MATRIX : 0) + wm * 32 * S::ROW;
                    auto key = [](int row) { return row & (S::RUNS < 16 ? S::RUNS - 1 : 15); };
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<u32x2 *>(mine + c * S::ROW + ((4 * d + e / 4) ^ key(c)) * 16 + 8 * h) =
                                u32x2{pack_bf16_rne(o[d][e] * by, o[d][e + 1] * by), pack_bf16_rne(o[d][e + 2] * by, o[d][e + 3] * by)};
                    const int w_tok = w0 / p.group, w_head = w0 - w_tok * p.group;  // of the wave's first row
                    const float per = 1.0f / (float)p.group;
                    const int run = lane % S::RUNS;
#pragma unroll
                    for (int i = 0; i < S::RUNS / 2; ++i) {
                        const int row = i * (64 / S::RUNS) + lane / S::RUNS;
                        const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + row * S::ROW + (run ^ key(row)) * 16);
                        if (w0 + row >= rows || run >= runs) continue;
                        // (w_head + row) / group: small numbers, or the next token at most.
                        const int x = w_head + row, next = p.group >= 32 ? (x >= p.group ? 1 : 0) : (int)(((float)x + 0.5f) * per);
                        uint16_t *const dst = p.out + (int64_t)(seq.row0 + w_tok + next) * p.o_tok + (int64_t)(kvh * p.group + x - next * p.group) * p.o_head;
                        *reinterpret_cast<u32x4_any *>(dst + 8 * run) = v;
                    }
                }
            } else {
                float *const slot = p.part + (int64_t)(2 * blockIdx.x + (pos == start ? 0 : 1)) * attend_part_floats(DP, M);
                if (h == 0) put(slot + 2 * (wm * 32 + c), Pair{top, sum});
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        put(slot + 2 * M + 2 * (((wm * DT + d) * 8 + e / 2) * 64 + lane), Pair{o[d][e], o[d][e + 1]});
            }
        }
        if (wt == 0 && __builtin_amdgcn_readfirstlane((int)wild)) {
            const int64_t head0 = (int64_t)kvh * p.group;
            const WildRows again = {p.q + seq.row0 * p.q_tok + head0 * p.q_head, p.out + seq.row0 * p.o_tok + head0 * p.o_head,
                                    p.kc + (kvh * p.kc_head + (S::PAGED ? 0 : seq.row0 * p.kc_tok)) * ES,
                                    p.vc + (kvh * p.vc_head + (S::PAGED ? 0 : seq.row0 * p.vc_tok)) * ES,
                                    S::PAGED ? p.pages + b * p.pages_row : nullptr,
                                    whole ? nullptr : p.part + (int64_t)(2 * blockIdx.x + (pos == start ? 0 : 1)) * attend_part_floats(DP, M),
                                    p.q_tok, p.q_head, p.o_tok, p.o_head, p.kc_page * ES, p.kc_tok * ES, p.vc_page * ES, p.vc_tok * ES,
                                    p.page_mul, minus ? -unit_scale : unit_scale, capped ? p.softcap * LOG2E : 0.0f,
                                    S::F8 && p.v_scale ? p.v_scale[kvh] : 1.0f, p.page_shift, p.page, p.page_count, row0 + 32 * wm, min(row0 + 32 * wm + 32, rows), p.group,
                                    p.dim, first, seq.held, windowed ? p.window : 0, p.causal, base + t_from * TT, min(base + t_to * TT, seq.held)};
            wild_rows<DP, S::F8>(again, [&](int r) { return 2 * (r - row0); }, [&](int r, int x) {
                const int c = (r - row0) & 31, d = x >> 5, e = 4 * (x >> 3 & 3) + (x & 3), half = x >> 2 & 1;
                return 2 * M + 2 * (((wm * DT + d) * 8 + e / 2) * 64 + c + 32 * half) + (e & 1);
            });
        }
        if (SHARE && !whole && tid == 0)
            parts[pos == start ? 0 : 1] = Part{seq0 + unit * units.run, units.run, row0, rows, kvh, seq.row0};
        pos += numbered;
    }

    // ---- the parts' slots are written before their counters say so; the last workgroup to count joins ----
    if constexpr (!SHARE) return;
    __syncthreads();
    join_parts<M, DP, S::THREADS, S::F8>(p, share, parts, joins, [](int item, int &row, int &at) {
        const int l = item & 63, e = 2 * (item >> 6 & 7), d = (item >> 9) % DT, set = (item >> 9) / DT;
        row = 32 * set + (l & 31);
        at = 32 * d + 8 * (e >> 2) + 4 * (l >> 5) + (e & 3);
    });
}

}  // namespace attend
}  // namespace sq8
