// sq8_chunk.hip — attention of chunks of few new tokens over a paged cache: the formula of sq8_attend_kernel.h, in the manner of
// the attention of one new token (sq8_paged.hip).
//
// Bound by the cache's bytes. The rows of a tile, (token, query head) pairs of one kv head with the head running fastest, are the
// columns of both products, 16 · NC of them, on v_mfma_f32_16x16x32_bf16:
//   S[token, row] = K · Qᵀ   (first operand: 16 tokens × 32 values)
//   O[value, row] += Vᵀ · P  (first operand: 16 values × 32 tokens)
// A lane (c = lane mod 16, h = lane / 16) ends with S of tokens 4h .. 4h + 3 of each 16 for rows 16n + c, and the second product
// takes its 32 tokens in the order (4h + r of the first 16, 4h + r of the second): the probabilities are its operand as they
// lie, and keys and values go from memory to registers in whole rows, without LDS, values transposed within a lane (DV · c + i to
// instruction i). Keys and values are read once for all 16 · NC rows.
//
// A tile is 128 tokens, 32 a wave; the tiles of all units are shared out evenly, and units that several workgroups have are joined
// by the last (sq8_attend_device.h). Softmax in fp32, its maximum moved only past 8 powers of two; probabilities in two bf16
// parts, which leave out 2^-16 of one at most. A new token's rows see different tokens: only tiles at the ends of what they see
// compare places, and a value there that some rows do not see is looked over for infinities and NaN (wild_rows).
//
// 32 sequences of 4 new tokens behind ragged contexts of up to 8192, 32 heads on 8 of 128 in e4m3 (287 MB), take 81 µs, 3.5 TB/s
// (69 from the last cache level), of which some ten are the start and the join; 32 of 8 behind 8192 in bf16 (1074 MB) 263, 4.1 TB/s;
// 16 tokens of one sequence behind 500 12.1 µs, a chain of latencies (with tiles of 64 rows 26: a quarter of the workgroups, and
// four times the join). Before, tiles of 64 rows in LDS took 170 and 33 for the first and the last. How many rows share what is read: sq8_text_plan.hip.
// A row's lookups of pages that 16 tokens do not fill cost 5 to 10 % more.
#include "sq8_attend_device.h"

namespace sq8 {
namespace attend {
namespace {

constexpr int WAVES = 4, TILE = 32 * WAVES;

template <int DP, int NC, bool E4M3, bool PAGE16>
__global__ void __launch_bounds__(64 * WAVES, chunk_held(DP, NC)) chunk_kernel(const AttendArgs p) {
    constexpr int ES = E4M3 ? 1 : 2, M = 16 * NC;
    constexpr int STEPS = DP / 32;            // instructions of 16 tokens' scores
    constexpr int KRUNS = DP * ES / 64;       // 16-byte runs of a key a lane reads
    constexpr int DV = DP / 16;               // values of a token a lane reads: instructions of the second product
    constexpr int VN = DV * ES / 4;           // and their dwords
    constexpr float LOG2E = 1.4426950408889634f;
    __shared__ __attribute__((aligned(16))) f32x4 joined[WAVES - 1][NC][DV][64];
    __shared__ float tops[WAVES][M], totals[WAVES][M];
    __shared__ int joins[2], wilds[WAVES];
    __shared__ Part parts[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, h = lane >> 4;
    const bool full = p.dim == DP, capped = p.softcap > 0.0f;
    // The bytes of a row a lane reads (past `dim`, the row's first), and PAGE16: with its row's place from the 16 tokens' first.
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

    int upto = 0;
    const int total = all_units<M, TILE, true>(p, lane, upto) * p.kv_heads;
    const Share share(total, gridDim.x);
    const int start = share.first(min((int)blockIdx.x, share.groups)), end = share.first(min((int)blockIdx.x + 1, share.groups));
    if (start >= end) return;
    int b, before;
    find_unit<M, TILE, true>(p, start, lane, upto, b, before);
    int seq0 = before * p.kv_heads;
    Sequence seq;
    Units units;
    auto enter = [&]() {
        const Sequence s = sequence(p, b);
        seq.row0 = __builtin_amdgcn_readfirstlane(s.row0);
        seq.count = __builtin_amdgcn_readfirstlane(s.count);
        seq.held = __builtin_amdgcn_readfirstlane(s.held);
        units = units_of<M, TILE, true>(p, seq);
    };
    enter();
    if (tid < 2) parts[tid].tiles = 0;

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
        const int numbered = min(units.run - part0, end - pos);
        const int rows = seq.count * p.group, row0 = tile * M;
        const int first = seq.held - seq.count;  // the place of the chunk's first token

        // ---- the tokens that these rows see ----
        const int tok0 = row0 / p.group, tokN = (min(row0 + M, rows) - 1) / p.group;
        const bool windowed = p.causal && p.window > 0;
        auto last_of = [&](int tok) { return p.causal ? min(first + tok, seq.held - 1) : seq.held - 1; };
        auto first_of = [&](int tok) { return windowed ? first + tok - p.window + 1 : 0; };
        const int hi_min = last_of(tok0), hi_max = last_of(tokN), lo_min = max(first_of(tok0), 0), lo_max = first_of(tokN);
        const int base = lo_min & ~15;
        const int tiles = max(0, (hi_max + 1 - base + TILE - 1) / TILE);
        const int t_from = min(part0, tiles), t_to = min(part0 + numbered, tiles);

        // ---- the rows: row 16n + c's values in the order the keys' lanes hold them ----
        bf16x8 q[NC][STEPS];
        int toks[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int r = min(row0 + 16 * n + c, rows - 1), head = r % p.group;
            toks[n] = r / p.group;
            const uint16_t *const from = p.q + (int64_t)(seq.row0 + toks[n]) * p.q_tok + (int64_t)(kvh * p.group + head) * p.q_head;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int d = E4M3 ? 64 * (s >> 1) + 16 * h + 8 * (s & 1) : 32 * s + 8 * h;
                u32x4 v = {0, 0, 0, 0};
                if (d < p.dim) v = *reinterpret_cast<const u32x4 *>(from + d);
                q[n][s] = __builtin_bit_cast(bf16x8, v);
            }
        }
        // Scores in units of log2, or where they are capped, in those of the cap.
        const float score_scale = p.scale * (E4M3 && p.k_scale ? p.k_scale[kvh] : 1.0f) * (capped ? 1.0f / p.softcap : LOG2E);
        const uint8_t *const kbase = p.kc + (int64_t)kvh * p.kc_head * ES;
        const uint8_t *const vbase = p.vc + (int64_t)kvh * p.vc_head * ES;
        // Read as constant memory: scalar loads, for which the vector loads under way need not be waited for.
        const auto pages = (const __attribute__((address_space(4))) int32_t *)(p.pages + (int64_t)b * p.pages_row);
        auto page_of = [&](int token) { return (int)(((uint64_t)(uint32_t)token * p.page_mul) >> p.page_shift); };
        auto inside = [&](int id) { return (unsigned)id < (unsigned)p.page_count; };

        // The pages of a wave's 32 tokens, by their indices as read. PAGE16: each 16 tokens lie in one page, whose index is uniform
        // and read one tile before its use. Else each lane looks up its own tokens': of its two keys, of its eight values.
        constexpr int IDS = PAGE16 ? 2 : 10;
        struct Where {
            int id[IDS];
        };
        auto token_of = [&](int token, int i) {  // i < 2: a key's, else a value's
            const int t = i < 2 ? 16 * i + (PAGE16 ? 0 : c) : 16 * ((i - 2) >> 2) + 4 * h + ((i - 2) & 3);
            return min(token + t, PAGE16 ? (seq.held - 1) & ~15 : seq.held - 1);
        };
        auto locate = [&](int token) {
            Where w;
#pragma unroll
            for (int i = 0; i < IDS; ++i) w.id[i] = pages[page_of(token_of(token, i))];
            return w;
        };
        auto row_of = [&](const Where &w, int token, int i, int64_t page_stride, int64_t tok_stride) {
            const int t = token_of(token, i);
            return (inside(w.id[i]) ? w.id[i] : 0) * page_stride + (t - page_of(t) * p.page) * tok_stride;
        };
        // Tokens on a page outside the pools, in the order of the lane's eight.
        auto bad_of = [&](const Where &w) {
            if constexpr (PAGE16) return (inside(w.id[0]) ? 0u : 0x0Fu) | (inside(w.id[1]) ? 0u : 0xF0u);
            uint32_t bad = 0;
#pragma unroll
            for (int i = 2; i < IDS; ++i) bad |= inside(w.id[i]) ? 0u : 1u << (i - 2);
            return bad;
        };
        Raw<4> k[2][KRUNS];
        auto load_k = [&](const Where &w, int token) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint8_t *const row = kbase + row_of(w, token, t, p.kc_page, p.kc_tok) * ES;
#pragma unroll
                for (int s = 0; s < KRUNS; ++s) k[t][s] = load_raw<4>(row + (PAGE16 ? k_lane[s] : k_run[s]));
            }
        };
        Raw<VN> v[8];
        auto load_v = [&](const Where &w, int token) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = load_raw<VN>(vbase + row_of(w, token, PAGE16 ? i >> 2 : i + 2, p.vc_page, p.vc_tok) * ES + (PAGE16 ? v_lane[i & 3] : v_run));
        };
        // Values d and d + 1 of the lane's eight tokens, two tokens a dword.
        auto transposed = [&](int d, u32x4 (&t)[2]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t x = v[2 * j].d[d / (4 / ES)], y = v[2 * j + 1].d[d / (4 / ES)];
                if constexpr (E4M3) {
                    // bytes (x[d], y[d], x[d + 1], y[d + 1]), then as bf16
                    const uint32_t four = __builtin_amdgcn_perm(y, x, d & 2 ? 0x07030602u : 0x05010400u);
                    t[0][j] = bf16_of_e4m3<0>(four);
                    t[1][j] = bf16_of_e4m3<1>(four);
                } else {
                    t[0][j] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                    t[1][j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                }
            }
        };

        bool wild = false;  // these rows are to be done again by wild_rows
        float top[NC], sum[NC];  // of row 16n + c, in units of log2: the sum over this lane's tokens
        f32x4 o[NC][DV];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            top[n] = -INFINITY;
            sum[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < DV; ++i) o[n][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        // One tile, and the loads of the next: the keys' once the scores are done with this one's, the values' after the second
        // product. A run's last one loads nothing.
        int token = base + t_from * TILE + wave * 32;
        uint32_t bad = 0;  // of the tile at hand
        Where next;
        auto subtile = [&](auto last) {
            constexpr bool more = !decltype(last)::value;
            f32x4 s[NC][2] = {};
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
#pragma unroll
                    for (int n = 0; n < NC; ++n) s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[n][j], s[n][t], 0, 0, 0);
                }
            if (more) load_k(next, token + TILE);
            const Where later = more ? locate(token + 2 * TILE) : next;

            auto at = [&](int j) { return token + 16 * (j >> 2) + 4 * h + (j & 3); };  // token j of the lane's eight
            const bool edge = token < lo_max || token + 31 > hi_min || (PAGE16 ? bad != 0 : __any(bad != 0));
            if (edge) {
                // A token that no row sees may hold anything, and 0 · NaN is one: its values are zeros. One that some rows see may
                // hold an infinity or a NaN, which the others must not meet: wild_rows.
                uint32_t found = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = at(j);
                    const bool dead = t < lo_min || t > hi_max || (bad >> j & 1), some = t < lo_max || t > hi_min;
#pragma unroll
                    for (int d = 0; d < VN; ++d) {
                        v[j].d[d] = dead ? 0 : v[j].d[d];
                        const uint32_t none = E4M3 ? ((v[j].d[d] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u : unbounded(v[j].d[d]) & 0x80008000u;
                        found |= some ? none : 0u;
                    }
                }
                wild = wild || __any(found != 0);
            }
            bf16x8 prob[NC][2];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = s[n][j >> 2][j & 3] * score_scale;
                if (capped) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = p.softcap * LOG2E * tanh_rel(e[j]);
                }
                // What is left of a probability beside its first part is at least 2^-126, so that an infinite value meets no zero and no
                // other sign; but of a token that the row does not see it is 0.
                float least[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) least[j] = 0x1p-126f;
                if (edge) {
                    const int hi = last_of(toks[n]), lo = first_of(toks[n]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int t = at(j);
                        const bool dead = t < lo || t > hi || (bad >> j & 1);
                        e[j] = dead ? -INFINITY : e[j];
                        least[j] = dead ? 0.0f : least[j];
                    }
                }
                float m = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
                if (__any(m > top[n] + 8.0f)) {
                    m = fmaxf(over_rows<false>(m), top[n]);
                    const float keep = top[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[n] - m);
                    top[n] = m;
                    sum[n] *= keep;
#pragma unroll
                    for (int d = 0; d < DV; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[n][d][r] *= keep;
                }
                const float from = top[n] == -INFINITY ? 0.0f : top[n];
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(e[j] - from);
                sum[n] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                u32x4 part[2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = __float_as_uint(w[2 * j]), y = __float_as_uint(w[2 * j + 1]);
                    part[0][j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    part[1][j] = pack_bf16_rne(fmaxf(w[2 * j] - __uint_as_float(x & 0xFFFF0000u), least[2 * j]),
                                               fmaxf(w[2 * j + 1] - __uint_as_float(y & 0xFFFF0000u), least[2 * j + 1]));
                }
                prob[n][0] = __builtin_bit_cast(bf16x8, part[0]);
                prob[n][1] = __builtin_bit_cast(bf16x8, part[1]);
            }
#pragma unroll
            for (int d = 0; d < DV; d += 2) {
                u32x4 t[2];
                transposed(d, t);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int n = 0; n < NC; ++n)
#pragma unroll
                        for (int j = 1; j >= 0; --j)
                            o[n][d + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t[i]), prob[n][j], o[n][d + i], 0, 0, 0);
            }
            if (more) load_v(next, token + TILE);
            bad = bad_of(next);
            next = later;
            token += TILE;
        };
        if (t_from < t_to) {
            const Where now = locate(token);
            load_k(now, token);
            load_v(now, token);
            bad = bad_of(now);
            next = locate(token + TILE);
            for (int i = t_from + 1; i < t_to; ++i) subtile(std::false_type{});
            subtile(std::true_type{});
        }

        // ---- the waves' results joined, by the first ----
#pragma unroll
        for (int n = 0; n < NC; ++n) sum[n] = over_rows<true>(sum[n]);
        __syncthreads();  // the run before has been read
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            if (h == 0) { tops[wave][16 * n + c] = top[n]; totals[wave][16 * n + c] = sum[n]; }
            if (wave > 0) {
#pragma unroll
                for (int d = 0; d < DV; ++d) joined[wave - 1][n][d][lane] = o[n][d];
            }
        }
        if (lane == 0) wilds[wave] = wild;
        __syncthreads();
        const bool whole = numbered == units.run;
        if (wave == 0) {
            float *const slot = p.part + (int64_t)(2 * blockIdx.x + (pos == start ? 0 : 1)) * attend_part_floats(DP, M);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                float all = top[n];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) all = fmaxf(all, tops[w][16 * n + c]);
                const float from = all == -INFINITY ? 0.0f : all;
                float weight = __builtin_amdgcn_exp2f(top[n] - from);
                float l = sum[n] * weight;
#pragma unroll
                for (int d = 0; d < DV; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[n][d][r] *= weight;
#pragma unroll
                for (int w = 1; w < WAVES; ++w) {
                    weight = __builtin_amdgcn_exp2f(tops[w][16 * n + c] - from);
                    l += totals[w][16 * n + c] * weight;
#pragma unroll
                    for (int d = 0; d < DV; ++d) {
                        const f32x4 t = joined[w - 1][n][d][lane];
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[n][d][r] = __builtin_fmaf(t[r], weight, o[n][d][r]);
                    }
                }
                const int row = row0 + 16 * n + c;
                if (row < rows) {
                    if (whole) {
                        const float by = inverse(l) * (E4M3 && p.v_scale ? p.v_scale[kvh] : 1.0f);
                        uint16_t *const dst = p.out + (int64_t)(seq.row0 + toks[n]) * p.o_tok + (int64_t)(kvh * p.group + row % p.group) * p.o_head;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int x = DV * (4 * h + r);
                            if (x >= p.dim) continue;
#pragma unroll
                            for (int d = 0; d < DV; d += 2)
                                *reinterpret_cast<uint32_t *>(dst + x + d) = pack_bf16_rne(o[n][d][r] * by, o[n][d + 1][r] * by);
                        }
                    } else {
                        if (h == 0) put(slot + 2 * (16 * n + c), Pair{all, l});
#pragma unroll
                        for (int d = 0; d < DV; d += 2)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                put(slot + 2 * M + 2 * (((n * (DV / 2) + d / 2) * 4 + r) * 64 + lane), Pair{o[n][d][r], o[n][d + 1][r]});
                    }
                }
            }
        }
        if (wave == 0 && __builtin_amdgcn_readfirstlane(wilds[0] | wilds[1] | wilds[2] | wilds[3])) {
            const int64_t head0 = (int64_t)kvh * p.group;
            const WildRows again = {p.q + seq.row0 * p.q_tok + head0 * p.q_head, p.out + seq.row0 * p.o_tok + head0 * p.o_head, kbase, vbase,
                                    p.pages + b * p.pages_row,
                                    whole ? nullptr : p.part + (int64_t)(2 * blockIdx.x + (pos == start ? 0 : 1)) * attend_part_floats(DP, M),
                                    p.q_tok, p.q_head, p.o_tok, p.o_head, p.kc_page * ES, p.kc_tok * ES, p.vc_page * ES, p.vc_tok * ES,
                                    p.page_mul, score_scale, capped ? p.softcap * LOG2E : 0.0f, E4M3 && p.v_scale ? p.v_scale[kvh] : 1.0f,
                                    p.page_shift, p.page, p.page_count, row0, min(row0 + M, rows), p.group, p.dim, first, seq.held,
                                    windowed ? p.window : 0, p.causal, base + t_from * TILE, min(base + t_to * TILE, seq.held)};
            wild_rows<DP, E4M3>(again, [&](int r) { return 2 * (r - row0); }, [&](int r, int x) {
                const int n = (r - row0) >> 4, column = (r - row0) & 15, d = x % DV, y = x / DV;
                return 2 * M + 2 * (((n * (DV / 2) + d / 2) * 4 + (y & 3)) * 64 + column + 16 * (y >> 2)) + (d & 1);
            });
        }
        if (!whole && tid == 0) parts[pos == start ? 0 : 1] = Part{seq0 + unit * units.run, units.run, row0, rows, kvh, seq.row0};
        pos += numbered;
    }

    // The parts' slots are written (by the first wave) before their counters say so; the last to count joins.
    __syncthreads();
    join_parts<M, DP, 64 * WAVES, E4M3>(p, share, parts, joins, [](int item, int &row, int &at) {
        const int l = item & 63, r = item >> 6 & 3, d = 2 * ((item >> 8) % (DV / 2)), n = (item >> 8) / (DV / 2);
        row = 16 * n + (l & 15);
        at = DV * (4 * (l >> 4) + r) + d;
    });
}

// Whether 16 tokens lie in one page each, and a lane's offsets within one in 32 bits.
bool by_pages(const AttendArgs &p) { return p.page % 16 == 0 && 32 * (p.kc_tok > p.vc_tok ? p.kc_tok : p.vc_tok) <= INT32_MAX; }

template <int DP, int NC>
hipError_t launch(const AttendArgs &p, int groups, bool e4m3, hipStream_t stream) {
    const dim3 grid(groups), block(64 * WAVES);
    if (by_pages(p)) {
        if (e4m3) hipLaunchKernelGGL((chunk_kernel<DP, NC, true, true>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((chunk_kernel<DP, NC, false, true>), grid, block, 0, stream, p);
    } else {
        if (e4m3) hipLaunchKernelGGL((chunk_kernel<DP, NC, true, false>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((chunk_kernel<DP, NC, false, false>), grid, block, 0, stream, p);
    }
    return hipGetLastError();
}

template <int DP>
hipError_t pick(const AttendArgs &p, const AttendPlan &plan, bool e4m3, hipStream_t stream) {
    if (plan.rows == 16) return launch<DP, 1>(p, plan.groups, e4m3, stream);
    if (plan.rows == 32) return launch<DP, 2>(p, plan.groups, e4m3, stream);
    if constexpr (DP <= 128)
        if (plan.rows == 64) return launch<DP, 4>(p, plan.groups, e4m3, stream);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_chunk(const AttendArgs &p, const AttendPlan &plan, bool e4m3, hipStream_t stream) {
    switch (attend_dim(p.dim)) {
        case 64: return pick<64>(p, plan, e4m3, stream);
        case 128: return pick<128>(p, plan, e4m3, stream);
        default: return pick<256>(p, plan, e4m3, stream);
    }
}

}  // namespace attend
}  // namespace sq8
