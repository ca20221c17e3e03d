// sq8_attend_device.h — what the kernels of prompt and chunk attention share: the sequences' rows and tiles, how tiles are
// shared out over the workgroups, and the join of the parts of a unit that several of them had.
#pragma once

#include <hip/hip_runtime.h>

#include "sq8_device.h"
#include "sq8_text.h"
#include "sq8_text_device.h"
#include "sq8_wdirect_kernel.h"

namespace sq8 {
namespace attend {

// Bits 15 and 31: whether that bf16 of a pair is an infinity or a NaN. (Other bits: anything.)
__device__ __forceinline__ uint32_t unbounded(uint32_t d) { return (d & 0x7F807F80u) + 0x00800080u; }

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

// Units of a sequence: a tile of rows by a kv head, the head running fastest. Shared out (SHARE), each has as many tiles of
// keys as the sequence's longest.
struct Units {
    int tiles;   // of rows
    int run;     // tiles of keys of a unit that are numbered: 1 unless shared
};
template <int M, int TT, bool SHARE>
__device__ __forceinline__ Units units_of(const AttendArgs &p, const Sequence &s) {
    Units u;
    u.tiles = (int)(((int64_t)s.count * p.group + M - 1) / M);
    int base = 0;
    if (p.causal && p.window > 0) base = max(0, s.held - s.count - p.window + 1) & ~15;
    u.run = SHARE ? max(1, (s.held - base + TT - 1) / TT) : 1;
    return u;
}

// Rows of which some, but not all, see a token whose value is an infinity or a NaN, done again by one wave without the matrix
// cores, whose sums take in every token of a tile: a row at a time, 64 tokens a step, those that it sees.
struct WildRows {
    const uint16_t *q;
    uint16_t *out;
    const uint8_t *k, *v;       // the kv head's
    const int32_t *pages;       // or null
    float *slot;                // for a part of a unit; else null
    int64_t q_tok, q_head, o_tok, o_head, k_page, k_tok, v_page, v_tok;  // keys' and values' in bytes
    uint64_t page_mul;
    float scale, cap, v_scale;  // in units of log2; cap 0: none
    int page_shift, page, page_count, row0, rows, group, dim, first, held, window, causal, from, to;  // rows [row0, rows)
};
// `pair_at`, `value_at`: where in the slot a row's maximum and sum lie, and a value of it.
template <int DP, bool F8, class PairAt, class ValueAt>
__device__ __forceinline__ void wild_rows(const WildRows &w, PairAt pair_at, ValueAt value_at) {
    constexpr int N = DP / 64;  // values of a lane
    const int lane = threadIdx.x & 63;
    auto row_of = [&](int t, int64_t page_bytes, int64_t tok_bytes, bool &bad) -> int64_t {
        bad = false;
        if (!w.pages) return t * tok_bytes;
        const int page = (int)(((uint64_t)(uint32_t)t * w.page_mul) >> w.page_shift);
        int id = w.pages[page];
        bad = (unsigned)id >= (unsigned)w.page_count;
        return (bad ? 0 : id) * page_bytes + (int64_t)(t - page * w.page) * tok_bytes;
    };
    auto value = [&](const uint8_t *at, int i) { return F8 ? widen1<W_FP8>(at[i]) : bf16_f32(reinterpret_cast<const uint16_t *>(at)[i]); };
    for (int r = w.row0; r < w.rows; ++r) {
        const int tok = r / w.group, head = r - tok * w.group;
        const uint16_t *const q = w.q + tok * w.q_tok + head * w.q_head;
        const int hi = min(w.causal ? min(w.first + tok, w.held - 1) : w.held - 1, w.to - 1);
        const int lo = max(w.window > 0 ? w.first + tok - w.window + 1 : 0, w.from);
        float top = -INFINITY, sum = 0.0f, o[N] = {};
        for (int t0 = lo; t0 <= hi; t0 += 64) {
            bool bad;
            const uint8_t *const k = w.k + row_of(min(t0 + lane, hi), w.k_page, w.k_tok, bad);
            float s = 0.0f;
            for (int i = 0; i < w.dim; ++i) s = __builtin_fmaf(bf16_f32(q[i]), value(k, i), s);
            s *= w.scale;
            if (w.cap > 0.0f) s = w.cap * tanh_rel(s);
            if (bad || t0 + lane > hi) s = -INFINITY;
            float m = s;
#pragma unroll
            for (int i = 32; i >= 1; i >>= 1) m = fmaxf(m, __shfl_xor(m, i, 64));
            m = fmaxf(m, top);
            const float from = m == -INFINITY ? 0.0f : m, keep = __builtin_amdgcn_exp2f(top - from);
            top = m;
            float p = __builtin_amdgcn_exp2f(s - from), all = p;
#pragma unroll
            for (int i = 32; i >= 1; i >>= 1) all += __shfl_xor(all, i, 64);
            sum = sum * keep + all;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] *= keep;
            for (int j = 0; j < 64 && t0 + j <= hi; ++j) {
                const uint8_t *const v = w.v + row_of(t0 + j, w.v_page, w.v_tok, bad);
                if (bad) continue;
                const float weight = __shfl(p, j, 64);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (lane + 64 * i < w.dim) o[i] = __builtin_fmaf(weight, value(v, lane + 64 * i), o[i]);
            }
        }
        if (!w.slot) {
            const float by = inverse(sum) * w.v_scale;
            uint16_t *const out = w.out + tok * w.o_tok + head * w.o_head;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane + 64 * i < w.dim) out[lane + 64 * i] = (uint16_t)(pack_bf16_rne(o[i] * by, 0.0f) & 0xFFFFu);
        } else {
            if (lane == 0) put(w.slot + pair_at(r), Pair{top, sum});
#pragma unroll
            for (int i = 0; i < N; ++i)
                __hip_atomic_store(w.slot + value_at(r, lane + 64 * i), o[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    wd::wait_vmcnt<0>();
}

// The tiles of all sequences for one kv head, by 64 sequences at a time in every wave; `upto`: of the first 64, those of a lane's and
// before. Starts that do not ascend may count rows many times over: where the tiles of all kv heads would pass 32 bits, there
// are none (the host has refused sizes that could by themselves).
template <int M, int TT, bool SHARE>
__device__ __forceinline__ int all_units(const AttendArgs &p, int lane, int &upto) {
    auto of = [&](int i) {
        if (i >= p.sequences) return 0;
        const Units u = units_of<M, TT, SHARE>(p, sequence(p, i));
        return u.tiles * u.run;
    };
    int64_t total = 0, most = INT32_MAX / p.kv_heads;
    for (int i = 0; i < p.sequences; i += 64) {
        const int v = of(i + lane);
        // 64 values of up to 2^25 fit a scan; larger ones are summed one by one in 64 bits.
        if (__any(v >> 25)) {
            for (int l = 0; l < 64; ++l) total += __builtin_amdgcn_readlane(v, l);
            if (i == 0 && total <= most) upto = wave_scan(v, lane);
        } else {
            const int sum = wave_scan(v, lane);
            if (i == 0) upto = sum;
            total += __builtin_amdgcn_readlane(sum, 63);
        }
        if (total > most) return 0;
    }
    return (int)total;
}

// The sequence that holds tile number `start` of all, and the tiles of one kv head in the sequences before it.
template <int M, int TT, bool SHARE>
__device__ __forceinline__ void find_unit(const AttendArgs &p, int start, int lane, int upto, int &b, int &before) {
    before = b = 0;
    for (int i = 0; i < p.sequences; i += 64) {
        if (i > 0) {
            int v = 0;
            if (i + lane < p.sequences) {
                const Units u = units_of<M, TT, SHARE>(p, sequence(p, i + lane));
                v = u.tiles * u.run;
            }
            upto = wave_scan(v, lane);
        }
        const uint64_t past = __ballot((before + upto) * p.kv_heads > start);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            before += l > 0 ? __builtin_amdgcn_readlane(upto, l - 1) : 0;
            b = i + l;
            return;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
}

// A part of a unit: at most a workgroup's first unit and its last are parts.
struct Part {
    int first, tiles;     // the unit's numbered tiles (tiles 0: none)
    int row0, rows, kvh;  // first row of the tile in its sequence, the sequence's rows; its kv head
    int at;               // the sequence's first row of q
};

// The slots of this workgroup's parts have been written and a barrier passed: counted, and joined by the workgroup that counts
// last, in the order of the workgroups. A slot is M pairs (maximum, sum) and then, two by two, the unnormalised outputs:
// pair `item` is values at, at + 1 of row `row`, as `place` says. First a thread a row finds its
// maximum and sum over the slots, then a thread takes pairs of every slot, several at a time: the join waits for memory.
template <int M, int DP, int THREADS, bool F8, class Place>
__device__ __forceinline__ void join_parts(const AttendArgs &p, const Share &share, const Part *parts, int *joins, Place place) {
    __shared__ Pair stats[M];
    const int tid = threadIdx.x;
    if (parts[0].tiles == 0 && parts[1].tiles == 0) return;
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
        const float v_scale = F8 && p.v_scale ? p.v_scale[part.kvh] : 1.0f;
        auto slot_of = [&](int g) { return p.part + (int64_t)(g == g0 ? slot0 : 2 * g) * attend_part_floats(DP, M); };
        // A row's maximum, and what its outputs are multiplied by.
        for (int row = tid; row < M; row += THREADS) {
            float top = -INFINITY, sum = 0.0f;
            constexpr int ROUND = 8;  // slots whose loads are under way at once
            for (int g = g0; g <= g1; g += ROUND) {
                Pair s[ROUND];
#pragma unroll
                for (int k = 0; k < ROUND; ++k) s[k] = get(slot_of(min(g + k, g1)) + 2 * row);
                float most = top;
#pragma unroll
                for (int k = 0; k < ROUND; ++k) most = fmaxf(most, s[k].a);
                const float from = most == -INFINITY ? 0.0f : most;
                sum *= __builtin_amdgcn_exp2f(top - from);
                top = most;
#pragma unroll
                for (int k = 0; k < ROUND; ++k) sum = g + k > g1 ? sum : __builtin_fmaf(s[k].b, __builtin_amdgcn_exp2f(s[k].a - from), sum);
            }
            stats[row] = Pair{top == -INFINITY ? 0.0f : top, inverse(sum) * v_scale};
        }
        __syncthreads();
        constexpr int ITEMS = M * DP / 2, MANY = ITEMS / THREADS < 4 ? ITEMS / THREADS : 4, ROUND = 4;
        static_assert(ITEMS % (MANY * THREADS) == 0, "whole rounds");
        for (int item0 = tid; item0 < ITEMS; item0 += MANY * THREADS) {
            int row[MANY], at[MANY];
            bool any = false;
#pragma unroll
            for (int i = 0; i < MANY; ++i) {
                place(item0 + i * THREADS, row[i], at[i]);
                if (at[i] >= p.dim) row[i] = M;
                any = any || part.row0 + row[i] < part.rows;
            }
            if (!any) continue;
            float x[MANY] = {}, y[MANY] = {};
            for (int g = g0; g <= g1; g += ROUND) {
                Pair v[ROUND][MANY];
                float top[ROUND][MANY];
#pragma unroll
                for (int k = 0; k < ROUND; ++k)
#pragma unroll
                    for (int i = 0; i < MANY; ++i) {
                        const float *const slot = slot_of(min(g + k, g1));
                        top[k][i] = __hip_atomic_load(slot + 2 * min(row[i], M - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        v[k][i] = get(slot + 2 * M + 2 * (item0 + i * THREADS));
                    }
#pragma unroll
                for (int k = 0; k < ROUND; ++k)
#pragma unroll
                    for (int i = 0; i < MANY; ++i) {
                        if (g + k > g1) continue;
                        const float weight = __builtin_amdgcn_exp2f(top[k][i] - stats[min(row[i], M - 1)].a);
                        x[i] = __builtin_fmaf(v[k][i].a, weight, x[i]);
                        y[i] = __builtin_fmaf(v[k][i].b, weight, y[i]);
                    }
            }
#pragma unroll
            for (int i = 0; i < MANY; ++i) {
                const int r = part.row0 + row[i];
                if (row[i] >= M || r >= part.rows) continue;
                const int tok = r / p.group, head = part.kvh * p.group + (r - tok * p.group);
                const float by = stats[row[i]].b;
                *reinterpret_cast<uint32_t *>(p.out + (int64_t)(part.at + tok) * p.o_tok + (int64_t)head * p.o_head + at[i]) =
                    pack_bf16_rne(x[i] * by, y[i] * by);
            }
        }
        __syncthreads();
    }
}

}  // namespace attend
}  // namespace sq8
