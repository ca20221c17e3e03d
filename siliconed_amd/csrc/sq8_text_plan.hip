// sq8_text_plan.hip — the text decoder operators' launches: which kernel, tile and split of K a block-scaled product
// takes, how many workgroups a paged attention takes and the buffers that they need. Host code alone.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sq8_text.h"

namespace sq8 {
namespace {

// The tile kernels: rows, weight rows, workgroups a CU holds; microseconds a step of one block takes with one workgroup
// on a CU and with as many as it holds, for a bf16 C and for an fp32 one.
struct TileCost {
    int rows, columns, held;
    float one, all, one_f32, all_f32;
};
// F8_128_ONE has eight waves and four stages: 33 µs at M = 128, K = 4096, N = 24576 (GLU) where F8_128 takes 40 and F8_64x128
// 37.5, while two rounds of it are no match for two workgroups of F8_128 a CU (44 µs and 38 at M = 2048, K = N = 4096).
// Over M 20 to 8192, K 512 to 12288, N 512 to 24576, plain, GLU and fp32 out (28 shapes), the tile and split that these
// figures choose take at most a tenth longer than the best of all.
constexpr TileCost kTiles[F8_TILES] = {{256, 256, 1, 1.9f, 1.9f, 0.0f, 0.0f},
                                       {128, 128, 2, 0.85f, 1.36f, 1.25f, 2.2f},
                                       {128, 128, 1, 0.66f, 0.66f, 1.15f, 1.15f},
                                       {64, 128, 2, 0.47f, 0.82f, 0.78f, 1.29f},
                                       {64, 64, 2, 0.36f, 0.49f, 0.52f, 0.77f}};
// A launch and its first loads; the weight's bytes at the rate they are read with, and those that come into a CU with
// either operand; adding up the parts of a split K: once, for each part, and their bytes.
constexpr float kLaunch = 3.0f, kBytesMicrosecond = 5.0e6f, kIntoCU = 45.0e3f, kJoin = 1.6f, kJoinPart = 0.5f, kPartMicrosecond = 5.0e6f;

}  // namespace

// Up to 16 rows the short kernel: each of its workgroups reads its weight rows and all of A, and a CU takes in a bounded
// number of bytes a cycle, so 16 or 32 columns a workgroup by the bytes that the fullest CU takes. At M = 16, K = 4096:
// N = 6144 11.3 µs by 16 and 8.8 by 32, N = 4096 7.1 and 8.7, N = 24576 (GLU) 25.8 and 29.0. Values of up to F8_STAGED_GROUPS
// groups are quantized there: one row of K = 4096 by N = 4096 takes 6.6 µs so and 8.2 in two kernels, of K = 12288 15.3
// and 16.6, four rows of K = 4096 7.4 and 9.6. (GLUs, of three workgroups a CU and more, gain nothing: 25.0 and 24.2.)
// Above, the tile and the split of K with the least estimated time: rounds of workgroups times steps, not under the
// time the bytes take. At M = 64, K = 12288, N = 4096: 64 × 64 tiles 37.6 µs whole and 17.5 in four parts; at M = 2048
// of the same 256 × 256 160 and 128 × 128 120; at M = 8192, K = 4096, N = 24576 752 and 885.
// Rows too far apart for the tile kernels' 32-bit offsets go to the short kernel.
// Whole tiles sum K block by block, all alike, so rows have the same bits on any of them; a split's do not. From 4096 rows on
// and past 1024 columns there is none, as for the other products: there chunks of a call's rows give the call's bits. (It
// costs nothing: an fp32 C of 4097 × 2048 at K = 8192 takes 198 µs in two parts and 191 whole, at K = 16384 331 and 334.)
F8Plan f8_plan(const F8Args &p, bool glu, bool out_f32, int cus) {
    F8Plan plan = {F8_FAR, 1, 0, 0, false};
    if (p.M <= 0 || p.H <= 0) return plan;
    const int halves = glu ? 2 : 1;
    if (p.M <= 16) {
        auto fullest = [&](int columns) {
            const int64_t groups = (p.H + columns - 1) / columns;
            return ((groups + cus - 1) / cus) * (columns * halves + p.M);
        };
        const bool wide = fullest(32) < fullest(16);
        plan.values = p.x && !glu && (int64_t)p.M * p.KB <= F8_STAGED_GROUPS;
        plan.kernel = plan.values ? (wide ? F8_STAGED_WIDE : F8_STAGED) : wide ? F8_SHORT_WIDE : F8_SHORT;
        return plan;
    }
    const bool near = 256 * std::max(std::max(p.lda, p.ldw), 4 * p.ldsx) + p.K <= INT32_MAX &&
                      (!glu || ((int64_t)p.H + 256) * p.ldw + p.K <= INT32_MAX);
    if (!near) return plan;
    const bool whole = p.M >= 4096 && p.N > 1024;
    float best = 0.0f;
    for (int t = out_f32 ? F8_128 : F8_256; t < F8_TILES; ++t) {
        const TileCost &c = kTiles[t];
        const int64_t tiles = (int64_t)((p.M + c.rows - 1) / c.rows) * ((p.H * halves + c.columns - 1) / c.columns);
        for (int splits = 1; splits <= 8; ++splits) {
            if (splits > 1 && (t < F8_64x128 || p.KB < 4 * splits || whole)) break;
            const int64_t groups = tiles * splits, slots = (int64_t)cus * c.held, rest = groups % slots;
            const int steps = (p.KB + splits - 1) / splits;
            const float one = out_f32 ? c.one_f32 : c.one, all = out_f32 ? c.all_f32 : c.all;
            const float last = rest == 0 ? 0.0f : rest <= cus ? one : one + (all - one) * (float)(rest - cus) / (float)(slots - cus);
            float us = steps * ((float)(groups / slots) * all + last);
            us = std::max(us, ((float)p.N * p.K + (float)p.M * p.K) / kBytesMicrosecond);
            us = std::max(us, (float)groups * steps * (float)((c.rows + c.columns) * F8_GROUP) / ((float)std::min<int64_t>(groups, cus) * kIntoCU));
            const int64_t part = groups * c.rows * c.columns * 4;
            if (splits > 1) us += kJoin + kJoinPart * splits + (float)part / kPartMicrosecond;
            us += kLaunch;
            if (best == 0.0f || us < best) {
                best = us;
                plan = F8Plan{t, splits, splits > 1 ? part : 0, splits > 1 ? tiles * MARK : 0, false};
            }
        }
    }
    return plan;
}

// n / page for n < 2^31 as (n · mul) >> shift: s with 2^(s-1) < page ≤ 2^s, mul = floor(2^(31+s) / page) + 1 ≤ 2^32 + 1,
// the product's excess under n / 2^(31+s) < 2^-s ≤ 1/page.
void page_divisor(PagedArgs &p) {
    int s = 0;
    while ((1ll << s) < p.page) ++s;
    p.page_shift = 31 + s;
    p.page_mul = ((1ull << (31 + s)) / (uint64_t)p.page) + 1;
}

int paged_groups(const PagedArgs &p, int cus) {
    const int passes = (p.q_heads / p.kv_heads + 15) / 16;
    int64_t tokens = (int64_t)p.max_pages * p.page;
    if (p.window > 0) tokens = std::min<int64_t>(tokens, (int64_t)p.window + 31);  // (the window may be the largest int)
    const int64_t most = (int64_t)p.batch * p.kv_heads * passes * ((tokens + PAGED_TILE - 1) / PAGED_TILE);
    const int64_t full = paged_held(paged_dim(p.dim)) * (int64_t)cus;
    return (int)(most < 1 ? 1 : most < full ? most : full);
}

int64_t paged_part_bytes(const PagedArgs &p, int groups) {
    return groups == 1 ? 0 : (int64_t)2 * groups * paged_part_floats(paged_dim(p.dim)) * 4;
}

int64_t paged_marks(const PagedArgs &p) { return (int64_t)MARK * p.batch * p.kv_heads * ((p.q_heads / p.kv_heads + 15) / 16); }

}  // namespace sq8
