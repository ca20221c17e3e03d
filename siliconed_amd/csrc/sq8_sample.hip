// sq8_sample.hip — the next token of each row of logits, drawn with a given random number (include/siliconed_q8.h:
// sq8_sample_tokens).
//
//   w_i = exp((x_i − max x) / t);  in the order of falling x, equal ones by index: the first top_k, of these the fewest that
//   hold top_p of their sum, of these the ones with w ≥ min_p; then, by index, the first whose running sum passes u times the whole.
//
// Nothing is sorted. What is kept is always the order's first so many, so it is told by the key of the last one kept (the fp32
// logit's bits, made to rise with it) and, among logits equal to that, by the last index. Counts and sums over bins of keys
// find the bin that the cut lies in, then the same inside it, until a bin is one key.
//
// Weights are whole numbers of 2^-43 (from an exponential in 64 bits), summed as 64-bit integers: no order of additions
// changes a bit, so a cut or a draw is the formula's but where a border is nearer than some 2^-40 of the whole. (In fp32 the
// weights' errors would move each of a hundred thousand borders by 1e-7 of the whole: one draw in a hundred would differ.)
//
// A workgroup of 8 waves takes a row, and reads it at least twice: for the maximum, and for a list of the logits near it (by
// the threads' two largest each), in which the cut nearly always lies with top_k or a nucleus of some thousands. There the
// bin of the cut holds few, which are compared with each other, as are the last candidates by index. The whole sum that a nucleus
// is a part of is first bounded by fp32 exponentials (at temperatures of 2^-100 to 2^100); only where the bounds disagree on the cut is it summed exactly. A wide
// nucleus goes by bins over the row.
//
// 128 rows of 128 000 fp32 logits, every option set, take 37 µs: the first pass runs at the memory's rate (11 µs), the second, from
// the last cache level, 14, the rest is barriers and scans. One row of 32 000 with a nucleus 23 to 26 µs, of which the list and the
// fp32 sum are 10 (one CU's vector ALU) and the exact sum, one time in ten, 15 more. A nucleus past the list: 2 rows of 157 420
// 236 µs, two passes of 64-bit exponentials of 50 each, three of keys; another workgroup a row would halve it. 64 rows of 128 000
// with min_p alone 46 (92 where runs of logits under what it leaves were not passed over). With sixteen
// waves a row, whose registers spilled, and an atomic a listed logit the first two were 102 and 47.
#include <hip/hip_runtime.h>

#include "sq8_device.h"
#include "sq8_text.h"
#include "sq8_text_device.h"

namespace sq8 {
namespace {

constexpr int THREADS = 512, WAVES = THREADS / 64, BINS = THREADS, LOG_BINS = 9, LIST = 4096, SEG = LIST / WAVES, CHUNKS = 4096;
static_assert(BINS == 1 << LOG_BINS, "a bin a thread");
constexpr unsigned FEW = 256;  // of so many, each is compared with every other
constexpr int ONE = 43;  // a weight of 1 is 2^43: 2^20 of them fit 64 bits

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // (−0 is 0)
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// The sum of v over this lane and those before it.
template <typename T>
__device__ __forceinline__ T lanes_scan(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

struct Cut {
    uint32_t key;        // of the last one kept
    unsigned keep, ties; // how many of the logits equal to it are kept, and how many there are
    unsigned above;      // those of larger ones
    uint64_t sum;        // and their weights
};

template <bool BF16>
struct Row {
    static constexpr int E = BF16 ? 8 : 4;   // logits a load takes
    static constexpr int CHUNK = 64 * E;     // consecutive logits a wave takes at a time

    const void *at;
    int vocab;
    int lane, wave, tid;

    __device__ __forceinline__ float one(int i) const {
        float x = BF16 ? bf16_f32(static_cast<const uint16_t *>(at)[i]) : static_cast<const float *>(at)[i];
        return x == x ? x : -INFINITY;  // a NaN is not drawn
    }
    __device__ __forceinline__ u32x4 fetch(int i) const {
        if constexpr (BF16) return *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(at) + i);
        else return *reinterpret_cast<const u32x4_any *>(static_cast<const float *>(at) + i);
    }
    static __device__ __forceinline__ void logits(const u32x4 &d, float (&x)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = BF16 ? __uint_as_float(e & 1 ? d[e / 2 % 4] & 0xFFFF0000u : d[e / 2 % 4] << 16) : __uint_as_float(d[e % 4]);
            x[e] = v == v ? v : -INFINITY;
        }
    }
    // Eight (four) logits from i on; past the row's end, and for NaN, -inf.
    __device__ __forceinline__ void load(int i, float (&x)[E]) const {
        if (i + E <= vocab) {
            logits(fetch(i), x);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = i + e < vocab ? one(i + e) : -INFINITY;
        }
    }
    // f(first index, logits) of a lane's runs; a wave's lie side by side, and a lane's loads of 32 logits are under way at once.
    template <typename F>
    __device__ __forceinline__ void runs(F &&f) const {
        constexpr int STEP = THREADS * E, MANY = 32 / E;
        int first = 0;
        for (; first + MANY * STEP <= vocab; first += MANY * STEP) {
            u32x4 d[MANY];
#pragma unroll
            for (int j = 0; j < MANY; ++j) d[j] = fetch(first + j * STEP + tid * E);
#pragma unroll
            for (int j = 0; j < MANY; ++j) {
                float x[E];
                logits(d[j], x);
                f(first + j * STEP + tid * E, x);
            }
        }
        for (int i = first + tid * E; i < vocab; i += STEP) {
            float x[E];
            load(i, x);
            f(i, x);
        }
    }
};

template <bool BF16>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const SampleArgs p) {
    using R = Row<BF16>;
    constexpr int E = R::E;
    __shared__ uint64_t list[LIST];   // key and index of the logits near the top, a segment a wave
    __shared__ uint64_t acc[CHUNKS];  // sums: of bins, or of chunks of indices
    __shared__ uint32_t cnt[BINS];
    __shared__ uint64_t wave_sum[WAVES];
    __shared__ uint32_t wave_cnt[WAVES];
    __shared__ float wave_a[WAVES], wave_b[WAVES];
    __shared__ double table[64];
    __shared__ uint32_t crowded, gathered, found, found_cnt, found_has;
    __shared__ uint64_t found_sum;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t b = blockIdx.x;
    R row;
    row.at = BF16 ? static_cast<const void *>(static_cast<const uint16_t *>(p.logits) + b * p.ld)
                  : static_cast<const void *>(static_cast<const float *>(p.logits) + b * p.ld);
    row.vocab = p.vocab;
    row.lane = lane; row.wave = wave; row.tid = tid;
    const float t = p.temperature ? p.temperature[b] : 1.0f;
    const float top_p = p.top_p ? p.top_p[b] : 1.0f, min_p = p.min_p ? p.min_p[b] : 0.0f;
    const int want = p.top_k ? p.top_k[b] : 0;
    const bool by_count = want > 0 && want < p.vocab, by_sum = !(top_p >= 1.0f);
    const bool greedy = !(t > 0.0f) || (by_count && want == 1) || min_p > 1.0f;  // (no weight is more than 1: the first of the order is left)

    // ---- the largest logit, and each thread's own two ----
    float half[2] = {-INFINITY, -INFINITY};  // of the logits at even places, and at odd ones
    int half_at[2] = {INT32_MAX, INT32_MAX};
    float under = INFINITY;                    // the smallest but -inf
    row.runs([&](int i, const float (&x)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            under = fminf(under, x[e] > -INFINITY ? x[e] : INFINITY);
            if (x[e] > half[e & 1]) {
                half[e & 1] = x[e];
                half_at[e & 1] = i + e;
            }
        }
    });
    const float mine = fmaxf(half[0], half[1]);
    const int mine_at = half[0] > half[1] || (half[0] == half[1] && half_at[0] < half_at[1]) ? half_at[0] : half_at[1];
    if (tid < 64) table[tid] = exp2((double)tid * (1.0 / 64.0));
    {
        float top = mine, low = INFINITY;
#pragma unroll
        for (int e = 0; e < 2; ++e) low = half[e] > -INFINITY ? fminf(low, half[e]) : low;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            top = fmaxf(top, __shfl_xor(top, o, 64));
            low = fminf(low, __shfl_xor(low, o, 64));
        }
        if (lane == 0) {
            wave_a[wave] = top;
            wave_b[wave] = low;
        }
    }
    cnt[tid] = 0;
    acc[tid] = 0;
    if (tid == 0) crowded = 0;  // a wave's segment is too short
    __syncthreads();
    float top = wave_a[0], low = wave_b[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        top = fmaxf(top, wave_a[i]);
        low = fminf(low, wave_b[i]);
    }
    if (top == -INFINITY) {
        if (tid == 0) {
            p.tokens[b] = -1;
            if (p.logprobs) p.logprobs[b] = -INFINITY;
        }
        return;
    }
    if (greedy) {
        int at = mine == top ? mine_at : INT32_MAX;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
        if (lane == 0) wave_cnt[wave] = (uint32_t)at;
        __syncthreads();
        if (tid == 0) {
            for (int i = 0; i < WAVES; ++i) at = min(at, (int)wave_cnt[i]);
            p.tokens[b] = at;
            if (p.logprobs) p.logprobs[b] = 0.0f;
        }
        return;
    }

    // A weight, in units of 2^-43: 2^(k/64) from the table times 2^r, |r| ≤ 1/128, whose series to r⁴ is within 2^-44. (k in the
    // low bits of y + 1.5 · 2^52; the exponent added as a whole number; rounded to 2^-43 by the addition of 2^9.)
    const double per = -64.0 * 1.4426950408889634 / (double)t, top64 = (double)top;
    auto weight = [&](float x) -> uint64_t {
        constexpr double C = 0.6931471805599453 / 64.0;
        const double y = fmax((top64 - (double)x) * per, -64.0 * (ONE + 3)), near = y + 0x1.8p52;
        const int n = (int)(uint32_t)__double_as_longlong(near);
        const double r = y - (near - 0x1.8p52);
        const double e = fma(r, fma(r, fma(r, fma(r, C * C * C * C / 24.0, C * C * C / 6.0), C * C / 2.0), C), 1.0);
        const double v = __longlong_as_double(__double_as_longlong(table[n & 63] * e) + ((int64_t)(n >> 6) << 52)) + 0x1p9;
        const uint64_t w = (uint64_t)__double_as_longlong(v) - (uint64_t)__double_as_longlong(0x1p9);
        return x == top ? 1ull << ONE : w;
    };

    // Over the bins of cnt and acc, from the first: the one in which the counts reach `need`, or with `sums` the sums T.
    // Every thread gets its number (BINS: none) and what lies before it. The bins are cleared.
    unsigned before_cnt = 0, all_cnt = 0;
    uint64_t before_sum = 0, all_sum = 0;
    unsigned scan_cnt;
    uint64_t scan_sum;
    auto scan = [&]() {
        __syncthreads();
        const unsigned c = cnt[tid];
        const uint64_t s = acc[tid];
        const unsigned uc = lanes_scan(c, lane);
        const uint64_t us = lanes_scan(s, lane);
        if (lane == 63) {
            wave_cnt[wave] = uc;
            wave_sum[wave] = us;
        }
        cnt[tid] = 0;
        acc[tid] = 0;
        __syncthreads();
        before_cnt = 0;
        before_sum = 0;
        all_cnt = 0;
        all_sum = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            before_cnt += i < wave ? wave_cnt[i] : 0;
            before_sum += i < wave ? wave_sum[i] : 0;
            all_cnt += wave_cnt[i];
            all_sum += wave_sum[i];
        }
        scan_cnt = before_cnt + uc;   // with this thread's bin
        scan_sum = before_sum + us;
        before_cnt = scan_cnt - c;    // and without
        before_sum = scan_sum - s;
    };
    struct Place {
        unsigned bin, cnt, has;  // the bin, those before it and in it
        uint64_t sum;            // and the weights before it
    };
    auto place = [&](bool sums, unsigned need, double T, double T2) {  // after scan(); T2 ≥ T: the bin that holds both
        if (tid == 0) found = BINS;
        __syncthreads();
        const bool here = sums ? (double)before_sum < T && (double)scan_sum >= T2 : before_cnt < need && scan_cnt >= need;
        if (here) {
            found = tid;
            found_cnt = before_cnt;
            found_has = scan_cnt - before_cnt;
            found_sum = before_sum;
        }
        __syncthreads();
        const Place at = {found, found_cnt, found_has, found_sum};
        __syncthreads();
        return at;
    };

    const bool all_of_it = !by_count && !by_sum;  // no cut but min_p's
    const uint32_t top_key = key_of(top);
    Cut cut = {0, 0, 0, 0, 0};
    bool from_list = false;   // what is kept lies in the list
    uint64_t *const segment = list + wave * SEG;
    uint32_t listed = 0;      // of the wave's

    if (!all_of_it && top == INFINITY) {
        // The infinities share everything.
        row.runs([&](int, const float (&x)[E]) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (x[e] == INFINITY) atomicAdd(&cnt[0], 1u);
        });
        scan();
        cut.key = top_key;
        cut.ties = all_cnt;
        cut.keep = by_count ? min(all_cnt, (unsigned)want) : all_cnt;
        if (by_sum) cut.keep = max(1u, (unsigned)fmin((double)cut.keep, ceil((double)fmaxf(top_p, 0.0f) * (double)cut.keep)));
    } else if (!all_of_it) {
        // ---- bins of the distance from the top: first down to where some 2000 logits lie, or as many as
        // top_k (by the threads' largest ones), and those in a list; where the cut is not among them, down to where weights end ----
        float by = 0.0f;
        unsigned last = BINS - 1;
        const bool short_row = p.vocab <= LIST;
        auto bin_of = [&](float x) { return (unsigned)fminf((top - x) * by, (float)(BINS - 1)); };
        if (!short_row) {
            by = top > low ? (float)(BINS - 1) / (top - low) : 0.0f;
            if (!(by < 3e38f)) by = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (half[e] > -INFINITY) atomicAdd(&cnt[bin_of(half[e])], 1u);
            scan();
            const Place at = place(false, min(by_count ? min(max((unsigned)want, 64u), 900u) : 900u, all_cnt), 0.0, 0.0);
            last = at.bin;
        }
        double T = 0.0;
        uint64_t total = 0;
        bool wide = false;
        // Bins of distances down to `span`.
        auto spread = [&](float span) {
            by = span > 0.0f && span < INFINITY ? (float)(BINS - 1) / span : 0.0f;
            if (!(by < 3e38f)) by = 0.0f;
        };
        float least = 0.0f;  // the row's smallest logit, where it is needed
        auto find_least = [&]() {
            float v = under;
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) v = fminf(v, __shfl_xor(v, o, 64));
            __syncthreads();
            if (lane == 0) wave_b[wave] = v;
            __syncthreads();
            least = wave_b[0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) least = fminf(least, wave_b[i]);
        };
        auto far_span = [&]() { return by_count ? top - least : fminf(top - least, t * 31.2f); };  // (2^-45 at 31.19 t)
        if (short_row) {
            find_least();
            spread(far_span());
        }
        Place k_place = {BINS, 0, 0, 0}, p_place = {BINS, 0, 0, 0};
        float k_by = 0.0f, p_by = 0.0f;
        bool k_list = false, p_list = false;

        // From a bin of distances (by `with`) to one key, over the list or the row.
        // (`goal2` ≥ goal, among few: the key that holds both, or 0.)
        auto refine = [&](Place at, float with, bool sums, unsigned need, double goal, double goal2, bool in_list) {
            by = with;
            if (in_list && at.has <= FEW) {
                // Few in the bin: gathered behind the bins' sums, and every one compared with the others.
                uint64_t *const keys = acc + BINS, *const weights = keys + FEW;
                if (tid == 0) gathered = found = 0;
                __syncthreads();
                for (unsigned i = lane; i < listed; i += 64) {
                    const uint32_t key = (uint32_t)(segment[i] >> 32);
                    const float x = of_key(key);
                    if (bin_of(x) == at.bin) {
                        const uint32_t slot = atomicAdd(&gathered, 1u);
                        keys[slot] = key;
                        weights[slot] = sums ? weight(x) : 0;
                    }
                }
                __syncthreads();
                if ((unsigned)tid < at.has) {
                    const uint32_t key = (uint32_t)keys[tid];
                    unsigned more = at.cnt, same = 0;
                    uint64_t sum = at.sum;
                    for (unsigned j = 0; j < at.has; ++j) {
                        const uint32_t k = (uint32_t)keys[j];
                        more += k > key;
                        same += k == key;
                        if (sums) sum += k > key ? weights[j] : 0;
                    }
                    const bool here = sums ? (double)sum < goal && (double)(sum + same * weights[tid]) >= goal2 : more < need && more + same >= need;
                    if (here) {  // (its equals write the same)
                        found = key;
                        found_cnt = more;
                        found_has = same;
                        found_sum = sum;
                    }
                }
                __syncthreads();
                const Cut c = {found, 0, found_has, found_cnt, found_sum};
                __syncthreads();
                return c;
            }
            // The bin's keys: bin_of falls with the key, so both ends are found by halving (64 keys a step).
            auto first_key = [&](unsigned bin) {  // the smallest key whose bin is `bin` or less
                uint32_t lo = 0;                  // (key_of(-inf) and less are in the last bins)
                for (int s = 26; s > -6; s -= 6) {
                    const int sh = s < 0 ? 0 : s;
                    const uint64_t k = (uint64_t)lo + ((uint64_t)lane << sh);
                    const float x = k <= top_key ? of_key((uint32_t)k) : top;
                    const bool fits = k >= top_key || (x == x && x > -INFINITY && bin_of(x) <= bin);
                    const uint64_t yes = __ballot(fits);
                    const int l = yes ? __ffsll((unsigned long long)yes) - 1 : 64;
                    lo = l == 0 ? lo : (uint32_t)(lo + ((uint64_t)(l - 1) << sh) + (sh == 0 ? 1 : 0));
                    if (sh == 0) break;
                }
                return lo;
            };
            uint32_t lo = first_key(at.bin), hi = at.bin == 0 ? top_key : first_key(at.bin - 1) - 1;
            Cut c = {hi, 0, 0, at.cnt, at.sum};
            for (;;) {
                const uint32_t range = hi - lo;
                const int sh = range < BINS ? 0 : 32 - __builtin_clz(range) - LOG_BINS;
                auto put_in = [&](uint32_t key, float x) {
                    if (key < lo || key > hi) return;
                    atomicAdd(&cnt[(hi - key) >> sh], 1u);
                    if (sums) atomicAdd(reinterpret_cast<unsigned long long *>(&acc[(hi - key) >> sh]), (unsigned long long)weight(x));
                };
                if (in_list) {
                    for (unsigned i = lane; i < listed; i += 64) {
                        const uint32_t key = (uint32_t)(segment[i] >> 32);
                        put_in(key, of_key(key));
                    }
                } else {
                    row.runs([&](int, const float (&x)[E]) {
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (x[e] > -INFINITY) put_in(key_of(x[e]), x[e]);
                    });
                }
                scan();
                const Place q = place(sums, need - c.above, goal - (double)c.sum, goal - (double)c.sum);
                // (Rounding may leave the goal a hair past the bin's sums: then its last keys.)
                const unsigned bin = q.bin < BINS ? q.bin : range >> sh;
                if (q.bin < BINS) {
                    c.above += q.cnt;
                    c.sum += q.sum;
                    c.ties = q.has;
                }
                const uint32_t up = hi - (bin << sh);
                lo = sh == 0 ? up : max(lo, up - ((1u << sh) - 1));
                hi = up;
                if (sh == 0) break;
            }
            c.key = hi;
            return c;
        };
        for (int pass = 0; pass < 2; ++pass) {
            double rest32 = 0.0;  // what lies past the bins, from exponentials in fp32
            const bool sum_all = by_sum && !by_count && !wide;
            // (Only where fp32 holds what the exponents are made of: at temperatures past these, 1 / t may be 0, which -inf would make
            // NaNs of, or a difference past the largest number may weigh something.)
            const bool estimated = sum_all && t >= 0x1p-100f && t <= 0x1p100f;
            const float per32 = 1.4426950408889634f / t;
            auto put_in = [&](float x) {
                const unsigned bin = bin_of(x);
                if (bin > last) return;
                atomicAdd(&cnt[bin], 1u);
                if (by_sum) atomicAdd(reinterpret_cast<unsigned long long *>(&acc[bin]), (unsigned long long)weight(x));
            };
            if (!wide) {
                // The list first.
                const float rough = top - (float)(last + 2) / by;  // (no less than any that is in; by 0 gives -inf or a NaN)
                row.runs([&](int i, const float (&x)[E]) {
                    if (!estimated) {
                        float m = x[0];
#pragma unroll
                        for (int e = 1; e < E; ++e) m = fmaxf(m, x[e]);
                        if (!__any(!(m < rough))) return;
                    }
                    bool in[E];
                    uint64_t hit[E], all = 0;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        in[e] = x[e] > -INFINITY && bin_of(x[e]) <= last;
                        hit[e] = __ballot(in[e]);
                        all |= hit[e];
                    }
                    if (estimated) {
                        float w[E], sum = 0.0f;
#pragma unroll
                        for (int e = 0; e < E; ++e) w[e] = in[e] ? 0.0f : __builtin_amdgcn_exp2f((x[e] - top) * per32);
#pragma unroll
                        for (int e = 0; e < E; ++e) sum += w[e];
                        rest32 += (double)sum;
                    }
                    if (all == 0) return;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t to = __builtin_amdgcn_mbcnt_hi((uint32_t)(hit[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit[e], listed));
                        if (in[e] && to < SEG) segment[to] = (uint64_t)key_of(x[e]) << 32 | (uint32_t)(i + e);
                        listed += __popcll(hit[e]);
                    }
                });
                listed = __builtin_amdgcn_readfirstlane(listed);  // (a lane past the row's end has not counted to the last)
                if (listed > SEG && lane == 0) crowded = 1;
                __syncthreads();
            }
            if (!wide && !crowded) {
                for (unsigned i = lane; i < listed; i += 64) put_in(of_key((uint32_t)(segment[i] >> 32)));
            } else {
                row.runs([&](int, const float (&x)[E]) {
                    uint64_t w[E] = {};
                    if (by_sum) {
#pragma unroll
                        for (int e = 0; e < E; ++e) w[e] = weight(x[e]);  // (side by side: each is a long chain)
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const unsigned bin = bin_of(x[e]);
                        if (!(x[e] > -INFINITY) || bin > last) continue;
                        atomicAdd(&cnt[bin], 1u);
                        if (by_sum) atomicAdd(reinterpret_cast<unsigned long long *>(&acc[bin]), (unsigned long long)w[e]);
                    }
                });
            }
            scan();
            const unsigned in_bins = all_cnt;
            const uint64_t sum_bins = all_sum;
            const bool held = !wide && !crowded;
            // Sums over the workgroup of what the threads have.
            auto of_all = [&](uint64_t v) {
#pragma unroll
                for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
                __syncthreads();
                if (lane == 0) wave_sum[wave] = v;
                __syncthreads();
                v = 0;
#pragma unroll
                for (int i = 0; i < WAVES; ++i) v += wave_sum[i];
                __syncthreads();
                return v;
            };
            bool settled = false;
            if (sum_all) {
                // The cut for the least and the most that the rest can be: a weight in fp32 is within 2^-17 of its value (its exponent,
                // at most 45, three roundings; the exponential; eight in a sum), and a whole number of them within one. The same cut
                // for both is the cut; else, or without an estimate, the rest is summed exactly.
                const double est = (double)of_all((uint64_t)(rest32 * 0x1p43)), off = est * 0x1p-16 + (double)p.vocab + WAVES * 64.0;
                const double share_of = (double)fmaxf(top_p, 0.0f), held_sum = (double)sum_bins;
                const double low_T = estimated ? fmax(share_of * (held_sum + fmax(est - off, 0.0)), 1.0) : 0.0, high_T = fmax(share_of * (held_sum + est + off), 1.0);
                if (estimated && held_sum >= high_T && held) {
                    const Place both = place(true, 0, low_T, high_T);
                    if (both.bin < BINS && both.has <= FEW) {
                        const Cut c = refine(both, by, true, 0, low_T, high_T, true);
                        const uint64_t w = weight(of_key(c.key));
                        auto keep = [&](double goal) { return w ? (unsigned)fmin(fmax(ceil((goal - (double)c.sum) / (double)w), 1.0), (double)c.ties) : c.ties; };
                        settled = c.key != 0 && keep(low_T) == keep(high_T);
                        if (settled) {
                            cut = c;
                            cut.keep = keep(low_T);
                        }
                    }
                }
                if (settled) {
                    p_place.bin = BINS + 2;
                    p_list = true;
                } else if (held_sum >= low_T) {
                    uint64_t rest = 0;
                    row.runs([&](int, const float (&x)[E]) {
                        uint64_t w[E];  // (side by side: each is a long chain)
#pragma unroll
                        for (int e = 0; e < E; ++e) w[e] = weight(x[e]);
#pragma unroll
                        for (int e = 0; e < E; ++e) rest += x[e] > -INFINITY && bin_of(x[e]) <= last ? 0 : w[e];
                    });
                    total = sum_bins + of_all(rest);
                } else {
                    total = ~0ull;  // whatever it is, the cut lies past the bins
                }
            }
            if (wide && by_sum && !by_count) total = sum_bins;
            bool short_of = false;  // what is looked for lies past the bins
            if (by_count && k_place.bin == BINS) {
                k_place = place(false, want, 0.0, 0.0);
                if (k_place.bin == BINS) {
                    if (last == BINS - 1 && (wide || short_row)) {
                        // Fewer logits than top_k: all of them.
                        cut.key = key_of(least);
                        cut.above = in_bins;
                        k_place.bin = BINS + 1;
                        total = sum_bins;
                    } else {
                        short_of = true;
                    }
                } else {
                    k_by = by;
                    k_list = held;
                    if (by_sum) {
                        // The sum of the first top_k; the bins are needed again for the cut by sums.
                        const unsigned bc = before_cnt, sc = scan_cnt;
                        const uint64_t bs = before_sum, ss = scan_sum;
                        const Cut c = refine(k_place, k_by, false, want, 0.0, 0.0, k_list);
                        // The weights above the cut: over the source.
                        uint64_t sum = 0;
                        auto take = [&](uint32_t key, float x) { sum += key > c.key ? weight(x) : 0; };
                        if (k_list) {
                            for (unsigned i = lane; i < listed; i += 64) {
                                const uint32_t key = (uint32_t)(segment[i] >> 32);
                                take(key, of_key(key));
                            }
                        } else {
                            row.runs([&](int, const float (&x)[E]) {
#pragma unroll
                                for (int e = 0; e < E; ++e)
                                    if (x[e] > -INFINITY) take(key_of(x[e]), x[e]);
                            });
                        }
                        acc[tid] = sum;
                        scan();
                        total = all_sum + (uint64_t)(want - c.above) * weight(of_key(c.key));
                        cut = c;
                        before_cnt = bc; scan_cnt = sc; before_sum = bs; scan_sum = ss;
                    }
                }
            }
            if (by_sum && !short_of && p_place.bin == BINS) {
                T = fmax((double)fmaxf(top_p, 0.0f) * (double)total, 1.0);
                if ((double)sum_bins >= T) {
                    p_place = place(true, 0, T, T);
                    p_by = by;
                    p_list = held;
                } else if (wide || (short_row && last == BINS - 1)) {
                    p_place.bin = BINS + 1;  // everything of weight
                } else {
                    short_of = true;
                }
            }
            if (!short_of) break;
            wide = true;
            find_least();
            spread(far_span());
            last = BINS - 1;
            if (p_place.bin > BINS) p_place.bin = BINS;
        }

        // ---- the cut's key, and how many of the logits equal to it are kept ----
        if (by_sum && p_place.bin == BINS + 2) {
            from_list = p_list;  // settled above
        } else if (by_sum && p_place.bin < BINS) {
            const Cut k_cut = cut;
            cut = refine(p_place, p_by, true, 0, T, T, p_list);
            const uint64_t w = weight(of_key(cut.key));
            const double left = T - (double)cut.sum;
            cut.keep = w ? (unsigned)fmin(fmax(ceil(left / (double)w), 1.0), (double)cut.ties) : cut.ties;
            if (by_count && k_place.bin < BINS && cut.key == k_cut.key) cut.keep = min(cut.keep, want - k_cut.above);
            from_list = p_list;
        } else if (by_count && k_place.bin < BINS) {
            if (!by_sum) cut = refine(k_place, k_by, false, want, 0.0, 0.0, k_list);
            cut.keep = min(cut.ties, want - cut.above);
            from_list = k_list;
        } else {
            cut.key = 0;  // all
            cut.ties = cut.keep = 0;
            from_list = short_row && !crowded;
        }
    }

    // ---- by index: the first whose running sum of values over what is taken passes a goal ----
    // value(key, logit, index) of every logit; sums of chunks of indices, then the chunk in which they reach the goal, by one wave.
    const int chunks = (p.vocab + R::CHUNK - 1) / R::CHUNK;
    // (Logits under `least_x` have value 0: a run of nothing else is passed over.)
    auto select = [&](float least_x, auto &&value, auto &&goal, uint64_t &all) {
        __syncthreads();
        if (from_list) {
            // Few that count: each sums the others before it.
            uint64_t *const values = acc, *const places = acc + FEW;
            if (tid == 0) {
                gathered = 0;
                found_cnt = (uint32_t)p.vocab - 1;
            }
            __syncthreads();
            for (unsigned i = lane; i < listed; i += 64) {
                const uint32_t key = (uint32_t)(segment[i] >> 32), at = (uint32_t)segment[i];
                const uint64_t v = value(key, of_key(key), at);
                if (v) {
                    const uint32_t slot = atomicAdd(&gathered, 1u);
                    if (slot < FEW) {
                        values[slot] = v;
                        places[slot] = at;
                    }
                }
            }
            __syncthreads();
            const unsigned few = gathered;
            if (few <= FEW) {
                uint64_t sum = 0, before = 0;
                if ((unsigned)tid < few || tid == 0) {
                    const uint64_t own = (unsigned)tid < few ? places[tid] : 0;
                    for (unsigned j = 0; j < few; ++j) {
                        sum += values[j];
                        before += places[j] < own ? values[j] : 0;
                    }
                    if (tid == 0) wave_sum[0] = sum;
                    if ((unsigned)tid < few && !goal(before, sum) && goal(before + values[tid], sum)) found_cnt = (uint32_t)own;
                }
                __syncthreads();
                all = wave_sum[0];
                const uint32_t at = found_cnt;
                __syncthreads();
                return at;
            }
        }
        for (int i = tid; i < CHUNKS; i += THREADS) acc[i] = 0;
        __syncthreads();
        if (from_list) {
            for (unsigned i = lane; i < listed; i += 64) {
                const uint32_t key = (uint32_t)(segment[i] >> 32), at = (uint32_t)segment[i];
                const uint64_t v = value(key, of_key(key), at);
                if (v) atomicAdd(reinterpret_cast<unsigned long long *>(&acc[at / R::CHUNK]), (unsigned long long)v);
            }
        } else {
            for (int c = wave; c < chunks; c += WAVES) {
                float x[E];
                const int i = c * R::CHUNK + lane * E;
                row.load(i, x);
                float most = x[0];
#pragma unroll
                for (int e = 1; e < E; ++e) most = fmaxf(most, x[e]);
                uint64_t v = 0;
                if (__any(most >= least_x)) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint64_t one = value(key_of(x[e]), x[e], (uint32_t)(i + e));
                        v += x[e] > -INFINITY ? one : 0;
                    }
#pragma unroll
                    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
                }
                if (lane == 0) acc[c] = v;
            }
        }
        __syncthreads();
        uint64_t part[CHUNKS / THREADS], sum = 0;
#pragma unroll
        for (int j = 0; j < CHUNKS / THREADS; ++j) sum += part[j] = acc[tid * (CHUNKS / THREADS) + j];
        const uint64_t upto = lanes_scan(sum, lane);
        if (lane == 63) wave_sum[wave] = upto;
        if (tid == 0) found = 0xFFFFFFFFu;
        __syncthreads();
        uint64_t at = 0;
        all = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            at += i < wave ? wave_sum[i] : 0;
            all += wave_sum[i];
        }
        at += upto - sum;
#pragma unroll
        for (int j = 0; j < CHUNKS / THREADS; ++j) {
            if (!goal(at, all) && goal(at + part[j], all)) {
                found = tid * (CHUNKS / THREADS) + j;
                found_sum = at;
            }
            at += part[j];
        }
        __syncthreads();
        const uint32_t chunk = found;
        if (chunk != 0xFFFFFFFFu && wave == 0) {
            float x[E];
            const int i = (int)chunk * R::CHUNK + lane * E;
            row.load(i, x);
            uint64_t v[E], mine_sum = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) mine_sum += v[e] = x[e] > -INFINITY ? value(key_of(x[e]), x[e], (uint32_t)(i + e)) : 0;
            uint64_t s = found_sum + lanes_scan(mine_sum, lane) - mine_sum;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (!goal(s, all) && goal(s + v[e], all)) found_cnt = (uint32_t)(i + e);
                s += v[e];
            }
        }
        __syncthreads();
        return chunk != 0xFFFFFFFFu ? (uint32_t)found_cnt : (uint32_t)p.vocab - 1;
    };
    uint64_t total = 0;
    uint32_t last_at = 0xFFFFFFFFu;  // of the logits equal to the cut's, the last index kept
    if (cut.keep < cut.ties) {
        const unsigned need = cut.keep;
        last_at = select(of_key(cut.key), [&](uint32_t key, float, uint32_t) { return (uint64_t)(key == cut.key); },
                         [&](uint64_t s, uint64_t) { return s >= need; }, total);
    }
    const double least_weight = (double)min_p * (double)(1ull << ONE), u = (double)fminf(fmaxf(p.uniform[b], 0.0f), 0x1.fffffep-1f);
    // What min_p leaves lies above top + t · ln(min_p), less a ten-thousandth of t for all roundings (a weight's is half a unit of
    // thousands).
    float least_x = cut.key != 0 ? of_key(cut.key) : -INFINITY;
    if (min_p > 1e-9f && top < INFINITY) least_x = fmaxf(least_x, top - t * (1e-4f - logf(min_p)) - 1e-6f * fabsf(top));
    if (!(least_x <= top)) least_x = -INFINITY;
    const uint32_t token = select(
        least_x,
        [&](uint32_t key, float x, uint32_t at) -> uint64_t {
            const uint64_t w = weight(x);
            const bool taken = key > cut.key || (key == cut.key && at <= last_at);
            return taken && (key == top_key || (double)w >= least_weight) ? w : 0;
        },
        [&](uint64_t s, uint64_t all) { return (double)s > u * (double)all; }, total);
    if (tid == 0) {
        p.tokens[b] = (int32_t)token;
        if (p.logprobs) {
            const float x = row.one((int)token);
            const double d = x == top ? 0.0 : (top64 - (double)x) / (double)t;
            p.logprobs[b] = (float)(-d - log((double)total * 0x1p-43));
        }
    }
}

}  // namespace

hipError_t launch_sample(const SampleArgs &p, hipStream_t stream) {
    constexpr int64_t MOST = kMostThreads / THREADS;
    for (int64_t first = 0; first < p.rows; first += MOST) {
        SampleArgs part = p;
        part.logits = static_cast<const char *>(p.logits) + first * p.ld * (p.bf16 ? 2 : 4);
        part.uniform += first;
        if (p.temperature) part.temperature += first;
        if (p.top_p) part.top_p += first;
        if (p.min_p) part.min_p += first;
        if (p.top_k) part.top_k += first;
        part.tokens += first;
        if (p.logprobs) part.logprobs += first;
        const unsigned rows = (unsigned)(p.rows - first < MOST ? p.rows - first : MOST);
        if (p.bf16) hipLaunchKernelGGL(sample_kernel<true>, dim3(rows), dim3(THREADS), 0, stream, part);
        else hipLaunchKernelGGL(sample_kernel<false>, dim3(rows), dim3(THREADS), 0, stream, part);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace sq8
