// sq8_text.h — host/device interface of a text decoder's operators: the norm that adds the residual stream and
// writes 8-bit codes, products of e4m3 codes with a scale per 128 of K, the paged cache's append with the position
// rotation, attention of one new token over that cache, heads normed and turned, attention of prompts and
// chunks, and the draw of a token.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sq8 {

constexpr int F8_GROUP = 128;  // values of K that share a scale
// A launch's threads. (Of 2^32 or more the runtime starts what is left of their number without it, and says nothing.)
constexpr int64_t kMostThreads = UINT32_MAX;

// Correctly rounded quotients by one divisor s: from r = fl(1/s), q0 = fl(y·r) is within two ulps, one step
// q1 = q0 + r·(y − q0·s) within one, and the next is then the rounded quotient (Markstein 1990: r correctly rounded,
// q1 faithful, both steps fused). Four multiply-adds where a division is ten instructions. An infinite s: 0, or NaN
// for an infinite y (the remainder takes s as 0 there, as 0 · ∞ is NaN).
struct Quotient {
    float s, r;
    __device__ __forceinline__ explicit Quotient(float by) : s(fabsf(by) == INFINITY ? 0.0f : by), r(__fdiv_rn(1.0f, by)) {}
    __device__ __forceinline__ float of(float y) const {
        const float q0 = y * r;
        const float q1 = __builtin_fmaf(__builtin_fmaf(-q0, s, y), r, q0);
        return __builtin_fmaf(__builtin_fmaf(-q1, s, y), r, q1);
    }
};

// The counters that tell the last of several workgroups lie a line apart: side by side they held each other up (the
// attention of two sequences of 8192 took 22 µs, and 18 so).
constexpr int MARK = 32;

// Partial results lie where every XCD sees them: written and read past its own L2 (agent-scope accesses), so that the
// workgroup that joins them needs no fence, which would write back and drop that cache under everything still
// streaming through it (with fences the attention took twice as long at 48 sequences of up to 8192).
struct Pair {
    float a, b;
};
__device__ __forceinline__ void put(float *to, Pair v) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(to), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Pair get(const float *from) {
    return __builtin_bit_cast(Pair, __hip_atomic_load(reinterpret_cast<const uint64_t *>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// sq8_text_norm.hip. Element types by flag: bf16 or fp32.
struct AddNormArgs {
    const void *x;          // [rows, cols]
    const void *r;          // the residual stream, or null
    void *ro;               // the stream's sum (r's type), or null; may be r
    const float *w;         // [cols]
    uint8_t *codes;         // e4m3 or int8 [rows, cols]
    float *scales;          // e4m3: [rows, ⌈cols/128⌉]; int8: [rows]
    int64_t ldx, ldr, ldro, ldq, lds;
    float eps;
    int rows, cols;
    int x_bf16, r_bf16;
};
constexpr int kAddNormCols = 32768;
hipError_t launch_add_norm(const AddNormArgs &p, bool int8, int cus, hipStream_t stream);
hipError_t launch_quantize_groups(const void *x, bool x_bf16, int64_t ldx, int rows, int cols, uint8_t *codes, int64_t ldq,
                                  float *scales, int64_t lds, hipStream_t stream);
// rows × n bytes read lds apart → written ldd apart (n ≤ ldd; bytes [n, ldd) zero).
hipError_t launch_pad_bytes(const void *src, int64_t lds, void *dst, int64_t ldd, int64_t rows, int64_t n,
                            hipStream_t stream);

// sq8_f8_gemm.hip.
struct F8Args {
    const uint8_t *a;       // e4m3 [M, K], rows lda apart, 16-byte aligned rows
    const float *sx;        // [M, KB], rows ldsx apart
    const uint16_t *x;      // or null; bf16 [M, K], rows ldx apart, 16-byte aligned rows, that a and sx are to be of
    const uint8_t *w;       // e4m3 [N, K], rows ldw apart, 16-byte aligned rows
    const float *sw;        // [⌈N/128⌉ (GLU: 2⌈H/128⌉), KB], rows ldsw apart
    const float *bias;      // [N] or null
    void *c;                // [M, n_out]
    float *part;            // the sums of a split K's parts
    int *marks;             // the tiles' counters of parts that are done, zero between calls
    int64_t lda, ldsx, ldx, ldw, ldsw, ldc;
    int M, N, K;            // K a multiple of 16
    int KB;                 // ⌈K/128⌉
    int H;                  // the output's width: N, or N/2 for GLU
    int up_block;           // ⌈H/128⌉: the scale rows of a half, and the up half's first
    int c_vec;              // outputs a store may take: 8 or 4 (aligned base and rows), 0 for one at a time
    int sx_vec;             // four scales a load allowed (rows of whole fours)
};
// A product's kernels: the tiles (F8_128_ONE: one workgroup a CU), the short kernel of 16 and of 32 columns, rows too far
// apart for the tiles' offsets, and the short kernel that quantizes its values, of 16 and of 32 columns.
enum { F8_256 = 0, F8_128, F8_128_ONE, F8_64x128, F8_64, F8_TILES, F8_SHORT = F8_TILES, F8_SHORT_WIDE, F8_FAR, F8_STAGED, F8_STAGED_WIDE };
constexpr int F8_STAGED_GROUPS = 128;  // groups of 128 values that the staged kernel takes
// sq8_text_plan.hip. Which kernel a product runs on, and the parts its K is split in; part_bytes, marks: what F8Args::part
// and ::marks need.
struct F8Plan {
    int kernel, splits;
    int64_t part_bytes, marks;
    bool values;  // the kernel takes F8Args::x; else a and sx are to be there
};
F8Plan f8_plan(const F8Args &p, bool glu, bool out_f32, int cus);
hipError_t launch_f8_product(const F8Args &p, const F8Plan &plan, bool glu, bool out_f32, hipStream_t stream);

// sq8_paged.hip. Strides in elements.
struct AppendArgs {
    const uint16_t *q, *k, *v;          // bf16 [tokens, heads, dim]
    uint16_t *q_out;
    void *kc, *vc;                      // [pages, page, kv_heads, dim], bf16 or e4m3
    const float *k_scale, *v_scale;     // [kv_heads] or null (1); e4m3 only
    const float *table;                 // [positions, rot]: rot/2 cosines, then as many sines
    const int32_t *positions, *slots;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;
    int64_t kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head, table_row;
    int64_t slot_count;                 // pages · page
    int tokens, q_heads, kv_heads, dim, rot, page, max_position;
    int interleaved;
};
hipError_t launch_append_kv(const AppendArgs &p, bool e4m3, hipStream_t stream);

struct PagedArgs {
    const uint16_t *q;                  // bf16 [batch, q_heads, dim]
    const uint8_t *kc, *vc;             // as AppendArgs
    const float *k_scale, *v_scale;
    const int32_t *pages;               // [batch, max_pages], rows pages_row apart
    const int32_t *lengths;             // [batch]
    uint16_t *out;
    float *part;                        // partial results of split sequences: paged_part_bytes() bytes
    int *marks;                         // paged_marks() counters, zero before and after every call
    int64_t q_tok, q_head, o_tok, o_head;
    int64_t kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head, pages_row;
    float scale, softcap;
    int batch, q_heads, kv_heads, dim, page, page_count, max_pages, window;
    uint64_t page_mul;                  // page_divisor()'s
    int page_shift;
};
constexpr int PAGED_TILE = 128;  // tokens a workgroup takes at a time
constexpr int paged_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }  // the instance of a head's size
constexpr int paged_held(int dp) { return dp <= 128 ? 2 : 1; }                        // workgroups a CU holds (by their registers)
// A slot: maxima and sums [16][2], outputs [dp / 32][4][4][live][2]: pair, register and row of the first wave's lanes, head.
__host__ __device__ constexpr int paged_part_floats(int dp) { return 32 + 16 * dp; }
// sq8_text_plan.hip.
void page_divisor(int page, uint64_t &mul, int &shift);
// The workgroups a call of these sizes takes, and the partial results' bytes they need.
int paged_groups(const PagedArgs &p, int cus);
int64_t paged_part_bytes(const PagedArgs &p, int groups);
int64_t paged_marks(const PagedArgs &p);
hipError_t launch_zero_marks(int *marks, int64_t count, hipStream_t stream);
hipError_t launch_paged_attention(const PagedArgs &p, bool e4m3, int groups, hipStream_t stream);

// sq8_heads.hip. Strides in elements.
struct HeadsArgs {
    const uint16_t *q, *k, *v;          // bf16 [tokens, heads, dim]; v with a cache only
    uint16_t *q_out, *k_out;            // k_out without a cache only
    void *kc, *vc;                      // the cache's pools, or null
    const float *k_scale, *v_scale;
    const float *q_norm, *k_norm;       // [dim], or null: not normed
    const float *table;                 // as AppendArgs
    const int32_t *positions, *slots;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head, ko_tok, ko_head;
    int64_t kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head, table_row;
    int64_t slot_count;
    float eps;
    int tokens, q_heads, kv_heads, dim, rot, page, max_position;
    int interleaved;
    int lanes_log;                      // launch_norm_heads' own
};
constexpr int kNormHeadDim = 512;
hipError_t launch_norm_heads(HeadsArgs p, bool e4m3, hipStream_t stream);

// sq8_attend_kernel.h: attention of prompts over their own keys and values (pages null), or of chunks over a paged cache.
struct AttendArgs {
    const uint16_t *q;                  // bf16 [tokens, q_heads, dim]
    const uint8_t *kc, *vc;             // bf16 [tokens, kv_heads, dim] (kc_page unused), or the cache's pools
    const float *k_scale, *v_scale;
    const int32_t *starts;              // [sequences + 1], or null: one sequence of all tokens
    const int32_t *pages;               // [sequences, max_pages]
    const int32_t *lengths;             // [sequences]
    uint16_t *out;
    float *part;                        // partial results of shared units
    int *marks;                         // a counter a workgroup, zero before and after every call
    int64_t q_tok, q_head, o_tok, o_head;
    int64_t kc_page, kc_tok, kc_head, vc_page, vc_tok, vc_head, pages_row;
    float scale, softcap;
    int tokens, sequences, kv_heads, group, dim, page, page_count, max_pages, window, causal;
    int share;                          // units are shared out over the workgroups
    uint64_t page_mul;
    int page_shift;
};
constexpr int attend_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }  // the instance of a head's size
// Tokens of a tile that WT waves share, and the tiles that LDS holds (a slot of 64 tokens of 128 values or 32 of 256: 32 KB).
constexpr int attend_tokens(int wt) { return 32 * wt; }
constexpr int kAttendStages = 4;
// Waves a SIMD holds.
constexpr int attend_waves(int dp, int wt) { return dp * wt >= 256 ? 1 : 2; }
// sq8_chunk.hip: workgroups of `rows` rows (16 nc) that a CU holds, by their registers and LDS.
constexpr int chunk_held(int dp, int nc) { return dp < 256 && dp * nc <= 256 ? 2 : 1; }
// A slot of a shared unit: maxima and sums [rows][2], outputs.
__host__ __device__ constexpr int attend_part_floats(int dp, int rows) { return rows * (2 + dp); }
// sq8_text_plan.hip. The tile and the workgroups that a call takes, and what it needs of the context's buffers.
struct AttendPlan {
    int rows;                   // of a tile; narrow: of sq8_chunk.hip
    int groups, share, narrow;
    int64_t part_bytes, marks;
    double tiles;               // of all units, at most
    int threads;                // of a workgroup
};
AttendPlan attend_plan(const AttendArgs &p, bool e4m3, int cus);
hipError_t launch_attend(const AttendArgs &p, const AttendPlan &plan, bool e4m3, hipStream_t stream);
namespace attend {
// Where keys and values lie: rows of a projection; pages whose tokens are a multiple of 16 (16 tokens lie in one page); any
// pages; in bf16 or e4m3.
enum Source { ROWS = 0, PAGES16, PAGES, PAGES16_F8, PAGES_F8 };
hipError_t launch_chunk(const AttendArgs &p, const AttendPlan &plan, bool e4m3, hipStream_t stream);
template <int SOURCE>
hipError_t launch_source(const AttendArgs &p, const AttendPlan &plan, hipStream_t stream);
}  // namespace attend

// sq8_sample.hip.
struct SampleArgs {
    const void *logits;                 // [rows, vocab], rows ld apart, bf16 or fp32
    const float *uniform;               // [rows]
    const float *temperature, *top_p, *min_p;  // [rows] or null
    const int32_t *top_k;               // [rows] or null
    int32_t *tokens;                    // [rows]
    float *logprobs;                    // [rows] or null
    int64_t ld;
    int rows, vocab, bf16;
};
constexpr int kSampleVocab = 1 << 20;
hipError_t launch_sample(const SampleArgs &p, hipStream_t stream);

}  // namespace sq8
