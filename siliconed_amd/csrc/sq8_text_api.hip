// sq8_text_api.hip — the C ABI's text decoder operators (include/siliconed_q8.h): argument checks, staging of what
// the kernels do not read in place, status codes.
#include "siliconed_q8.h"

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "sq8_context.h"
#include "sq8_text.h"

namespace {

using sq8::aligned;
using sq8::DeviceScope;
using sq8::F8_GROUP;
using sq8::hip_status;
using sq8::reserve;

bool is_activation(int dtype) { return dtype == SQ8_BF16 || dtype == SQ8_F32; }
int groups_of(int k) { return (int)(((int64_t)k + F8_GROUP - 1) / F8_GROUP); }
int64_t up_to(int64_t v, int64_t step) { return (v + step - 1) / step * step; }

// `count` of the context's counters, zero between the calls that use them.
int reserve_marks(sq8_ctx *ctx, int64_t count, int *&marks) {
    const hipError_t e = sq8::reserve_cleared(ctx->marks, (size_t)count * sizeof(int), 65536, ctx->stream, ctx->aside, [&](void *at, size_t bytes) {
        return sq8::launch_zero_marks(static_cast<int *>(at), (int64_t)(bytes / sizeof(int)), ctx->stream);
    });
    if (e != hipSuccess) return hip_status(e);
    marks = static_cast<int *>(ctx->marks.at);
    return SQ8_OK;
}

struct F8Product {
    const void *a; int a_dtype; int64_t lda;    // SQ8_FP8_E4M3: codes with sx; else quantized here
    const float *sx; int64_t ldsx;
    const void *w; int64_t ldw;
    const float *sw; int64_t ldsw;
    const float *bias; int epilogue;
    void *c; int c_dtype; int64_t ldc;
    int m, k, n;
};

int run_f8(sq8_ctx *ctx, const F8Product &q, double *gpu_seconds) {
    if (!ctx || q.m < 0 || q.k < 0 || q.n < 0) return SQ8_EINVAL;
    if (q.epilogue != SQ8_EPI_NONE && q.epilogue != SQ8_EPI_SILU_GLU) return SQ8_EUNSUPPORTED;
    if (q.c_dtype != SQ8_BF16 && q.c_dtype != SQ8_F32) return SQ8_EUNSUPPORTED;
    const bool quantize = q.a_dtype != SQ8_FP8_E4M3;
    if (quantize && !is_activation(q.a_dtype)) return SQ8_EUNSUPPORTED;
    const bool glu = q.epilogue == SQ8_EPI_SILU_GLU;
    if (glu && q.n % 2 != 0) return SQ8_EINVAL;
    const int h = glu ? q.n / 2 : q.n, kb = groups_of(q.k);
    if (gpu_seconds) *gpu_seconds = 0.0;
    if (q.m == 0 || h == 0) return SQ8_OK;
    if (!q.c || q.ldc < h) return SQ8_EINVAL;
    if (q.k > 0 && (!q.a || !q.w || !q.sw || q.lda < q.k || q.ldw < q.k || q.ldsw < kb)) return SQ8_EINVAL;
    if (q.k > 0 && !quantize && (!q.sx || q.ldsx < kb)) return SQ8_EINVAL;

    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_status(scope.error);
    sq8::F8Args p;
    memset(&p, 0, sizeof(p));
    p.a = static_cast<const uint8_t *>(q.a);
    p.sx = q.sx;
    p.w = static_cast<const uint8_t *>(q.w);
    p.sw = q.sw;
    p.bias = q.bias;
    p.c = q.c;
    p.lda = q.lda; p.ldsx = q.ldsx; p.ldw = q.ldw; p.ldsw = q.ldsw; p.ldc = q.ldc;
    p.M = q.m; p.N = q.n; p.K = q.k; p.KB = kb; p.H = h;
    p.up_block = (h + F8_GROUP - 1) / F8_GROUP;
    const size_t esz = q.c_dtype == SQ8_F32 ? 4 : 2;
    p.c_vec = aligned(q.c, 8 * esz) && q.ldc % 8 == 0 ? 8 : aligned(q.c, 4 * esz) && q.ldc % 4 == 0 ? 4 : 0;

    // What the kernel does not read in place is copied first, rows padded with zero codes to whole 16-byte runs.
    const bool ragged = q.k % 16 != 0;
    const int64_t kp = up_to(q.k, 16);
    const bool pad_w = q.k > 0 && (ragged || !aligned(q.w, 16) || q.ldw % 16 != 0);
    const bool pad_a = q.k > 0 && !quantize && (ragged || !aligned(q.a, 16) || q.lda % 16 != 0);
    const int64_t scales_row = up_to(kb, 4);
    if (pad_w) {
        const int st = reserve(ctx, ctx->wpack, (size_t)(q.n * kp));
        if (st != SQ8_OK) return st;
    }
    if (quantize) p.lda = kp, p.ldsx = scales_row;
    if (pad_a) p.lda = kp;
    if (pad_w) p.ldw = kp;
    p.K = (int)kp;
    if (quantize && q.a_dtype == SQ8_BF16 && !ragged && aligned(q.a, 16) && q.lda % 8 == 0) {
        p.x = static_cast<const uint16_t *>(q.a);
        p.ldx = q.lda;
    }
    const sq8::F8Plan plan = sq8::f8_plan(p, glu, q.c_dtype == SQ8_F32, ctx->cus);
    const bool pass = quantize && !plan.values && q.k > 0;  // a quantization before the product
    if (pass || pad_a) {
        const int64_t codes = up_to((int64_t)q.m * kp, 16);
        const int st = reserve(ctx, ctx->scratch, (size_t)(codes + (pass ? q.m * scales_row * 4 : 0) + 16));
        if (st != SQ8_OK) return st;
    }
    if (plan.part_bytes > 0) {
        const int st = reserve(ctx, ctx->part, (size_t)plan.part_bytes);
        if (st != SQ8_OK) return st;
        p.part = static_cast<float *>(ctx->part.at);
        const int counted = reserve_marks(ctx, plan.marks, p.marks);
        if (counted != SQ8_OK) return counted;
    }
    hipError_t e = hipSuccess;
    if (gpu_seconds) e = hipEventRecord(ctx->begin, ctx->stream);
    if (e != hipSuccess) return hip_status(e);
    if (pass) {
        uint8_t *codes = static_cast<uint8_t *>(ctx->scratch.at);
        float *scales = reinterpret_cast<float *>(codes + up_to((int64_t)q.m * kp, 16));
        // Codes past k in a row's last run meet the weight's zero codes (its copy is padded with them), but must
        // not be NaN: cleared where there are any.
        if (ragged) {
            e = sq8::launch_pad_bytes(codes, kp, codes, kp, q.m, 0, ctx->stream);
            if (e != hipSuccess) return hip_status(e);
        }
        e = sq8::launch_quantize_groups(q.a, q.a_dtype == SQ8_BF16, q.lda, q.m, q.k, codes, kp, scales, scales_row, ctx->stream);
        if (e != hipSuccess) return e == hipErrorInvalidValue ? SQ8_EUNSUPPORTED : hip_status(e);
        p.a = codes;
        p.sx = scales;
    } else if (pad_a) {
        e = sq8::launch_pad_bytes(q.a, q.lda, ctx->scratch.at, kp, q.m, q.k, ctx->stream);
        if (e != hipSuccess) return hip_status(e);
        p.a = static_cast<const uint8_t *>(ctx->scratch.at);
    }
    if (pad_w) {
        e = sq8::launch_pad_bytes(q.w, q.ldw, ctx->wpack.at, kp, q.n, q.k, ctx->stream);
        if (e != hipSuccess) return hip_status(e);
        p.w = static_cast<const uint8_t *>(ctx->wpack.at);
    }
    p.sx_vec = aligned(p.sx, 16) && p.ldsx % 4 == 0 && (quantize || kb % 4 == 0);
    e = sq8::launch_f8_product(p, plan, glu, q.c_dtype == SQ8_F32, ctx->stream);
    if (e != hipSuccess) return e == hipErrorInvalidValue ? SQ8_EUNSUPPORTED : hip_status(e);
    if (gpu_seconds) {
        e = hipEventRecord(ctx->end, ctx->stream);
        if (e == hipSuccess) e = hipEventSynchronize(ctx->end);
        float ms = 0.0f;
        if (e == hipSuccess) e = hipEventElapsedTime(&ms, ctx->begin, ctx->end);
        if (e != hipSuccess) return hip_status(e);
        *gpu_seconds = ms * 1e-3;
    }
    return SQ8_OK;
}

int check_cache(const sq8_paged_cache *c, int q_heads) {
    if (!c || c->pages < 0 || c->page <= 0 || c->kv_heads <= 0 || c->dim <= 0 || q_heads <= 0) return SQ8_EINVAL;
    if (c->dtype != SQ8_BF16 && c->dtype != SQ8_FP8_E4M3) return SQ8_EUNSUPPORTED;
    if (c->pages > 0 && (!c->k || !c->v)) return SQ8_EINVAL;
    if (c->k_page < 0 || c->k_token < 0 || c->k_head < 0 || c->v_page < 0 || c->v_token < 0 || c->v_head < 0) return SQ8_EINVAL;
    return SQ8_OK;
}

}  // namespace

extern "C" {

int sq8_add_norm_quantized(sq8_ctx *ctx, const void *x, int x_dtype, int64_t ldx, const void *residual, int r_dtype,
                           int64_t ldr, void *residual_out, int64_t ldro, const float *w, float eps, void *codes,
                           int codes_dtype, int64_t ldq, float *scales, int64_t lds, int rows, int cols) {
    if (!ctx || rows < 0 || cols < 0) return SQ8_EINVAL;
    if (!is_activation(x_dtype) || (residual && !is_activation(r_dtype))) return SQ8_EUNSUPPORTED;
    if (codes_dtype != SQ8_FP8_E4M3 && codes_dtype != SQ8_INT8) return SQ8_EUNSUPPORTED;
    if (cols > sq8::kAddNormCols) return SQ8_EUNSUPPORTED;
    if (rows == 0 || cols == 0) return SQ8_OK;
    const bool int8 = codes_dtype == SQ8_INT8;
    if (!x || !w || !codes || !scales || ldx < cols || ldq < cols || (!int8 && lds < groups_of(cols))) return SQ8_EINVAL;
    if (residual ? ldr < cols || (residual_out && ldro < cols) : residual_out != nullptr) return SQ8_EINVAL;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_status(scope.error);
    sq8::AddNormArgs p;
    p.x = x; p.r = residual; p.ro = residual_out; p.w = w;
    p.codes = static_cast<uint8_t *>(codes);
    p.scales = scales;
    p.ldx = ldx; p.ldr = ldr; p.ldro = ldro; p.ldq = ldq; p.lds = lds;
    p.eps = eps;
    p.rows = rows; p.cols = cols;
    p.x_bf16 = x_dtype == SQ8_BF16; p.r_bf16 = r_dtype == SQ8_BF16;
    return hip_status(sq8::launch_add_norm(p, int8, ctx->cus, ctx->stream));
}

int sq8_quantize_groups(sq8_ctx *ctx, const void *x, int x_dtype, int64_t ldx, int rows, int cols, void *codes,
                        int64_t ldq, float *scales, int64_t lds) {
    if (!ctx || rows < 0 || cols < 0) return SQ8_EINVAL;
    if (!is_activation(x_dtype)) return SQ8_EUNSUPPORTED;
    if (rows == 0 || cols == 0) return SQ8_OK;
    if (!x || !codes || !scales || ldx < cols || ldq < cols || lds < groups_of(cols)) return SQ8_EINVAL;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_status(scope.error);
    const hipError_t e = sq8::launch_quantize_groups(x, x_dtype == SQ8_BF16, ldx, rows, cols, static_cast<uint8_t *>(codes),
                                                     ldq, scales, lds, ctx->stream);
    return e == hipErrorInvalidValue ? SQ8_EUNSUPPORTED : hip_status(e);
}

int sq8_linear_f8(sq8_ctx *ctx, const void *a, int64_t lda, const float *sx, int64_t ldsx, const void *w, int64_t ldw,
                  const float *sw, int64_t ldsw, const float *bias, int epilogue, void *c, int c_dtype, int64_t ldc, int m,
                  int k, int n, double *gpu_seconds) {
    const F8Product q = {a, SQ8_FP8_E4M3, lda, sx, ldsx, w, ldw, sw, ldsw, bias, epilogue, c, c_dtype, ldc, m, k, n};
    return run_f8(ctx, q, gpu_seconds);
}

int sq8_linear_f8_quantized(sq8_ctx *ctx, const void *a, int a_dtype, int64_t lda, const void *w, int64_t ldw,
                            const float *sw, int64_t ldsw, const float *bias, int epilogue, void *c, int c_dtype,
                            int64_t ldc, int m, int k, int n, double *gpu_seconds) {
    if (!is_activation(a_dtype)) return SQ8_EUNSUPPORTED;
    const F8Product q = {a, a_dtype, lda, nullptr, 0, w, ldw, sw, ldsw, bias, epilogue, c, c_dtype, ldc, m, k, n};
    return run_f8(ctx, q, gpu_seconds);
}

int sq8_append_kv(sq8_ctx *ctx, const uint16_t *q, int64_t q_token, int64_t q_head, const uint16_t *k, int64_t k_token,
                  int64_t k_head, const uint16_t *v, int64_t v_token, int64_t v_head, uint16_t *q_out, int64_t qo_token,
                  int64_t qo_head, const sq8_paged_cache *cache, const int32_t *positions, const int32_t *slots,
                  const float *table, int64_t table_row, int max_position, int rot, int interleaved, int tokens, int q_heads) {
    if (!ctx || tokens < 0 || rot < 0) return SQ8_EINVAL;
    const int st = check_cache(cache, q_heads);
    if (st != SQ8_OK) return st;
    if (rot > cache->dim) return SQ8_EINVAL;
    if (cache->dim % 2 != 0 || rot % 2 != 0) return SQ8_EUNSUPPORTED;
    if (tokens == 0) return SQ8_OK;
    if (!q || !k || !v || !q_out || !slots || (rot > 0 && (!positions || !table || max_position <= 0 || table_row < rot)))
        return SQ8_EINVAL;
    if (q_token < 0 || q_head < 0 || k_token < 0 || k_head < 0 || v_token < 0 || v_head < 0 || qo_token < 0 || qo_head < 0)
        return SQ8_EINVAL;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_status(scope.error);
    const bool e4m3 = cache->dtype == SQ8_FP8_E4M3;
    sq8::AppendArgs p;
    p.q = q; p.k = k; p.v = v; p.q_out = q_out;
    p.kc = cache->k; p.vc = cache->v;
    p.k_scale = cache->k_scale; p.v_scale = cache->v_scale;
    p.table = table; p.positions = positions; p.slots = slots;
    p.q_tok = q_token; p.q_head = q_head; p.k_tok = k_token; p.k_head = k_head; p.v_tok = v_token; p.v_head = v_head;
    p.qo_tok = qo_token; p.qo_head = qo_head;
    p.kc_page = cache->k_page; p.kc_tok = cache->k_token; p.kc_head = cache->k_head;
    p.vc_page = cache->v_page; p.vc_tok = cache->v_token; p.vc_head = cache->v_head;
    p.table_row = table_row;
    p.slot_count = (int64_t)cache->pages * cache->page;
    p.tokens = tokens; p.q_heads = q_heads; p.kv_heads = cache->kv_heads; p.dim = cache->dim; p.rot = rot;
    p.page = cache->page; p.max_position = max_position; p.interleaved = interleaved != 0;
    const hipError_t e = sq8::launch_append_kv(p, e4m3, ctx->stream);
    return e == hipErrorInvalidValue ? SQ8_EUNSUPPORTED : hip_status(e);
}

int sq8_paged_attention(sq8_ctx *ctx, const uint16_t *q, int64_t q_token, int64_t q_head, const sq8_paged_cache *cache,
                        const int32_t *table, int64_t table_row, int max_pages, const int32_t *lengths, float scale,
                        float softcap, int window, uint16_t *out, int64_t o_token, int64_t o_head, int batch, int q_heads) {
    if (!ctx || batch < 0 || max_pages < 0 || window < 0 || !(softcap >= 0.0f)) return SQ8_EINVAL;
    int st = check_cache(cache, q_heads);
    if (st != SQ8_OK) return st;
    if (q_heads % cache->kv_heads != 0) return SQ8_EINVAL;
    // A cap that no score comes near is none (c · tanh(s / c) is s in fp32, and c · log2(e) may overflow). Capped by less
    // than 2^-60, every exponential is 1: as good by 2^-60, whose reciprocal does not overflow.
    if (softcap > 0x1p100f) softcap = 0.0f;
    else if (softcap > 0.0f && softcap < 0x1p-60f) softcap = 0x1p-60f;
    const bool e4m3 = cache->dtype == SQ8_FP8_E4M3;
    if (cache->dim > 256 || cache->dim % (e4m3 || cache->dim > 128 ? 16 : 8) != 0) return SQ8_EUNSUPPORTED;
    // Token numbers, and the tiles of a batch over its heads, are 32-bit.
    if ((int64_t)max_pages * cache->page > INT32_MAX - 4096 ||
        (double)((int64_t)max_pages * cache->page / 128 + 2) * q_heads * batch > INT32_MAX)
        return SQ8_EUNSUPPORTED;
    if (batch == 0) return SQ8_OK;
    if (!q || !out || !lengths || q_token < 0 || q_head < 0 || o_token < 0 || o_head < 0) return SQ8_EINVAL;
    if (max_pages > 0 && (!table || table_row < max_pages)) return SQ8_EINVAL;
    // Pages to read with no pool to read them from.
    if (max_pages > 0 && cache->pages == 0) max_pages = 0;
    const int64_t caches = cache->k_page | cache->k_token | cache->k_head | cache->v_page | cache->v_token | cache->v_head;
    if (!aligned(q, 16) || !aligned(out, 4) || (q_token | q_head) % 8 != 0 || (o_token | o_head) % 2 != 0 ||
        !aligned(cache->k, 16) || !aligned(cache->v, 16) || caches % (e4m3 ? 16 : 8) != 0)
        return SQ8_EUNSUPPORTED;
    DeviceScope scope(ctx->device);
    if (scope.error != hipSuccess) return hip_status(scope.error);
    sq8::PagedArgs p;
    memset(&p, 0, sizeof(p));
    p.q = q;
    p.kc = static_cast<const uint8_t *>(cache->k);
    p.vc = static_cast<const uint8_t *>(cache->v);
    p.k_scale = cache->k_scale; p.v_scale = cache->v_scale;
    p.pages = table; p.lengths = lengths; p.out = out;
    p.q_tok = q_token; p.q_head = q_head; p.o_tok = o_token; p.o_head = o_head;
    p.kc_page = cache->k_page; p.kc_tok = cache->k_token; p.kc_head = cache->k_head;
    p.vc_page = cache->v_page; p.vc_tok = cache->v_token; p.vc_head = cache->v_head;
    p.pages_row = table_row;
    p.scale = scale; p.softcap = softcap;
    p.batch = batch; p.q_heads = q_heads; p.kv_heads = cache->kv_heads; p.dim = cache->dim;
    p.page = cache->page; p.page_count = cache->pages; p.max_pages = max_pages; p.window = window;
    sq8::page_divisor(p);
    const int groups = sq8::paged_groups(p, ctx->cus);
    const int64_t bytes = sq8::paged_part_bytes(p, groups);
    if (bytes > 0) {
        st = reserve(ctx, ctx->part, (size_t)bytes);
        if (st != SQ8_OK) return st;
        p.part = static_cast<float *>(ctx->part.at);
        st = reserve_marks(ctx, sq8::paged_marks(p), p.marks);
        if (st != SQ8_OK) return st;
    }
    return hip_status(sq8::launch_paged_attention(p, e4m3, groups, ctx->stream));
}

}  // extern "C"
