// text_bind.cpp — the text decoder's operators from Python: a call's tensors are checked, its outputs allocated and
// the C ABI's entry called in one native step. At one token a kernel takes 3 to 8 µs, and the same in Python (a dozen
// attributes of tensors, two allocations, a foreign call of twenty arguments) took 9 to 13: the calls, not the GPU,
// set the pace of a decoder.
//
// The library is loaded by _abi.py, which hands over its entries' addresses (bind) when a text operator is first
// called: nothing else of the library needs this module. A function here returns its
// outputs, or the status of a call that the library refused, an int, for _abi.py to raise. A tensor that does not fit
// raises ValueError.
#include <Python.h>
#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "siliconed_q8.h"

namespace {

using at::Tensor;

struct Entries {
    decltype(&sq8_add_norm_quantized) add_norm_quantized;
    decltype(&sq8_quantize_groups) quantize_groups;
    decltype(&sq8_linear_f8) linear_f8;
    decltype(&sq8_linear_f8_quantized) linear_f8_quantized;
    decltype(&sq8_append_kv) append_kv;
    decltype(&sq8_paged_attention) paged_attention;
    decltype(&sq8_norm_append_kv) norm_append_kv;
    decltype(&sq8_norm_rotate) norm_rotate;
    decltype(&sq8_prompt_attention) prompt_attention;
    decltype(&sq8_chunk_attention) chunk_attention;
    decltype(&sq8_sample_tokens) sample_tokens;
    decltype(&sq8_device) device;
} entries;

constexpr int64_t kGroup = 128;  // values of K that share a scale
constexpr auto kF8 = at::kFloat8_e4m3fn;

int64_t groups(int64_t k) { return (k + kGroup - 1) / kGroup; }

const Tensor &tensor(PyObject *o, const char *what) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
    return THPVariable_Unpack(o);
}
// A tensor or None.
const Tensor *maybe(PyObject *o, const char *what) { return o == Py_None ? nullptr : &tensor(o, what); }

int count32(int64_t v, const char *what) {
    TORCH_CHECK_VALUE(v <= INT32_MAX, what, " has more than 2^31 - 1 rows, columns or heads");
    return (int)v;
}

// The row stride of a matrix on the GPU whose rows are contiguous.
int64_t rows_of(const Tensor &t, const char *what) {
    TORCH_CHECK_VALUE(t.is_cuda(), what, " must be on the GPU");
    TORCH_CHECK_VALUE(t.dim() == 2, what, " must be 2-D, not ", t.sizes());
    const int64_t rows = t.size(0), cols = t.size(1);
    TORCH_CHECK_VALUE(t.stride(1) == 1 || cols <= 1 || rows == 0, what, " must have contiguous rows");
    return rows > 1 ? t.stride(0) : std::max<int64_t>(cols, 1);
}
int64_t rows_of(const Tensor &t, const char *what, int64_t rows, int64_t cols) {
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, what, " must be [", rows, ", ", cols, "], not ",
                      t.sizes());
    return rows_of(t, what);
}

int activation(const Tensor &t, const char *what) {
    const auto type = t.scalar_type();
    TORCH_CHECK_VALUE(type == at::kBFloat16 || type == at::kFloat, what, " must be bfloat16 or float32, not ", type);
    return type == at::kFloat ? SQ8_F32 : SQ8_BF16;
}

// A contiguous vector's address.
template <typename T>
const T *vector_of(const Tensor &t, int64_t count, const char *what) {
    constexpr auto type = std::is_same<T, float>::value ? at::kFloat : at::kInt;
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.numel() == count && t.is_contiguous() && t.is_cuda(), what, " must be ", count,
                      " contiguous ", type, " values on the GPU");
    return static_cast<const T *>(t.data_ptr());
}

// bf16 [rows, heads, dim], a head's values contiguous.
struct Heads {
    uint16_t *at;
    int64_t row, head;
};
Heads heads_of(const Tensor &t, const char *what, int64_t rows, int64_t heads, int64_t dim) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 && t.dim() == 3 && t.size(0) == rows && t.size(1) == heads &&
                          t.size(2) == dim && t.is_cuda(),
                      what, " must be bfloat16 [", rows, ", ", heads, ", ", dim, "] on the GPU, not ", t.scalar_type(), " ", t.sizes());
    TORCH_CHECK_VALUE(t.stride(2) == 1 || dim <= 1, what, " must have contiguous heads");
    // (Torch leaves the stride of a dimension of one anything.)
    return {static_cast<uint16_t *>(t.data_ptr()), rows > 1 ? t.stride(0) : 0, heads > 1 ? t.stride(1) : 0};
}
int64_t queries(const Tensor &q) {
    TORCH_CHECK_VALUE(q.dim() == 3, "q must be [tokens, heads, dim], not ", q.sizes());
    return q.size(0);
}

// What a ctypes object holds: the context's handle, a cache's description.
template <typename T>
T held(PyObject *o, const char *what) {
    Py_buffer view;
    TORCH_CHECK_TYPE(PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) == 0, what, " expected");
    const bool fits = view.len == (Py_ssize_t)sizeof(T);
    T value{};
    if (fits) memcpy(&value, view.buf, sizeof(T));
    PyBuffer_Release(&view);
    TORCH_CHECK_TYPE(fits, what, " expected");
    return value;
}
sq8_ctx *context(PyObject *o) { return o == Py_None ? nullptr : held<sq8_ctx *>(o, "a context"); }

// A call's tensors lie on the context's GPU: the kernels would fault on another's addresses. (A null context is the
// library's to refuse.)
struct Named {
    const Tensor *t;
    const char *what;
};
void on_device(const sq8_ctx *ctx, std::initializer_list<Named> all) {
    if (!ctx) return;
    const int device = entries.device(ctx);
    for (const Named &n : all)
        TORCH_CHECK_VALUE(!n.t || n.t->get_device() == device, n.what, " must be on the context's GPU, cuda:", device, ", not ",
                          n.t->device());
}

double number(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
bool truth(PyObject *o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v != 0;
}
int integer(PyObject *o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, "an argument is out of range");
    return (int)v;
}

// The entry's call without the interpreter's lock.
template <typename F>
int call(F &&f) {
    PyThreadState *const state = PyEval_SaveThread();
    const int status = f();
    PyEval_RestoreThread(state);
    return status;
}

PyObject *give(Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject *same(PyObject *o) {
    Py_INCREF(o);
    return o;
}

void expect(Py_ssize_t given, Py_ssize_t wanted) { TORCH_CHECK_TYPE(given == wanted, wanted, " arguments expected, not ", given); }

// ctx, x, w, eps, residual, residual_out, int8, codes, scales → (codes, scales, residual_out)
PyObject *add_norm_quantized(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &x = tensor(a[1], "x"), &w = tensor(a[2], "w");
    const float eps = (float)number(a[3]);
    const Tensor *const residual = maybe(a[4], "residual");
    PyObject *const out = a[5] == Py_None ? a[4] : a[5];
    const Tensor *const residual_out = maybe(out, "residual_out");
    const bool int8 = truth(a[6]);
    const int64_t ldx = rows_of(x, "x"), rows = x.size(0), cols = x.size(1);
    const auto type = int8 ? at::kChar : kF8;
    Tensor codes, scales;
    if (a[7] == Py_None) {
        codes = at::empty({rows, cols}, x.options().dtype(type));
    } else {
        codes = tensor(a[7], "codes");
        TORCH_CHECK_VALUE(codes.scalar_type() == type, "codes must be ", type);
    }
    const int64_t ldq = rows_of(codes, "codes", rows, cols);
    int64_t lds = 0;
    if (a[8] != Py_None) scales = tensor(a[8], "scales");
    else if (int8) scales = at::empty({rows}, x.options().dtype(at::kFloat));
    else scales = at::empty({rows, groups(cols)}, x.options().dtype(at::kFloat));
    if (int8) {
        vector_of<float>(scales, rows, "scales");
    } else {
        TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat, "scales must be float32");
        lds = rows_of(scales, "scales", rows, groups(cols));
    }
    const void *r = nullptr;
    void *ro = nullptr;
    int r_type = 0;
    int64_t ldr = 0, ldro = 0;
    if (residual) {
        TORCH_CHECK_VALUE(residual_out->scalar_type() == residual->scalar_type(), "residual_out must be of the residual's type");
        r = residual->data_ptr();
        r_type = activation(*residual, "residual");
        ldr = rows_of(*residual, "residual", rows, cols);
        ro = residual_out->data_ptr();
        ldro = rows_of(*residual_out, "residual_out", rows, cols);
    } else {
        TORCH_CHECK_VALUE(!residual_out, "residual_out needs a residual");
    }
    const float *const weights = vector_of<float>(w, cols, "w");
    const int x_type = activation(x, "x"), r32 = count32(rows, "x"), c32 = count32(cols, "x");
    on_device(ctx, {{&x, "x"}, {&w, "w"}, {residual, "residual"}, {residual_out, "residual_out"}, {&codes, "codes"}, {&scales, "scales"}});
    const int status = call([&] {
        return entries.add_norm_quantized(ctx, x.data_ptr(), x_type, ldx, r, r_type, ldr, ro, ldro, weights, eps, codes.data_ptr(),
                                          int8 ? SQ8_INT8 : SQ8_FP8_E4M3, ldq, static_cast<float *>(scales.data_ptr()), lds, r32, c32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    PyObject *const all = PyTuple_New(3);
    if (!all) throw python_error();
    PyTuple_SET_ITEM(all, 0, a[7] == Py_None ? give(std::move(codes)) : same(a[7]));
    PyTuple_SET_ITEM(all, 1, a[8] == Py_None ? give(std::move(scales)) : same(a[8]));
    PyTuple_SET_ITEM(all, 2, same(out));
    return all;
    END_HANDLE_TH_ERRORS
}

// ctx, x, codes, scales → (codes, scales)
PyObject *quantize_groups(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 4);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &x = tensor(a[1], "x");
    const int64_t ldx = rows_of(x, "x"), rows = x.size(0), cols = x.size(1);
    Tensor codes = a[2] == Py_None ? at::empty({rows, cols}, x.options().dtype(kF8)) : tensor(a[2], "codes");
    Tensor scales = a[3] == Py_None ? at::empty({rows, groups(cols)}, x.options().dtype(at::kFloat)) : tensor(a[3], "scales");
    TORCH_CHECK_VALUE(codes.scalar_type() == kF8 && scales.scalar_type() == at::kFloat, "codes must be float8_e4m3fn, scales float32");
    const int64_t ldq = rows_of(codes, "codes", rows, cols), lds = rows_of(scales, "scales", rows, groups(cols));
    const int x_type = activation(x, "x"), r32 = count32(rows, "x"), c32 = count32(cols, "x");
    on_device(ctx, {{&x, "x"}, {&codes, "codes"}, {&scales, "scales"}});
    const int status = call([&] {
        return entries.quantize_groups(ctx, x.data_ptr(), x_type, ldx, r32, c32, codes.data_ptr(), ldq,
                                       static_cast<float *>(scales.data_ptr()), lds);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    PyObject *const all = PyTuple_New(2);
    if (!all) throw python_error();
    PyTuple_SET_ITEM(all, 0, a[2] == Py_None ? give(std::move(codes)) : same(a[2]));
    PyTuple_SET_ITEM(all, 1, a[3] == Py_None ? give(std::move(scales)) : same(a[3]));
    return all;
    END_HANDLE_TH_ERRORS
}

// ctx, a, sx (None: a is quantized first), w, scale, bias, glu, out, f32, timed → out, or (out, seconds)
PyObject *product_f8(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &x = tensor(a[1], "the activation"), &w = tensor(a[3], "w"), &scale = tensor(a[4], "scale");
    const Tensor *const sx = maybe(a[2], "sx"), *const bias = maybe(a[5], "bias");
    const bool glu = truth(a[6]), f32 = truth(a[8]), timed = truth(a[9]);
    const int64_t lda = rows_of(x, "the activation"), m = x.size(0), k = x.size(1);
    int64_t ldsx = 0;
    if (sx) {
        TORCH_CHECK_VALUE(x.scalar_type() == kF8 && sx->scalar_type() == at::kFloat,
                          "codes must be float8_e4m3fn [m, k], sx float32 [m, ceil(k / 128)]");
        ldsx = rows_of(*sx, "sx", m, groups(k));
    }
    const int x_type = sx ? (int)SQ8_FP8_E4M3 : activation(x, "x");
    TORCH_CHECK_VALUE(w.scalar_type() == kF8 && w.dim() == 2, "w must be float8_e4m3fn codes [n, k]");
    const int64_t wide = w.size(0), ldw = rows_of(w, "w", wide, k);
    TORCH_CHECK_VALUE(!glu || wide % 2 == 0, "a GLU weight has an even number of rows");
    const int64_t h = glu ? wide / 2 : wide;
    TORCH_CHECK_VALUE(scale.scalar_type() == at::kFloat, "scale must be float32");
    const int64_t lds = rows_of(scale, "scale", glu ? 2 * groups(h) : groups(h), groups(k));
    const float *const b = bias ? vector_of<float>(*bias, wide, "bias") : nullptr;
    Tensor out = a[7] != Py_None ? tensor(a[7], "out") : at::empty({m, h}, x.options().dtype(f32 ? at::kFloat : at::kBFloat16));
    const int64_t ldc = rows_of(out, "out", m, h);
    const int c_type = activation(out, "out"), epilogue = glu ? SQ8_EPI_SILU_GLU : SQ8_EPI_NONE;
    const int m32 = count32(m, "the activation"), k32 = count32(k, "w"), n32 = count32(wide, "w");
    double seconds = 0.0, *const at = timed ? &seconds : nullptr;
    const uint8_t *const codes = static_cast<const uint8_t *>(w.data_ptr());
    const float *const sw = static_cast<const float *>(scale.data_ptr());
    on_device(ctx, {{&x, "the activation"}, {sx, "sx"}, {&w, "w"}, {&scale, "scale"}, {bias, "bias"}, {&out, "out"}});
    const int status = call([&] {
        return sx ? entries.linear_f8(ctx, x.data_ptr(), lda, static_cast<const float *>(sx->data_ptr()), ldsx, codes, ldw, sw, lds, b,
                                      epilogue, out.data_ptr(), c_type, ldc, m32, k32, n32, at)
                  : entries.linear_f8_quantized(ctx, x.data_ptr(), x_type, lda, codes, ldw, sw, lds, b, epilogue, out.data_ptr(),
                                                c_type, ldc, m32, k32, n32, at);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    PyObject *const result = a[7] == Py_None ? give(std::move(out)) : same(a[7]);
    return timed ? Py_BuildValue("(Nd)", result, seconds) : result;
    END_HANDLE_TH_ERRORS
}

// ctx, q, k, v, cache, positions, slots, table, q_out, interleaved → q_out
PyObject *append_kv(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
    const sq8_paged_cache cache = held<sq8_paged_cache>(a[4], "a cache's description");
    const Tensor &positions = tensor(a[5], "positions"), &slots = tensor(a[6], "slots"), &table = tensor(a[7], "table");
    const int64_t tokens = queries(q), heads = q.size(1);
    Tensor out = a[8] == Py_None ? at::empty({tokens, heads, cache.dim}, q.options()) : tensor(a[8], "q_out");
    const Heads qh = heads_of(q, "q", tokens, heads, cache.dim), kh = heads_of(k, "k", tokens, cache.kv_heads, cache.dim);
    const Heads vh = heads_of(v, "v", tokens, cache.kv_heads, cache.dim), oh = heads_of(out, "q_out", tokens, heads, cache.dim);
    TORCH_CHECK_VALUE(table.scalar_type() == at::kFloat, "table must be float32 [positions, rot]");
    const int64_t row = rows_of(table, "table");
    const int32_t *const at = vector_of<int32_t>(positions, tokens, "positions"), *const to = vector_of<int32_t>(slots, tokens, "slots");
    const int most = count32(table.size(0), "table"), rot = count32(table.size(1), "table"), interleaved = truth(a[9]);
    const int t32 = count32(tokens, "q"), h32 = count32(heads, "q");
    on_device(ctx, {{&q, "q"}, {&k, "k"}, {&v, "v"}, {&positions, "positions"}, {&slots, "slots"}, {&table, "table"}, {&out, "q_out"}});
    const int status = call([&] {
        return entries.append_kv(ctx, qh.at, qh.row, qh.head, kh.at, kh.row, kh.head, vh.at, vh.row, vh.head, oh.at, oh.row, oh.head,
                                 &cache, at, to, static_cast<const float *>(table.data_ptr()), row, most, rot, interleaved, t32, h32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    return a[8] == Py_None ? give(std::move(out)) : same(a[8]);
    END_HANDLE_TH_ERRORS
}

// ctx, q, cache, pages, lengths, scale (None: 1/sqrt(dim)), softcap, window, out → out
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &q = tensor(a[1], "q"), &pages = tensor(a[3], "pages"), &lengths = tensor(a[4], "lengths");
    const sq8_paged_cache cache = held<sq8_paged_cache>(a[2], "a cache's description");
    const int64_t batch = queries(q), heads = q.size(1);
    Tensor out = a[8] == Py_None ? at::empty({batch, heads, cache.dim}, q.options()) : tensor(a[8], "out");
    const Heads qh = heads_of(q, "q", batch, heads, cache.dim), oh = heads_of(out, "out", batch, heads, cache.dim);
    TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt && pages.dim() == 2 && pages.size(0) == batch, "pages must be int32 [", batch,
                      ", most pages]");
    const int64_t row = rows_of(pages, "pages");
    const int32_t *const held_tokens = vector_of<int32_t>(lengths, batch, "lengths");
    const float scale = (float)(a[5] == Py_None ? 1.0 / std::sqrt((double)cache.dim) : number(a[5])), softcap = (float)number(a[6]);
    const int window = integer(a[7]), most = count32(pages.size(1), "pages"), b32 = count32(batch, "q"), h32 = count32(heads, "q");
    on_device(ctx, {{&q, "q"}, {&pages, "pages"}, {&lengths, "lengths"}, {&out, "out"}});
    const int status = call([&] {
        return entries.paged_attention(ctx, qh.at, qh.row, qh.head, &cache, static_cast<const int32_t *>(pages.data_ptr()), row, most,
                                       held_tokens, scale, softcap, window, oh.at, oh.row, oh.head, b32, h32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    return a[8] == Py_None ? give(std::move(out)) : same(a[8]);
    END_HANDLE_TH_ERRORS
}

// A position table: its rows, positions and turned values.
struct Table {
    const float *at;
    int64_t row;
    int most, rot;
};
Table table_of(const Tensor &t) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, "table must be float32 [positions, rot]");
    const int64_t row = rows_of(t, "table");
    return {static_cast<const float *>(t.data_ptr()), row, count32(t.size(0), "table"), count32(t.size(1), "table")};
}
// A vector that may be left out.
const float *maybe_vector(const Tensor *t, int64_t dim, const char *what) { return t ? vector_of<float>(*t, dim, what) : nullptr; }

// ctx, q, k, v, cache, positions, slots, table, q_norm, k_norm, eps, q_out, interleaved → q_out
PyObject *norm_append_kv(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 13);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
    const sq8_paged_cache cache = held<sq8_paged_cache>(a[4], "a cache's description");
    const Tensor &positions = tensor(a[5], "positions"), &slots = tensor(a[6], "slots"), &table = tensor(a[7], "table");
    const Tensor *const q_norm = maybe(a[8], "q_norm"), *const k_norm = maybe(a[9], "k_norm");
    const float eps = (float)number(a[10]);
    const int64_t tokens = queries(q), heads = q.size(1);
    Tensor out = a[11] == Py_None ? at::empty({tokens, heads, cache.dim}, q.options()) : tensor(a[11], "q_out");
    const Heads qh = heads_of(q, "q", tokens, heads, cache.dim), kh = heads_of(k, "k", tokens, cache.kv_heads, cache.dim);
    const Heads vh = heads_of(v, "v", tokens, cache.kv_heads, cache.dim), oh = heads_of(out, "q_out", tokens, heads, cache.dim);
    const Table angles = table_of(table);
    const int32_t *const at = vector_of<int32_t>(positions, tokens, "positions"), *const to = vector_of<int32_t>(slots, tokens, "slots");
    const float *const qn = maybe_vector(q_norm, cache.dim, "q_norm"), *const kn = maybe_vector(k_norm, cache.dim, "k_norm");
    const int interleaved = truth(a[12]), t32 = count32(tokens, "q"), h32 = count32(heads, "q");
    on_device(ctx, {{&q, "q"}, {&k, "k"}, {&v, "v"}, {&positions, "positions"}, {&slots, "slots"}, {&table, "table"},
                    {q_norm, "q_norm"}, {k_norm, "k_norm"}, {&out, "q_out"}});
    const int status = call([&] {
        return entries.norm_append_kv(ctx, qh.at, qh.row, qh.head, kh.at, kh.row, kh.head, vh.at, vh.row, vh.head, oh.at, oh.row, oh.head,
                                      &cache, at, to, angles.at, angles.row, angles.most, angles.rot, interleaved, qn, kn, eps, t32, h32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    return a[11] == Py_None ? give(std::move(out)) : same(a[11]);
    END_HANDLE_TH_ERRORS
}

// ctx, q, k (or None), positions, table (None with positions: not turned), q_norm, k_norm, eps, q_out, k_out, interleaved →
// (q_out, k_out)
PyObject *norm_rotate(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 11);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &q = tensor(a[1], "q");
    const Tensor *const k = maybe(a[2], "k"), *const positions = maybe(a[3], "positions"), *const table = maybe(a[4], "table");
    const Tensor *const q_norm = maybe(a[5], "q_norm"), *const k_norm = maybe(a[6], "k_norm");
    const float eps = (float)number(a[7]);
    const int64_t tokens = queries(q), heads = q.size(1), dim = q.size(2), kv_heads = k && k->dim() == 3 ? k->size(1) : 0;
    Tensor q_out = a[8] == Py_None ? at::empty({tokens, heads, dim}, q.options()) : tensor(a[8], "q_out"), k_out;
    const Heads qh = heads_of(q, "q", tokens, heads, dim), oh = heads_of(q_out, "q_out", tokens, heads, dim);
    Heads kh{}, ko{};
    TORCH_CHECK_VALUE(k || (a[9] == Py_None && !k_norm), "k_out and k_norm belong to k");
    if (k) {
        kh = heads_of(*k, "k", tokens, kv_heads, dim);
        k_out = a[9] == Py_None ? at::empty({tokens, kv_heads, dim}, k->options()) : tensor(a[9], "k_out");
        ko = heads_of(k_out, "k_out", tokens, kv_heads, dim);
    }
    TORCH_CHECK_VALUE(!positions == !table, "positions and table belong together");
    Table angles{};
    const int32_t *at = nullptr;
    if (table) {
        angles = table_of(*table);
        at = vector_of<int32_t>(*positions, tokens, "positions");
    }
    const float *const qn = maybe_vector(q_norm, dim, "q_norm"), *const kn = maybe_vector(k_norm, dim, "k_norm");
    const int interleaved = truth(a[10]), t32 = count32(tokens, "q"), h32 = count32(heads, "q"), kv32 = count32(kv_heads, "k");
    const int d32 = count32(dim, "q");
    on_device(ctx, {{&q, "q"}, {k, "k"}, {positions, "positions"}, {table, "table"}, {q_norm, "q_norm"}, {k_norm, "k_norm"},
                    {&q_out, "q_out"}, {k ? &k_out : nullptr, "k_out"}});
    const int status = call([&] {
        return entries.norm_rotate(ctx, qh.at, qh.row, qh.head, kh.at, kh.row, kh.head, oh.at, oh.row, oh.head, ko.at, ko.row, ko.head,
                                   at, angles.at, angles.row, angles.most, angles.rot, interleaved, qn, kn, eps, t32, h32, kv32, d32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    PyObject *const all = PyTuple_New(2);
    if (!all) throw python_error();
    PyTuple_SET_ITEM(all, 0, a[8] == Py_None ? give(std::move(q_out)) : same(a[8]));
    PyTuple_SET_ITEM(all, 1, k && a[9] == Py_None ? give(std::move(k_out)) : same(a[9]));
    return all;
    END_HANDLE_TH_ERRORS
}

// Where a batch's sequences begin: [sequences + 1], or null with one sequence of all rows.
const int32_t *starts_of(const Tensor *t, int64_t &sequences) {
    if (!t) {
        sequences = 1;
        return nullptr;
    }
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) >= 1, "starts must be int32 [sequences + 1]");
    sequences = t->size(0) - 1;
    return vector_of<int32_t>(*t, t->size(0), "starts");
}

// ctx, q, k, v, starts (None: one sequence), scale (None: 1/sqrt(dim)), softcap, window, causal, out → out
PyObject *prompt_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &q = tensor(a[1], "q"), &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
    const Tensor *const starts = maybe(a[4], "starts");
    const int64_t tokens = queries(q), heads = q.size(1), dim = q.size(2);
    TORCH_CHECK_VALUE(k.dim() == 3, "k must be [tokens, kv heads, dim], not ", k.sizes());
    const int64_t kv_heads = k.size(1);
    Tensor out = a[9] == Py_None ? at::empty({tokens, heads, dim}, q.options()) : tensor(a[9], "out");
    const Heads qh = heads_of(q, "q", tokens, heads, dim), kh = heads_of(k, "k", tokens, kv_heads, dim);
    const Heads vh = heads_of(v, "v", tokens, kv_heads, dim), oh = heads_of(out, "out", tokens, heads, dim);
    int64_t sequences;
    const int32_t *const from = starts_of(starts, sequences);
    const float scale = (float)(a[5] == Py_None ? 1.0 / std::sqrt((double)dim) : number(a[5])), softcap = (float)number(a[6]);
    const int window = integer(a[7]), causal = truth(a[8]), t32 = count32(tokens, "q"), h32 = count32(heads, "q");
    const int kv32 = count32(kv_heads, "k"), d32 = count32(dim, "q"), s32 = count32(sequences, "starts");
    on_device(ctx, {{&q, "q"}, {&k, "k"}, {&v, "v"}, {starts, "starts"}, {&out, "out"}});
    const int status = call([&] {
        return entries.prompt_attention(ctx, qh.at, qh.row, qh.head, kh.at, kh.row, kh.head, vh.at, vh.row, vh.head, from, s32, scale,
                                        softcap, window, causal, oh.at, oh.row, oh.head, t32, h32, kv32, d32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    return a[9] == Py_None ? give(std::move(out)) : same(a[9]);
    END_HANDLE_TH_ERRORS
}

// ctx, q, cache, pages, lengths, starts (None: one sequence), scale (None: 1/sqrt(dim)), softcap, window, out → out
PyObject *chunk_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 10);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &q = tensor(a[1], "q"), &pages = tensor(a[3], "pages"), &lengths = tensor(a[4], "lengths");
    const sq8_paged_cache cache = held<sq8_paged_cache>(a[2], "a cache's description");
    const Tensor *const starts = maybe(a[5], "starts");
    const int64_t tokens = queries(q), heads = q.size(1);
    Tensor out = a[9] == Py_None ? at::empty({tokens, heads, cache.dim}, q.options()) : tensor(a[9], "out");
    const Heads qh = heads_of(q, "q", tokens, heads, cache.dim), oh = heads_of(out, "out", tokens, heads, cache.dim);
    int64_t sequences;
    const int32_t *const from = starts_of(starts, sequences);
    TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt && pages.dim() == 2 && pages.size(0) == sequences, "pages must be int32 [",
                      sequences, ", most pages]");
    const int64_t row = rows_of(pages, "pages");
    const int32_t *const held_tokens = vector_of<int32_t>(lengths, sequences, "lengths");
    const float scale = (float)(a[6] == Py_None ? 1.0 / std::sqrt((double)cache.dim) : number(a[6])), softcap = (float)number(a[7]);
    const int window = integer(a[8]), most = count32(pages.size(1), "pages"), t32 = count32(tokens, "q"), h32 = count32(heads, "q");
    const int s32 = count32(sequences, "starts");
    on_device(ctx, {{&q, "q"}, {&pages, "pages"}, {&lengths, "lengths"}, {starts, "starts"}, {&out, "out"}});
    const int status = call([&] {
        return entries.chunk_attention(ctx, qh.at, qh.row, qh.head, &cache, static_cast<const int32_t *>(pages.data_ptr()), row, most,
                                       held_tokens, from, s32, scale, softcap, window, oh.at, oh.row, oh.head, t32, h32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    return a[9] == Py_None ? give(std::move(out)) : same(a[9]);
    END_HANDLE_TH_ERRORS
}

// ctx, logits, uniform, temperature, top_k, top_p, min_p (each or None), tokens, logprobs → (tokens, logprobs)
PyObject *sample_tokens(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect(n, 9);
    sq8_ctx *const ctx = context(a[0]);
    const Tensor &logits = tensor(a[1], "logits"), &uniform = tensor(a[2], "uniform");
    const Tensor *const temperature = maybe(a[3], "temperature"), *const top_k = maybe(a[4], "top_k");
    const Tensor *const top_p = maybe(a[5], "top_p"), *const min_p = maybe(a[6], "min_p");
    const int64_t ld = rows_of(logits, "logits"), rows = logits.size(0), vocab = logits.size(1);
    const int type = activation(logits, "logits"), r32 = count32(rows, "logits"), v32 = count32(vocab, "logits");
    Tensor tokens = a[7] == Py_None ? at::empty({rows}, logits.options().dtype(at::kInt)) : tensor(a[7], "tokens");
    Tensor logprobs = a[8] == Py_None ? at::empty({rows}, logits.options().dtype(at::kFloat)) : tensor(a[8], "logprobs");
    const float *const u = vector_of<float>(uniform, rows, "uniform"), *const t = maybe_vector(temperature, rows, "temperature");
    const int32_t *const k = top_k ? vector_of<int32_t>(*top_k, rows, "top_k") : nullptr;
    const float *const tp = maybe_vector(top_p, rows, "top_p"), *const mp = maybe_vector(min_p, rows, "min_p");
    vector_of<int32_t>(tokens, rows, "tokens");
    vector_of<float>(logprobs, rows, "logprobs");
    on_device(ctx, {{&logits, "logits"}, {&uniform, "uniform"}, {temperature, "temperature"}, {top_k, "top_k"}, {top_p, "top_p"},
                    {min_p, "min_p"}, {&tokens, "tokens"}, {&logprobs, "logprobs"}});
    const int status = call([&] {
        return entries.sample_tokens(ctx, logits.data_ptr(), type, ld, u, t, k, tp, mp, static_cast<int32_t *>(tokens.data_ptr()),
                                     static_cast<float *>(logprobs.data_ptr()), r32, v32);
    });
    if (status != SQ8_OK) return PyLong_FromLong(status);
    PyObject *const all = PyTuple_New(2);
    if (!all) throw python_error();
    PyTuple_SET_ITEM(all, 0, a[7] == Py_None ? give(std::move(tokens)) : same(a[7]));
    PyTuple_SET_ITEM(all, 1, a[8] == Py_None ? give(std::move(logprobs)) : same(a[8]));
    return all;
    END_HANDLE_TH_ERRORS
}

// The library's entries: their addresses, in the order of Entries.
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    constexpr Py_ssize_t wanted = sizeof(Entries) / sizeof(void *);
    expect(n, wanted);
    void *at[wanted];
    for (Py_ssize_t i = 0; i < n; ++i) {
        at[i] = PyLong_AsVoidPtr(a[i]);
        if (!at[i]) {
            if (PyErr_Occurred()) throw python_error();
            TORCH_CHECK_VALUE(false, "an entry is missing");
        }
    }
    memcpy(&entries, at, sizeof(entries));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define TEXT_OP(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TEXT_OP(bind), TEXT_OP(add_norm_quantized), TEXT_OP(quantize_groups), TEXT_OP(product_f8),
                         TEXT_OP(append_kv), TEXT_OP(paged_attention), TEXT_OP(norm_append_kv), TEXT_OP(norm_rotate),
                         TEXT_OP(prompt_attention), TEXT_OP(chunk_attention), TEXT_OP(sample_tokens), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_text_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__text_bind() { return PyModule_Create(&module); }
