// sq8_context.h — the C ABI's context and what its entry points share on the host.
#pragma once

#include <hip/hip_runtime.h>
#include <rocblas/rocblas.h>
#include <stdint.h>

#include "siliconed_q8.h"
#include "sq8_buffers.h"

struct sq8_ctx {
    int device;
    hipStream_t stream;
    hipEvent_t begin, end;
    sq8::Buffer scratch;    // bf16 copy of an fp32 activation (the reference's rounding scratch)
    sq8::Buffer wpack;      // [K, N] codes repacked for the weight-direct kernels, per product
    sq8::Buffer part;       // partial sums: the skinny kernel's and a block-scaled product's K split, a paged attention's
                            // split sequences
    sq8::Buffer marks;      // the counters of those last two, zero between calls
    sq8::SetAside *aside;   // what these outgrew while a captured graph may use it
    rocblas_handle blas;    // the bf16-weight product's library GEMM (created on its first call)
    int wd_tile;            // measurement knobs, read once at sq8_create (SQ8_TILE, SQ8_Q8_TILE, SQ8_SPLITS): a
    int q8_tile;            // forced weight-direct / block-scale tile, or -1 (the product's own choice); the
    int i8_tile;            // the W8A8 tile SQ8_TILE forces (the K-group tiles only), or -1
    int splits;             // skinny kernel's K split count (1: none, the default)
    int cus;                // the device's compute units, read once here: the tile rules' rounds
};

namespace sq8 {

inline int hip_status(hipError_t e) { return e == hipSuccess ? SQ8_OK : -(int)e; }

// Makes the context's device current for the scope, restoring the caller's afterwards.
struct DeviceScope {
    int previous = -1;
    hipError_t error = hipSuccess;
    explicit DeviceScope(int device) {
        error = hipGetDevice(&previous);
        if (error == hipSuccess && previous != device) error = hipSetDevice(device);
    }
    ~DeviceScope() {
        int now = -1;
        if (previous >= 0 && hipGetDevice(&now) == hipSuccess && now != previous) (void)hipSetDevice(previous);
    }
};

inline bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// Grows one of the context's buffers to `bytes` (never shrinks; freed with the context).
inline int reserve(sq8_ctx *ctx, Buffer &b, size_t bytes) { return hip_status(reserve(b, bytes, ctx->stream, ctx->aside)); }

}  // namespace sq8
