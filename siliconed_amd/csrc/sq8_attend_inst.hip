// sq8_attend_inst.hip — the prompt and chunk attention's kernels of one source of keys and values (SQ8_SOURCE).
#include "sq8_attend_kernel.h"

namespace sq8 {
namespace attend {
namespace {

template <int DP, int WM, int WT>
hipError_t launch(const AttendArgs &p, int groups, hipStream_t stream) {
    hipLaunchKernelGGL((attend_kernel<DP, WM, WT, SQ8_SOURCE, SQ8_SOURCE != ROWS>), dim3(groups), dim3(64 * WM * WT), 0, stream, p);
    return hipGetLastError();
}

template <int DP>
hipError_t pick(const AttendArgs &p, const AttendPlan &plan, hipStream_t stream) {
    if (plan.rows == 128) return launch<DP, 4, 1>(p, plan.groups, stream);
    if constexpr (DP <= 128) {
        if constexpr (SQ8_SOURCE == ROWS)
            if (plan.rows == 64) return launch<DP, 2, 2>(p, plan.groups, stream);
        if constexpr (DP == 128 || SQ8_SOURCE <= PAGES)
            if (plan.rows == 256) return launch<DP, 8, 1>(p, plan.groups, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace

template <>
hipError_t launch_source<SQ8_SOURCE>(const AttendArgs &p, const AttendPlan &plan, hipStream_t stream) {
    switch (attend_dim(p.dim)) {
        case 64: return pick<64>(p, plan, stream);
        case 128: return pick<128>(p, plan, stream);
        default: return pick<256>(p, plan, stream);
    }
}

}  // namespace attend
}  // namespace sq8
