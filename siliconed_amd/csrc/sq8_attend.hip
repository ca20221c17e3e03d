// sq8_attend.hip — which source's kernels a prompt's or chunk's attention runs on (sq8_attend_inst.hip).
#include <algorithm>

#include "sq8_text.h"

namespace sq8 {

hipError_t launch_attend(const AttendArgs &p, const AttendPlan &plan, bool e4m3, hipStream_t stream) {
    if (p.sequences == 0 || p.tokens == 0) return hipSuccess;
    if (plan.narrow) return attend::launch_chunk(p, plan, e4m3, stream);
    if (!p.pages) return attend::launch_source<attend::ROWS>(p, plan, stream);
    if (p.page % 16 == 0)
        return e4m3 ? attend::launch_source<attend::PAGES16_F8>(p, plan, stream) : attend::launch_source<attend::PAGES16>(p, plan, stream);
    return e4m3 ? attend::launch_source<attend::PAGES_F8>(p, plan, stream) : attend::launch_source<attend::PAGES>(p, plan, stream);
}

}  // namespace sq8
