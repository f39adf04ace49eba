// experts_rows_kernel for Q8_0, Q4_0, Q4_1, Q5_1.
#include "experts_rows.h"

namespace jitnn {

KernelRef experts_rows_ref_q32(int fmt, int groups, bool dual) {
    switch (fmt) {
    case F_Q8_0: return experts_rows_pick<F_Q8_0>(groups, dual);
    case F_Q4_0: return experts_rows_pick<F_Q4_0>(groups, dual);
    case F_Q4_1: return experts_rows_pick<F_Q4_1>(groups, dual);
    case F_Q5_1: return experts_rows_pick<F_Q5_1>(groups, dual);
    default: return {nullptr, 0};
    }
}

void experts_rows_launch_q32(int fmt, const ExpertRowsArgs &a, unsigned blocks, bool dual, hipStream_t s) {
    switch (fmt) {
    case F_Q8_0: experts_rows_go<F_Q8_0>(a, blocks, dual, s); break;
    case F_Q4_0: experts_rows_go<F_Q4_0>(a, blocks, dual, s); break;
    case F_Q4_1: experts_rows_go<F_Q4_1>(a, blocks, dual, s); break;
    case F_Q5_1: experts_rows_go<F_Q5_1>(a, blocks, dual, s); break;
    }
}

}  // namespace jitnn
