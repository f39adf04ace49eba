// experts_rows_kernel for Q8_0, Q4_0, Q4_1, Q5_1.
#include "experts_rows.h"

namespace jitnn {

RowsKernelRef experts_rows_ref_q32(int fmt, int groups, bool pair) {
    switch (fmt) {
    case F_Q8_0: return experts_rows_pick<F_Q8_0>(groups, pair);
    case F_Q4_0: return experts_rows_pick<F_Q4_0>(groups, pair);
    case F_Q4_1: return experts_rows_pick<F_Q4_1>(groups, pair);
    case F_Q5_1: return experts_rows_pick<F_Q5_1>(groups, pair);
    default: return {};
    }
}

}  // namespace jitnn
