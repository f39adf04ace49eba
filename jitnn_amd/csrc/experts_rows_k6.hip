// experts_rows_kernel for Q6_K, Q2_K.
#include "experts_rows.h"

namespace jitnn {

RowsKernelRef experts_rows_ref_k6(int fmt, int groups, bool pair) {
    switch (fmt) {
    case F_Q6_K: return experts_rows_pick<F_Q6_K>(groups, pair);
    case F_Q2_K: return experts_rows_pick<F_Q2_K>(groups, pair);
    default: return {};
    }
}

}  // namespace jitnn
