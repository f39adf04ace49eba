// experts_rows_kernel for Q4_K, Q5_K.
#include "experts_rows.h"

namespace jitnn {

RowsKernelRef experts_rows_ref_k(int fmt, int groups, bool pair) {
    switch (fmt) {
    case F_Q4_K: return experts_rows_pick<F_Q4_K>(groups, pair);
    case F_Q5_K: return experts_rows_pick<F_Q5_K>(groups, pair);
    default: return {};
    }
}

}  // namespace jitnn
