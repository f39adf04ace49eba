// experts_rows_kernel for Q4_K, Q5_K.
#include "experts_rows.h"

namespace jitnn {

KernelRef experts_rows_ref_k(int fmt, int groups, bool dual) {
    switch (fmt) {
    case F_Q4_K: return experts_rows_pick<F_Q4_K>(groups, dual);
    case F_Q5_K: return experts_rows_pick<F_Q5_K>(groups, dual);
    default: return {nullptr, 0};
    }
}

void experts_rows_launch_k(int fmt, const ExpertRowsArgs &a, unsigned blocks, bool dual, hipStream_t s) {
    switch (fmt) {
    case F_Q4_K: experts_rows_go<F_Q4_K>(a, blocks, dual, s); break;
    case F_Q5_K: experts_rows_go<F_Q5_K>(a, blocks, dual, s); break;
    }
}

}  // namespace jitnn
