// experts_rows_kernel for Q6_K, Q2_K.
#include "experts_rows.h"

namespace jitnn {

KernelRef experts_rows_ref_k6(int fmt, int groups, bool dual) {
    switch (fmt) {
    case F_Q6_K: return experts_rows_pick<F_Q6_K>(groups, dual);
    case F_Q2_K: return experts_rows_pick<F_Q2_K>(groups, dual);
    default: return {nullptr, 0};
    }
}

void experts_rows_launch_k6(int fmt, const ExpertRowsArgs &a, unsigned blocks, bool dual, hipStream_t s) {
    switch (fmt) {
    case F_Q6_K: experts_rows_go<F_Q6_K>(a, blocks, dual, s); break;
    case F_Q2_K: experts_rows_go<F_Q2_K>(a, blocks, dual, s); break;
    }
}

}  // namespace jitnn
