// The experts' products of few tokens for Q4_K, Q5_K, Q2_K, Q6_K.
#include "experts_few.h"

namespace jitnn {

ExpertFewKernel experts_few_up_k(int fmt, bool aligned, int waves) {
    switch (fmt) {
    case F_Q4_K: return experts_few_up_pick<U8<F_Q4_K>>(waves);
    case F_Q5_K: return experts_few_up_pick<U8<F_Q5_K>>(waves);
    case F_Q2_K: return experts_few_up_pick<U8<F_Q2_K>>(waves);
    case F_Q6_K: return aligned ? experts_few_up_pick<U8Q6<true>>(waves) : experts_few_up_pick<U8Q6<false>>(waves);
    default: return nullptr;
    }
}

ExpertFewKernel experts_few_down_k(int fmt, bool aligned, int stretches, int waves) {
    switch (fmt) {
    case F_Q4_K: return experts_few_down_pick<U8<F_Q4_K>>(stretches, waves);
    case F_Q5_K: return experts_few_down_pick<U8<F_Q5_K>>(stretches, waves);
    case F_Q2_K: return experts_few_down_pick<U8<F_Q2_K>>(stretches, waves);
    case F_Q6_K: return aligned ? experts_few_down_pick<U8Q6<true>>(stretches, waves) : experts_few_down_pick<U8Q6<false>>(stretches, waves);
    default: return nullptr;
    }
}

}  // namespace jitnn
