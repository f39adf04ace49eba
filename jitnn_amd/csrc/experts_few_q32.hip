// The experts' products of few tokens for Q8_0, Q4_0, Q4_1, Q5_1.
#include "experts_few.h"

namespace jitnn {

ExpertFewKernel experts_few_up_q32(int fmt, int waves) {
    switch (fmt) {
    case F_Q8_0: return experts_few_up_pick<U8<F_Q8_0>>(waves);
    case F_Q4_0: return experts_few_up_pick<U8<F_Q4_0>>(waves);
    case F_Q4_1: return experts_few_up_pick<U8<F_Q4_1>>(waves);
    case F_Q5_1: return experts_few_up_pick<U8<F_Q5_1>>(waves);
    default: return nullptr;
    }
}

ExpertFewKernel experts_few_down_q32(int fmt, int stretches, int waves) {
    switch (fmt) {
    case F_Q8_0: return experts_few_down_pick<U8<F_Q8_0>>(stretches, waves);
    case F_Q4_0: return experts_few_down_pick<U8<F_Q4_0>>(stretches, waves);
    case F_Q4_1: return experts_few_down_pick<U8<F_Q4_1>>(stretches, waves);
    case F_Q5_1: return experts_few_down_pick<U8<F_Q5_1>>(stretches, waves);
    default: return nullptr;
    }
}

}  // namespace jitnn
