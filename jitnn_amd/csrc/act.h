// The activations of a feed-forward layer, in FP32.  A value that is not a number stays one.
#pragma once
#include "common.h"
#include "experts.h"

namespace jitnn {

// (expf, not __expf: the latter's error grows with its argument, 6e-7 of the result at 10)
__device__ __forceinline__ float act_silu(float v) { return v / (1.f + expf(-v)); }

__device__ __forceinline__ float activate(int act, float v) {
    switch (act) {  // (the same for all lanes)
    case ACT_RELU: return v < 0.f ? 0.f : v;
    case ACT_SILU: return act_silu(v);
    case ACT_GELU: return 0.5f * v * erfcf(-0.70710678f * v);  // (1 + erf would cancel for large negative values)
    case ACT_GELU_TANH: {  // 0.5 v (1 + tanh u) = v / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
        const float u2 = v * __builtin_fmaf(0.0713548163f * v, v, 1.59576912f);
        return v / (1.f + expf(-u2));
    }
    default: return v;
    }
}

}  // namespace jitnn
