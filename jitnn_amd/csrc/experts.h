// Host entry points of the mixture of experts - the router (router.hip), the experts' products (experts.hip and the units beside it) - and the
// argument blocks of their kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace jitnn {

enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_COUNT = 5 };

constexpr int MAX_EXPERTS = 512, MAX_USED = 64;

// ---- router.h
struct RouterArgs {
    const float *x, *w;  // [tokens, d], [experts, d]
    const float *bias;   // [experts] or nullptr: added for the choice, not for the weights
    double *logits;      // [tokens, experts]
    int *ids;            // [tokens, used]
    float *weights;      // [tokens, used]
    // the slots (token x used + place) of each expert: list[offsets[e]] .. list[offsets[e + 1] - 1]; nullptr: not wanted
    int *offsets, *list;  // [experts + 1], [tokens x used]
    int tokens, experts, d, used;
    bool sigmoid, normalise;
    float scale;
};
bool router_needs_logits(int tokens, int experts, int d, bool lists);  // whether a launch of this size reads and writes `logits`
void router_launch(const RouterArgs &a, hipStream_t s);
// the lists of choices that somebody else made; an id outside [0, experts) is on none
void expert_lists_launch(const int *ids, int slots, int experts, int *offsets, int *list, hipStream_t s);

// ---- experts.hip
struct ExpertWeights {
    int fmt, n, k;  // of one expert: [n, k]
    const uint8_t *w;
    size_t expert_bytes;
};
// y [slots, n] = the product of each slot's expert with row slot / per_row of x, in FP32 on the dequantiser's values: any format
void experts_value_launch(const ExpertWeights &w, int experts, const int *ids, int slots, int per_row, const float *x, float *y, hipStream_t s);
// h [count] = act(g) * u (h may be g)
void experts_gate_launch(int act, const float *g, const float *u, float *h, size_t count, int cus, hipStream_t s);
// y [tokens, n] = res (or 0) + the sum over a token's places j of weights[j] * part[token x used + j]; an id outside [0, experts) counts for nothing
void experts_combine_launch(const float *part, const int *ids, const float *weights, const float *res, float *y, int tokens, int used, int experts, int n, int cus,
                            hipStream_t s);

// ---- the epilogue of a linear, where its kernel has none: y [count] = act(y) + res (or 0)
void linear_epilogue_launch(int act, const float *res, float *y, size_t count, int cus, hipStream_t s);

}  // namespace jitnn
