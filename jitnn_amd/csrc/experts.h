// Host entry points of the mixture of experts - the router (router.hip), the experts' products (experts.hip and the units beside it) - and the
// argument blocks of their kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "tu.h"

namespace jitnn {

enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_COUNT = 5 };

constexpr int MAX_EXPERTS = 512, MAX_USED = 64;

// ---- router.h
// The slots (token x used + place) of each expert, one expert's after the other, and their chunks of at most chunk_rows: [0].x their number, then
// {expert, place of the first slot in the list, slots, 0} each.
struct ExpertLists {
    int *list = nullptr;   // [slots]; nullptr: not wanted
    int4 *chunks = nullptr;  // [1 + chunks_most()]
    int chunk_rows = 8;
    static int chunks_most(int slots, int experts, int chunk_rows) { return (slots < experts ? slots : experts) + slots / chunk_rows; }
};
// Rows of activations to be prepared as operands (experts_rows.h): x [rows, k], k a multiple of 4, to the layouts that have a place.
struct ExpertPrepare {
    const float *x = nullptr;
    int rows = 0, k = 0;
    uint8_t *ops[3] = {};  // per layout (GR_LAYOUT_*): nullptr - not wanted
    float *inv[3] = {};    // [rows, columns]
    __host__ __device__ int units() const { return ops[0] || ops[1] || ops[2] ? (rows + 7) / 8 * ((k + 255) / 256) : 0; }  // of a wave's work
};
struct RouterArgs {
    const float *x, *w;  // [tokens, d], [experts, d]
    const float *bias;   // [experts] or nullptr: added for the choice, not for the weights
    double *logits;      // [splits][tokens, experts]
    int *ids;            // [tokens, used]
    float *weights;      // [tokens, used]
    ExpertLists lists;
    ExpertPrepare prepare;  // beside the lists, in their launch
    int tokens, experts, d, used;
    bool sigmoid, normalise;
    float scale;
    int splits;  // (set with the launch of the logits)
};
// what `logits` takes; choice_follows: router_launch without lists, which may need none
size_t router_logits_bytes(int tokens, int experts, int d, bool choice_follows);
void router_logits_launch(RouterArgs &a, hipStream_t s);
void router_launch(RouterArgs a, hipStream_t s);
// the lists of choices that somebody else made; an id outside [0, experts) is on none
void expert_lists_launch(const int *ids, int slots, int experts, const ExpertLists &lists, const ExpertPrepare &prepare, hipStream_t s);

struct ExpertWeights {
    int fmt, n, k;  // of one expert: [n, k]
    const uint8_t *w;
    size_t expert_bytes;
};
// ---- experts_rows.h: the same on the matrix cores
struct ExpertRowsArgs {
    const uint8_t *w, *w2;  // [experts][n rows]
    size_t expert_bytes;
    const uint8_t *ops;     // the prepared rows (experts_prepare_launch), in the layout of the format
    const float *inv;
    const int *list;
    const int4 *chunks;
    float *y;               // [slots, n]
    size_t split_floats;    // from one split's y to the next one's
    int n, k, experts, per_row, act, nblocks, splits;
};
typedef void (*RowsKernel)(const ExpertRowsArgs);
struct RowsKernelRef {
    RowsKernel fn;
    size_t lds;
    int threads, tiles, groups;  // tiles: of 16 weight rows (of each matrix of a pair) per workgroup; groups: of eight rows per chunk, at most
};
size_t experts_ops_bytes(size_t rows, int k);  // the operands of so many rows, and their scales behind them
ExpertPrepare experts_prepare(const float *x, int rows, int k, uint8_t *const *places);  // places: per layout (GR_LAYOUT_*), nullptr - not wanted
void experts_prepare_launch(const ExpertPrepare &p, hipStream_t s);
// the kernel for chunks of so many groups of eight rows (or of the most it has, where they are more).  pair: y = act(w x) * (w2 x)
RowsKernelRef experts_rows_kernel_ref(int fmt, int groups, bool pair);
RowsKernelRef experts_rows_ref_k(int fmt, int groups, bool pair);    // experts_rows_k.hip: Q4_K, Q5_K
RowsKernelRef experts_rows_ref_k6(int fmt, int groups, bool pair);   // experts_rows_k6.hip: Q6_K, Q2_K
RowsKernelRef experts_rows_ref_q32(int fmt, int groups, bool pair);  // experts_rows_q32.hip: Q8_0, Q4_0, Q4_1, Q5_1
// chunks_most: no more of them are there
void experts_rows_launch(const RowsKernelRef &k, ExpertRowsArgs a, int chunks_most, hipStream_t s);

// ---- experts_few.h: few tokens, INT8 products
struct ExpertFewArgs {
    const uint8_t *w, *w2;  // [experts][n rows of k values]; up: gate and up, down: w2 not used
    size_t expert_bytes;
    const float *x;         // up: [tokens, k]; down: [tokens, used, k]
    const int *ids;         // [tokens, used]
    const float *weights;   // down: [tokens, used]
    const float *res;       // down: [tokens, n] or nullptr
    float *y;               // up: [tokens, used, n]; down: [parts][tokens, n] (may be res)
    int n, k, used, experts, act, blocks;
    unsigned by_rows;       // up: reciprocal of n / 4
    RouterArgs route;       // up: logits that are there, of which every wave makes the choice for itself (and the first one leaves it at ids and weights); logits nullptr: ids are there
};
// whether rows of k values (up) and `used` of ffn values behind one another (down) have a kernel; in how many parts (one at least), each with a y to be added up, the latter
bool experts_few_chooses(int experts);  // whether the first launch can make the choices
bool experts_few_up_supported(int fmt, int k);
bool experts_few_down_supported(int fmt, int ffn, int used);
int experts_few_down_parts(int ffn, int used);
void experts_few_up_launch(int fmt, ExpertFewArgs a, int tokens, int cus, hipStream_t s);
void experts_few_down_launch(int fmt, ExpertFewArgs a, int tokens, int cus, hipStream_t s);
typedef void (*ExpertFewKernel)(const ExpertFewArgs);
ExpertFewKernel experts_few_up_k(int fmt, bool aligned, int waves);     // experts_few_k.hip: Q4_K, Q5_K, Q6_K, Q2_K
ExpertFewKernel experts_few_up_q32(int fmt, int waves);                 // experts_few_q32.hip: Q8_0, Q4_0, Q4_1, Q5_1
ExpertFewKernel experts_few_down_k(int fmt, bool aligned, int stretches, int waves);
ExpertFewKernel experts_few_down_q32(int fmt, int stretches, int waves);

// ---- experts.hip
// y [slots, n] = the product of each slot's expert with row slot / per_row of x, in FP32 on the dequantiser's values: Q5_0 and Q3_K blocks as a file has them
void experts_value_launch(const ExpertWeights &w, int experts, const int *ids, int slots, int per_row, const float *x, float *y, hipStream_t s);
// h [count] = act(g) * u (h may be g)
void experts_gate_launch(int act, const float *g, const float *u, float *h, size_t count, int cus, hipStream_t s);
// y [tokens, n] = res (or 0) + the sum over a token's places j of weights[j] * part[token x used + j], part in `splits` arrays to be added up; an id outside
// [0, experts) counts for nothing
void experts_combine_launch(const float *part, int splits, const int *ids, const float *weights, const float *res, float *y, int tokens, int used, int experts, int n,
                            hipStream_t s);

// ---- the epilogue of a linear, where its kernel has none: y [count] = act(y) + res (or 0)
void linear_epilogue_launch(int act, const float *res, float *y, size_t count, int cus, hipStream_t s);

}  // namespace jitnn
