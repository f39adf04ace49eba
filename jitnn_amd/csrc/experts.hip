// The experts' products for the formats that the matrix cores' kernels have no operands of, the gate, the weighted sum of a token's experts, and what launches those kernels.
#include "experts.h"

#include <algorithm>

#include "act.h"
#include "dequant.h"
#include "experts_few.h"
#include "experts_rows.h"
#include "serving.h"

namespace jitnn {

// One wave per weight row of the slot's expert, every lane dequantises quads of the row.  grid (ceil(n / 4), slots up to 65535, and so on along z).
template <int FMT>
__global__ void __launch_bounds__(256) experts_value_kernel(const ExpertWeights w, int experts, const int *__restrict__ ids, int slots, int per_row, const float *__restrict__ x,
                                                             float *__restrict__ y) {
    const int lane = threadIdx.x & 63, row = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const long long slot = (long long)blockIdx.z * 65535 + blockIdx.y;
    if (slot >= slots || row >= w.n) return;
    const int e = ids[slot];
    if ((unsigned)e >= (unsigned)experts) return;
    const uint8_t *wr = w.w + (size_t)e * w.expert_bytes + (size_t)row * ((size_t)(w.k / block_values(FMT)) * block_bytes(FMT));
    const float *xr = x + (size_t)(slot / per_row) * w.k;
    float acc = 0.f;
    for (int f = lane; f < (w.k >> 2); f += 64) {
        const float4 v = dequant4<FMT>(wr, (size_t)f * 4), xv = reinterpret_cast<const float4 *>(xr)[f];
        acc = __builtin_fmaf(v.w, xv.w, __builtin_fmaf(v.z, xv.z, __builtin_fmaf(v.y, xv.y, __builtin_fmaf(v.x, xv.x, acc))));
    }
    acc = wave_sum(acc);
    if (lane == 0) y[(size_t)slot * w.n + row] = acc;
}

template <int FMT>
static void value(const ExpertWeights &w, int experts, const int *ids, int slots, int per_row, const float *x, float *y, hipStream_t s) {
    const dim3 grid((w.n + 3) / 4, std::min(slots, 65535), (slots + 65534) / 65535);
    hipLaunchKernelGGL(experts_value_kernel<FMT>, grid, dim3(256), 0, s, w, experts, ids, slots, per_row, x, y);
}

void experts_value_launch(const ExpertWeights &w, int experts, const int *ids, int slots, int per_row, const float *x, float *y, hipStream_t s) {
    if (w.fmt == F_Q5_0) value<F_Q5_0>(w, experts, ids, slots, per_row, x, y, s);
    else value<F_Q3_K>(w, experts, ids, slots, per_row, x, y, s);
}

// ---- few tokens

static bool quants32(int fmt) { return block_values(fmt) == 32; }

bool experts_few_chooses(int experts) { return experts <= FEW_CHOICE; }

bool experts_few_up_supported(int fmt, int k) {
    return (quants32(fmt) ? fmt != F_Q5_0 && k % 64 == 0 : fmt != F_Q3_K) && k <= 1024 * I8_MAX_WAVES;  // (rows of whole chunks of 64 values)
}

static int few_stretches(int ffn, int used) { return (int)(((long long)used * ffn + 1023) / 1024); }
int experts_few_down_parts(int ffn, int used) { return (few_stretches(ffn, used) + 2 * I8_MAX_WAVES - 1) / (2 * I8_MAX_WAVES); }

bool experts_few_down_supported(int fmt, int ffn, int used) {
    return (quants32(fmt) ? fmt != F_Q5_0 && ffn % 64 == 0 : fmt != F_Q3_K) && experts_few_down_parts(ffn, used) <= 8;
}

// Workgroups for `groups` row groups of each of `tokens`, so many waves a CU in all and every workgroup as many turns as the others.
static int few_blocks(int groups, int tokens, int waves, int cus, int waves_per_cu) {
    const int most = std::max(1, std::max(1, waves_per_cu / waves) * cus / tokens), turns = (groups + most - 1) / most;
    return (groups + turns - 1) / turns;
}

void experts_few_up_launch(int fmt, ExpertFewArgs a, int tokens, int cus, hipStream_t s) {
    const int waves = (a.k + 1023) / 1024;
    const bool aligned = a.k % 512 == 0 && (((uintptr_t)a.w | (uintptr_t)a.w2) & 3) == 0;
    a.blocks = few_blocks(a.used * (a.n / 4), tokens, waves, cus, 8);
    a.by_rows = reciprocal((unsigned)(a.n / 4));
    const ExpertFewKernel fn = quants32(fmt) ? experts_few_up_q32(fmt, waves) : experts_few_up_k(fmt, aligned, waves);
    hipLaunchKernelGGL(fn, dim3(a.blocks, tokens), dim3(64 * waves), (size_t)waves * EF_WAVE_LDS, s, a);
}

void experts_few_down_launch(int fmt, ExpertFewArgs a, int tokens, int cus, hipStream_t s) {
    const int all = few_stretches(a.k, a.used), parts = experts_few_down_parts(a.k, a.used), each = (all + parts - 1) / parts, stretches = each > I8_MAX_WAVES ? 2 : 1,
              waves = (each + stretches - 1) / stretches;
    const bool aligned = a.k % 512 == 0 && ((uintptr_t)a.w & 3) == 0;
    a.blocks = few_blocks(a.n / 4, tokens * parts, waves, cus, 16);
    const ExpertFewKernel fn = quants32(fmt) ? experts_few_down_q32(fmt, stretches, waves) : experts_few_down_k(fmt, aligned, stretches, waves);
    hipLaunchKernelGGL(fn, dim3(a.blocks, tokens, parts), dim3(64 * waves), (size_t)waves * EF_WAVE_LDS, s, a);
}

// ---- on the matrix cores

size_t experts_ops_bytes(size_t rows, int k) {
    const size_t columns = rows * ((k + 255) / 256);
    return columns * (ER_OP_BYTES + sizeof(float));
}

ExpertPrepare experts_prepare(const float *x, int rows, int k, uint8_t *const *places) {
    ExpertPrepare p;
    p.x = x;
    p.rows = rows;
    p.k = k;
    for (int l = 0; l < GR_LAYOUTS; ++l) {
        p.ops[l] = places[l];
        p.inv[l] = places[l] ? reinterpret_cast<float *>(places[l] + (size_t)rows * ((k + 255) / 256) * ER_OP_BYTES) : nullptr;
    }
    return p;
}

__global__ void __launch_bounds__(64) experts_prepare_kernel(const ExpertPrepare p) { experts_prepare_unit(p, (int)blockIdx.x, threadIdx.x); }

void experts_prepare_launch(const ExpertPrepare &p, hipStream_t s) { hipLaunchKernelGGL(experts_prepare_kernel, dim3(p.units()), dim3(64), 0, s, p); }

RowsKernelRef experts_rows_kernel_ref(int fmt, int groups, bool pair) {
    return fmt == F_Q4_K || fmt == F_Q5_K ? experts_rows_ref_k(fmt, groups, pair) : fmt == F_Q6_K || fmt == F_Q2_K ? experts_rows_ref_k6(fmt, groups, pair)
                                                                                                                   : experts_rows_ref_q32(fmt, groups, pair);
}

void experts_rows_launch(const RowsKernelRef &k, ExpertRowsArgs a, int chunks_most, hipStream_t s) {
    a.nblocks = (a.n / 16 + k.tiles - 1) / k.tiles;
    hipLaunchKernelGGL(k.fn, dim3((unsigned)a.nblocks * (unsigned)a.splits * (unsigned)chunks_most), dim3(k.threads), k.lds, s, a);
}

static __global__ void __launch_bounds__(256) experts_gate_kernel(int act, const float *g, const float *__restrict__ u, float *h, size_t count4, unsigned stride) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < count4; i += stride) {
        float4 v = reinterpret_cast<const float4 *>(g)[i];
        const float4 m = reinterpret_cast<const float4 *>(u)[i];
        v = make_float4(activate(act, v.x) * m.x, activate(act, v.y) * m.y, activate(act, v.z) * m.z, activate(act, v.w) * m.w);
        reinterpret_cast<float4 *>(h)[i] = v;
    }
}

void experts_gate_launch(int act, const float *g, const float *u, float *h, size_t count, int cus, hipStream_t s) {
    const size_t count4 = count / 4;
    const unsigned blocks = (unsigned)std::min<size_t>((count4 + 255) / 256, (size_t)cus * 8);
    hipLaunchKernelGGL(experts_gate_kernel, dim3(blocks), dim3(256), 0, s, act, g, u, h, count4, blocks * 256);
}

// grid (ceil(n / 1024), tokens), 256 threads, four values each.  (res may be y)
static __global__ void __launch_bounds__(256) experts_combine_kernel(const float *__restrict__ part, int splits, size_t split_floats, const int *__restrict__ ids, const float *__restrict__ weights, const float *res,
                                                                     float *y, int used, int experts, int n) {
    const int t = (int)blockIdx.y, i = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
    if (i >= n) return;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < used; ++j) {
        const size_t slot = (size_t)t * used + j;
        if ((unsigned)ids[slot] >= (unsigned)experts) continue;
        const float w = weights[slot];
        float4 p = *reinterpret_cast<const float4 *>(part + slot * n + i);
        for (int z = 1; z < splits; ++z) {
            const float4 v = *reinterpret_cast<const float4 *>(part + z * split_floats + slot * n + i);
            p = make_float4(p.x + v.x, p.y + v.y, p.z + v.z, p.w + v.w);
        }
        sum.x = __builtin_fmaf(w, p.x, sum.x);
        sum.y = __builtin_fmaf(w, p.y, sum.y);
        sum.z = __builtin_fmaf(w, p.z, sum.z);
        sum.w = __builtin_fmaf(w, p.w, sum.w);
    }
    if (res) {
        const float4 r = *reinterpret_cast<const float4 *>(res + (size_t)t * n + i);
        sum = make_float4(sum.x + r.x, sum.y + r.y, sum.z + r.z, sum.w + r.w);
    }
    *reinterpret_cast<float4 *>(y + (size_t)t * n + i) = sum;
}

void experts_combine_launch(const float *part, int splits, const int *ids, const float *weights, const float *res, float *y, int tokens, int used, int experts, int n,
                            hipStream_t s) {
    hipLaunchKernelGGL(experts_combine_kernel, dim3((n + 1023) / 1024, tokens), dim3(256), 0, s, part, splits, (size_t)tokens * used * n, ids, weights, res, y, used, experts, n);
}

// (any alignment: outputs and residuals of linears need none)
static __global__ void __launch_bounds__(256) linear_epilogue_kernel(int act, const float *__restrict__ res, float *__restrict__ y, size_t count, unsigned stride) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < count; i += stride) {
        const float v = activate(act, y[i]);
        y[i] = res ? v + res[i] : v;
    }
}

void linear_epilogue_launch(int act, const float *res, float *y, size_t count, int cus, hipStream_t s) {
    const unsigned blocks = (unsigned)std::min<size_t>((count + 255) / 256, (size_t)cus * 16);
    hipLaunchKernelGGL(linear_epilogue_kernel, dim3(blocks), dim3(256), 0, s, act, res, y, count, blocks * 256);
}

}  // namespace jitnn
