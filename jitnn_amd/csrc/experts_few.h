// The experts' products of a few (token, expert) pairs: INT8 matrix-core products on the raw quants, gemv_i8.h's units and its activations in three byte digits.
//
// A launch per product, a token along blockIdx.y.  Gate and up: a workgroup's waves hold the token's row as digits - the same one for all its experts - and walk the
// rows of all of them, four at a time, gate and up by turns.  Down: the token's experts stand one behind the other as ONE long row, used x ffn values of which each
// stretch meets another expert's weights and has been multiplied by that expert's share, so that y is one dot product per row of d_model: no joining launch, and
// the order of the sums does not depend on the launch's shape.
// A row with a value that is not finite gives a row of NaN.
// Bound by memory: one token, two of eight experts of 4096 x 14336, gate and up in Q4_K 132 MB in 27.2 us (4.9 TB/s), down in Q6_K 96 MB in 23.2 (4.1), 51.1 us for the layer; eight of
// 128 of 2048 x 768 14 MB in 9.8 and 10 MB in 8.6: starts and dependent reads - logits, choice, weights.
#pragma once
#include "act.h"
#include "common.h"
#include "experts.h"
#include "gemv_i8.h"
#include "router.h"

namespace jitnn {

constexpr int FEW_CHOICE = 128;  // experts of which the first kernel makes the choice itself

// Turns between two joins of the waves' sums, and a wave's LDS: the digits while they are staged, then two windows of sums.
constexpr int EF_FLUSH = 24;
constexpr size_t EF_WAVE_LDS = (size_t)2 * EF_FLUSH * 16 * sizeof(float);
static_assert(EF_WAVE_LDS >= 16 * 3 * 64, "sixteen chunks of three planes");

// The digits hold a chunk to 2^-127 at best.  Where a wave's values are all below 2^-63 - products of two small numbers reach that - they are staged times
// 2^64, and its sums count that much less; beside a larger value the same steps are nothing.
__device__ __forceinline__ float few_lift(float4 (&xv)[4]) {
    uint32_t am = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        am = max(max(am, max(__float_as_uint(xv[i].x) & 0x7fffffffu, __float_as_uint(xv[i].y) & 0x7fffffffu)),
                 max(__float_as_uint(xv[i].z) & 0x7fffffffu, __float_as_uint(xv[i].w) & 0x7fffffffu));
    if (__builtin_amdgcn_ballot_w64(am >= 64u << 23) != 0) return 1.f;
    const float up = 0x1p64f;
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = make_float4(xv[i].x * up, xv[i].y * up, xv[i].z * up, xv[i].w * up);
    return 0x1p-64f;
}

// The values as their digits hold them, 2^-22 of a chunk's largest and less: so the sums of x, which meet the offsets of quants and minima, are those of what the quants meet, and
// a rounding counts with the quant less its offset.  (Half as far off: two of eight experts of 4096 x 14336 1.3e-6 -> 6.2e-7 against 64 bits, for 0.3 us.)
__device__ __forceinline__ void few_round(float4 (&xv)[4]) {
    uint32_t am = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        am = max(max(am, max(__float_as_uint(xv[i].x) & 0x7fffffffu, __float_as_uint(xv[i].y) & 0x7fffffffu)),
                 max(__float_as_uint(xv[i].z) & 0x7fffffffu, __float_as_uint(xv[i].w) & 0x7fffffffu));
    am = max(am, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)am, 0xB1, 0xF, 0xF, true));  // quad_perm [1,0,3,2]
    am = max(am, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)am, 0x4E, 0xF, 0xF, true));  // quad_perm [2,3,0,1]
    if (__builtin_amdgcn_ballot_w64(am - 0x7f7ffffeu < 2u) != 0) {  // (the two largest finite values would become infinite: the next one below, which does not)
        auto finite = [](float v) {
            const uint32_t u = __float_as_uint(v), m = u & 0x7fffffffu;
            return m - 0x7f7ffffeu < 2u ? __uint_as_float(u - (m - 0x7f7ffffdu)) : v;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = make_float4(finite(xv[i].x), finite(xv[i].y), finite(xv[i].z), finite(xv[i].w));
        am = am - 0x7f7ffffeu < 2u ? 0x7f7ffffdu : am;
    }
    // (the scale that i8_stage takes, which finds these values whole: the exponent behind the rounding, which the two largest mantissas of 24 bits raise)
    const uint32_t eb = min(max((am + 2u) >> 23, 22u), 254u);
    const float up = __uint_as_float((275u - eb) << 23), down = __uint_as_float((eb - 21u) << 23);
    auto rounded = [&](float v) { return (__builtin_fmaf(v, up, 12582912.f) - 12582912.f) * down; };
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = make_float4(rounded(xv[i].x), rounded(xv[i].y), rounded(xv[i].z), rounded(xv[i].w));
}

// Two DPP steps fold the sixteen chunks of a row in a wave to four sums.
__device__ __forceinline__ void few_emit(float acc, float *part, int turn, int lane) {
    acc += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(acc), 0x114, 0xF, 0xF, true));  // row_shr:4
    acc += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(acc), 0x118, 0xF, 0xF, true));  // row_shr:8
    if ((lane & 15) >= 12) part[turn * 16 + (lane >> 4) * 4 + (lane & 3)] = acc;
}
// The sums of all waves for row jj of a turn, in wave order.
template <int MAXW>
__device__ __forceinline__ float few_joined(const uint8_t *smem, int waves, int turn, int jj) {
    float part[MAXW], sum = 0.f;
#pragma unroll
    for (int w = 0; w < MAXW; ++w) {
        const float *p = reinterpret_cast<const float *>(smem + (size_t)min(w, waves - 1) * EF_WAVE_LDS) + turn * 16 + jj;
        part[w] = (p[0] + p[4]) + (p[8] + p[12]);
    }
#pragma unroll
    for (int w = 0; w < MAXW; ++w) sum += w < waves ? part[w] : 0.f;
    return sum;
}

// h [token, used, ffn] = act(gate x) * (up x).  grid (a.blocks, tokens), a wave per 1024 values of a row; gate and up of one format.
template <class U, int PF, int MAXW>
__global__ void __launch_bounds__(64 * MAXW, 4) experts_few_up_kernel(const ExpertFewArgs a) {
    constexpr int NB = PF + 1;
    static_assert(EF_FLUSH % NB == 0 && EF_FLUSH % 2 == 0, "whole rings and pairs per window");
    extern __shared__ __align__(16) uint8_t ef_smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (a.k + 1023) >> 10;
    float *const part = reinterpret_cast<float *>(ef_smem + (size_t)wave * EF_WAVE_LDS);
    const int b = lane >> 2, j = lane & 3, chunks = a.k >> 6, token = (int)blockIdx.y;
    const bool inrow = wave * 16 + b < chunks;
    const int c = inrow ? wave * 16 + b : chunks - 1;
    const uint32_t rowbytes = (uint32_t)(a.k / block_values(U::FMT)) * block_bytes(U::FMT);
    const typename U::Off off = U::offsets(c, (uint32_t)j * rowbytes);
    const float *const x = a.x + (size_t)token * a.k;
    float4 xv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) xv[i] = reinterpret_cast<const float4 *>(x + U::x_first(c, j))[i];
    // the token's experts, one a lane; those that are none read nothing
    int mine;
    if (a.route.logits) {  // (up to 3 us before a wave's first weights, of 128 experts; a launch in front took 4 and more)
        double l[FEW_CHOICE / 64];
        load_logits(a.route, token, lane, l);
        float weight;
        choose_experts(a.route, l, lane, mine, weight);
        if (blockIdx.x == 0 && wave == 0) store_choice(a.route, token, lane, mine, weight);
    } else {
        mine = lane < a.used ? a.ids[(size_t)token * a.used + lane] : -1;
    }
    const int per = a.n >> 2, groups = a.used * per;  // groups of four rows: of an expert (its rows are a multiple of 32), of the token
    const int turns = 2 * ((groups + a.blocks - 1) / a.blocks);
    typename U::Raw buf[NB];
    auto fill = [&](typename U::Raw &dst, int t) {
        const int g = (int)blockIdx.x + (t >> 1) * a.blocks;
        int place = (int)__umulhi((unsigned)g, a.by_rows), row = g - place * per;  // (the reciprocal is too small by less than one part in 2^32: one off at most)
        if (row >= per) {
            ++place;
            row -= per;
        }
        const int e = __builtin_amdgcn_readlane(mine, place & 63);
        // (nothing of a group behind the last one, nor of an expert that does not exist: by arithmetic, so that the descriptor stays in scalar registers)
        const int extent = __builtin_amdgcn_readfirstlane(g < groups && (unsigned)e < (unsigned)a.experts ? -1 : 0);
        const uint8_t *const base = (t & 1 ? a.w2 : a.w) + (size_t)(unsigned)(e & extent) * a.expert_bytes;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, extent, 0x00020000);
        U::load(dst, rs, off, (uint32_t)(row * 4 & extent) * rowbytes);
    };
#pragma unroll
    for (int i = 0; i < NB; ++i) fill(buf[i], i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t m = inrow ? 0xffffffffu : 0u;
        xv[i] = make_float4(__uint_as_float(__float_as_uint(xv[i].x) & m), __uint_as_float(__float_as_uint(xv[i].y) & m), __uint_as_float(__float_as_uint(xv[i].z) & m),
                            __uint_as_float(__float_as_uint(xv[i].w) & m));
    }
    uint32_t xa[1][16];
    float sinv[1], sums[1][U::NSUM];
    const float lift = few_lift(xv);
    few_round(xv);
    const float odd = i8_stage<U>(xv, reinterpret_cast<u32x4 *>(part), b, j, xa[0], sinv[0], sums[0]) ? NAN : 0.f;
    for (int t0 = 0, half = 0; t0 < turns; t0 += EF_FLUSH, half ^= 1) {
        const int tend = min(t0 + EF_FLUSH, turns);
#pragma unroll 1
        for (int tb = t0; tb < tend; tb += NB) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int t = tb + i;
                if (t < tend) {
                    float acc[1];
                    i8_dot<U, 1>(buf[i], c, xa, sinv, sums, acc);
                    few_emit((inrow ? acc[0] * lift : 0.f) + odd, part, half * EF_FLUSH + t - t0, lane);
                }
                fill(buf[i], t + NB);
            }
        }
        __syncthreads();
        for (int o = tid; o < 2 * (tend - t0); o += 64 * waves) {
            const int pr = o >> 2, jj = o & 3, g = (int)blockIdx.x + (t0 / 2 + pr) * a.blocks;
            if (g < groups) {
                const float gate = few_joined<MAXW>(ef_smem, waves, half * EF_FLUSH + 2 * pr, jj), up = few_joined<MAXW>(ef_smem, waves, half * EF_FLUSH + 2 * pr + 1, jj);
                a.y[(size_t)token * groups * 4 + 4 * g + jj] = activate(a.act, gate) * up;
            }
        }
    }
}

// y [token, n] = res + the sum over the token's places of share * (down h).  grid (a.blocks, tokens, parts); wave w takes stretches w, w + waves, ... (S at most) of 1024 values of its
// part of the long row, which has a y of its own.
template <class U, int S, int PF, int MAXW>
__global__ void __launch_bounds__(64 * MAXW, MAXW > 8 ? 4 : 2) experts_few_down_kernel(const ExpertFewArgs a) {
    constexpr int NB = PF + 1;
    static_assert(EF_FLUSH % NB == 0, "whole rings per window");
    extern __shared__ __align__(16) uint8_t ef_smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)(blockDim.x >> 6);
    float *const part = reinterpret_cast<float *>(ef_smem + (size_t)wave * EF_WAVE_LDS);
    const int b = lane >> 2, j = lane & 3, per = a.k >> 6, chunks = a.used * per, token = (int)blockIdx.y, first = (int)blockIdx.z * S * waves * 16;
    const uint32_t rowbytes = (uint32_t)(a.k / block_values(U::FMT)) * block_bytes(U::FMT);
    const int groups = a.n >> 2, turns = (groups + a.blocks - 1) / a.blocks;
    typename U::Off off[S];
    bool live[S];
    int cc[S];
    float4 xv[S][4];
    float share[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int at = first + (wave + s * waves) * 16 + b;
        const int c = min(at, chunks - 1), place = c / per;
        cc[s] = c - place * per;
        const int e = a.ids[(size_t)token * a.used + place];
        live[s] = at < chunks && (unsigned)e < (unsigned)a.experts;
        share[s] = a.weights[(size_t)token * a.used + place];
        off[s] = U::offsets(cc[s], (uint32_t)(live[s] ? e : 0) * (uint32_t)a.expert_bytes + (uint32_t)j * rowbytes);
        const float *const h = a.x + ((size_t)token * a.used + place) * a.k + U::x_first(cc[s], j);
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[s][i] = reinterpret_cast<const float4 *>(h)[i];
    }
    typename U::Raw buf[NB][S];
    auto fill = [&](typename U::Raw &dst, int s, int t) {
        const int g = (int)blockIdx.x + t * a.blocks, extent = __builtin_amdgcn_readfirstlane((g - groups) >> 31);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.w), 0, extent, 0x00020000);
        U::load(dst, rs, off[s], (uint32_t)(4 * g & extent) * rowbytes);
    };
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int s = 0; s < S; ++s) fill(buf[i][s], s, i);
    }
    __builtin_amdgcn_sched_barrier(0);
    uint32_t xa[S][1][16];
    float sinv[S][1], sums[S][1][U::NSUM], lift[S], odd = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const float f = live[s] ? share[s] : 0.f;
        auto times = [&](float v) { return live[s] ? v * f : 0.f; };
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[s][i] = make_float4(times(xv[s][i].x), times(xv[s][i].y), times(xv[s][i].z), times(xv[s][i].w));
        lift[s] = few_lift(xv[s]);
        few_round(xv[s]);
        odd = i8_stage<U>(xv[s], reinterpret_cast<u32x4 *>(part), b, j, xa[s][0], sinv[s][0], sums[s][0]) ? NAN : odd;
    }
    for (int t0 = 0, half = 0; t0 < turns; t0 += EF_FLUSH, half ^= 1) {
        const int tend = min(t0 + EF_FLUSH, turns);
#pragma unroll 1
        for (int tb = t0; tb < tend; tb += NB) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int t = tb + i;
                float sum = odd;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    if (t < tend) {
                        float acc[1];
                        i8_dot<U, 1>(buf[i][s], cc[s], xa[s], sinv[s], sums[s], acc);
                        sum += live[s] ? acc[0] * lift[s] : 0.f;
                    }
                    fill(buf[i][s], s, t + NB);
                }
                if (t < tend) few_emit(sum, part, half * EF_FLUSH + t - t0, lane);
            }
        }
        __syncthreads();
        for (int o = tid; o < 4 * (tend - t0); o += 64 * waves) {
            const int tt = o >> 2, jj = o & 3, g = (int)blockIdx.x + (t0 + tt) * a.blocks;
            if (g < groups) {
                const size_t to = ((size_t)blockIdx.z * gridDim.y + token) * a.n + 4 * g + jj;
                const float sum = few_joined<MAXW>(ef_smem, waves, half * EF_FLUSH + tt, jj);
                a.y[to] = a.res ? sum + a.res[to] : sum;
            }
        }
    }
}

template <class U>
static ExpertFewKernel experts_few_up_pick(int waves) {
    return waves <= 4 ? experts_few_up_kernel<U, 2, 4> : experts_few_up_kernel<U, 1, 16>;
}
template <class U>
static ExpertFewKernel experts_few_down_pick(int stretches, int waves) {
    if (stretches > 1) return experts_few_down_kernel<U, 2, 0, 16>;
    return waves <= 8 ? experts_few_down_kernel<U, 1, 2, 8> : experts_few_down_kernel<U, 1, 1, 16>;
}

}  // namespace jitnn
