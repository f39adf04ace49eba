// The router of a mixture of experts: logits l = x W^T, the `used` experts of a token, their weights.
//
// The sums are FP64: an expert next to the border of the choice has to fall on the same side whatever the order of a sum, and with FP32 sums one
// token in some ten thousand fell on another.  A product of two FP32 values is exact in FP64, so two orders of a sum differ by about 2^-50.
// The FP64 instructions cost little: 1000 tokens x 128 experts x 2048 values are 262 M multiply-adds, 7 us at the device's rate.
#pragma once
#include "common.h"
#include "experts.h"

namespace jitnn {

template <int CTRL>
__device__ __forceinline__ unsigned long long dpp64(unsigned long long v) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp((int)(unsigned)v, (int)(unsigned)v, CTRL, 0xF, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp((int)(unsigned)(v >> 32), (int)(unsigned)(v >> 32), CTRL, 0xF, 0xF, false);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ unsigned long long lane64(unsigned long long v, int lane) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), lane);
    return (unsigned long long)hi << 32 | lo;
}
// over the 64 lanes of a wave, for every lane
template <class T, class Op>
__device__ __forceinline__ T wave_fold64(T v, Op op) {
    auto other = [](unsigned long long b) { return __builtin_bit_cast(T, b); };
    v = op(v, other(dpp64<0xB1>(__builtin_bit_cast(unsigned long long, v))));   // quad_perm [1,0,3,2]
    v = op(v, other(dpp64<0x4E>(__builtin_bit_cast(unsigned long long, v))));   // quad_perm [2,3,0,1]
    v = op(v, other(dpp64<0x141>(__builtin_bit_cast(unsigned long long, v))));  // row_half_mirror
    v = op(v, other(dpp64<0x140>(__builtin_bit_cast(unsigned long long, v))));  // row_mirror
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    return op(op(other(lane64(b, 0)), other(lane64(b, 16))), op(other(lane64(b, 32)), other(lane64(b, 48))));
}
__device__ __forceinline__ double wave_sum64(double v) { return wave_fold64(v, [](double a, double b) { return a + b; }); }
__device__ __forceinline__ double wave_max64(double v) { return wave_fold64(v, [](double a, double b) { return fmax(a, b); }); }
__device__ __forceinline__ unsigned wave_maxu(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xF, 0xF, false));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xF, 0xF, false));
    auto lane = [&](int i) { return (unsigned)__builtin_amdgcn_readlane((int)v, i); };
    return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}

// A number of which a larger value has the larger one; 1 for what is not a number, so that 0 is below all.
__device__ __forceinline__ unsigned long long order_of(double v) {
    if (v != v) return 1;
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);  // (-0 as 0: they are equal)
    return b >> 63 ? ~b : b | 1ull << 63;
}

// The choice of one token by one wave: lane i has the logits l of experts i, i + 64, ... (L of them at most); lane j < used gets the token's j-th expert and its weight.
// A turn takes the largest of the lanes' largest: by the upper halves of their orders, where two lanes share that by the lower ones, and where they are equal by
// index.  Only the lane whose expert was taken looks for its next one.
template <int L>
__device__ __forceinline__ void choose_experts(const RouterArgs &a, const double (&l)[L], int lane, int &id, float &weight) {
    double top = -INFINITY, sum = 0;
    if (!a.sigmoid && (a.bias || !a.normalise)) {
#pragma unroll
        for (int i = 0; i < L; ++i)
            if (64 * i + lane < a.experts) top = fmax(top, l[i]);
        top = wave_max64(top);
#pragma unroll
        for (int i = 0; i < L; ++i)
            if (64 * i + lane < a.experts) sum += exp(l[i] - top);
        sum = wave_sum64(sum);
    }
    auto share = [&](double v) { return a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - top) / sum; };
    unsigned long long key[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        key[i] = 0;
        if (64 * i + lane < a.experts) key[i] = order_of(a.bias ? share(l[i]) + (double)a.bias[64 * i + lane] : l[i]);
    }
    unsigned long long best = 0;
    int which = 0;
    double logit = 0;
    auto look = [&]() {
        best = 0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            if (key[i] > best) {
                best = key[i];
                which = i;
                logit = l[i];
            }
        }
    };
    look();
    id = 0;
    double mine = -INFINITY;
    for (int j = 0; j < a.used; ++j) {
        const unsigned hi = (unsigned)(best >> 32), most = wave_maxu(hi);
        unsigned long long have = __builtin_amdgcn_ballot_w64(hi == most);
        if (have & (have - 1)) {
            const unsigned lo = hi == most ? (unsigned)best : 0u, most_lo = wave_maxu(lo);
            const bool equal = hi == most && (unsigned)best == most_lo;
            have = __builtin_amdgcn_ballot_w64(equal);
            if (have & (have - 1)) {
                const unsigned first = ~wave_maxu(equal ? ~(unsigned)(64 * which + lane) : 0u);
                have = 1ull << (first & 63u);
            }
        }
        const int winner = __builtin_ctzll(have);
        const int at = 64 * __builtin_amdgcn_readlane(which, winner) + winner;
        const double v = __builtin_bit_cast(double, lane64(__builtin_bit_cast(unsigned long long, logit), winner));
        if (lane == j) {
            id = at;
            mine = v;
        }
        if (lane == winner) {
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (i == which) key[i] = 0;
            look();
        }
    }
    double w;
    if (a.normalise) {
        // (softmax: by the largest of the chosen, whose weight then is no quotient of two small numbers)
        const bool chosen = lane < a.used;
        const double m = a.sigmoid ? 0.0 : wave_max64(mine);
        const double e = !chosen ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-mine)) : exp(mine - m);
        w = e / wave_sum64(e);
    } else {
        w = share(mine);
    }
    weight = (float)(w * (double)a.scale);
}

// The logits of token t, added up over the splits they were computed in.
template <int L>
__device__ __forceinline__ void load_logits(const RouterArgs &a, int t, int lane, double (&l)[L]) {
    const double *p = a.logits + (size_t)t * a.experts;
#pragma unroll
    for (int i = 0; i < L; ++i) l[i] = p[min(64 * i + lane, a.experts - 1)];
    for (int z = 1; z < a.splits; ++z) {
        p += (size_t)a.tokens * a.experts;
#pragma unroll
        for (int i = 0; i < L; ++i) l[i] += p[min(64 * i + lane, a.experts - 1)];
    }
}

__device__ __forceinline__ void store_choice(const RouterArgs &a, int t, int lane, int id, float weight) {
    if (lane < a.used) {
        a.ids[(size_t)t * a.used + lane] = id;
        a.weights[(size_t)t * a.used + lane] = weight;
    }
}

}  // namespace jitnn
