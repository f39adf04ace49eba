// The router of a mixture of experts: logits l = x W^T, the `used` experts of a token, their weights.
//
// The sums are FP64: an expert next to the border of the choice has to fall on the same side whatever the order of a sum, and with FP32 sums one
// token in some ten thousand fell on another.  A product of two FP32 values is exact in FP64, so two orders of a sum differ by about 2^-50.
// The FP64 instructions cost little: 1000 tokens x 128 experts x 2048 values are 262 M multiply-adds, 7 us at the device's rate.
#pragma once
#include "common.h"
#include "experts.h"

namespace jitnn {

typedef double f64x4 __attribute__((ext_vector_type(4)));

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
__device__ __forceinline__ unsigned long long wave_maxu64(unsigned long long v) {
    return wave_fold64(v, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
}

// A number of which a larger value has the larger one; 1 for what is not a number, so that 0 is below all.
__device__ __forceinline__ unsigned long long order_of(double v) {
    if (v != v) return 1;
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);  // (-0 as 0: they are equal)
    return b >> 63 ? ~b : b | 1ull << 63;
}

// One logit: the wave's 64 lanes take four values of the row at a time.
__device__ __forceinline__ double router_dot(const float *__restrict__ x, const float *__restrict__ w, int d, int lane) {
    double acc[4] = {0, 0, 0, 0};
    int i = 4 * lane;
    for (; i + 3 * 256 < d; i += 4 * 256) {
        float4 xv[4], wv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            xv[j] = *reinterpret_cast<const float4 *>(x + i + 256 * j);
            wv[j] = *reinterpret_cast<const float4 *>(w + i + 256 * j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc[j] = fma((double)xv[j].w, (double)wv[j].w, fma((double)xv[j].z, (double)wv[j].z, fma((double)xv[j].y, (double)wv[j].y, fma((double)xv[j].x, (double)wv[j].x, acc[j]))));
    }
    for (; i < d; i += 256) {
        const float4 xv = *reinterpret_cast<const float4 *>(x + i), wv = *reinterpret_cast<const float4 *>(w + i);
        acc[0] = fma((double)xv.w, (double)wv.w, fma((double)xv.z, (double)wv.z, fma((double)xv.y, (double)wv.y, fma((double)xv.x, (double)wv.x, acc[0]))));
    }
    return wave_sum64((acc[0] + acc[1]) + (acc[2] + acc[3]));
}

// Few tokens: a wave per logit.  grid (ceil(experts / 4), tokens), 256 threads.
static __global__ void __launch_bounds__(256) router_logits_kernel(const RouterArgs a) {
    const int lane = threadIdx.x & 63, e = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (e >= a.experts) return;
    const double l = router_dot(a.x + (size_t)blockIdx.y * a.d, a.w + (size_t)e * a.d, a.d, lane);
    if (lane == 0) a.logits[(size_t)blockIdx.y * a.experts + e] = l;
}

// Many tokens: a workgroup's tile is 16 tokens x 16 experts, its four waves share out the values of a row, sixteen at a time: lane r + 16 q holds
// four consecutive values of row r, and product i of a step takes value i of each - the same four places of x and W, in whatever order.
// grid (ceil(tokens / 16), ceil(experts / 16)), 256 threads.
static __global__ void __launch_bounds__(256) router_tiles_kernel(const RouterArgs a) {
    __shared__ f64x4 sums[3][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int t0 = (int)blockIdx.x * 16, e0 = (int)blockIdx.y * 16;
    const float *xp = a.x + (size_t)min(t0 + r, a.tokens - 1) * a.d + 4 * q, *wp = a.w + (size_t)min(e0 + r, a.experts - 1) * a.d + 4 * q;
    f64x4 acc = {0, 0, 0, 0};
    auto step = [&](const float4 &xv, const float4 &wv) {
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv.x, (double)wv.x, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv.y, (double)wv.y, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv.z, (double)wv.z, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv.w, (double)wv.w, acc, 0, 0, 0);
    };
    int at = 16 * wave;
    for (; at + 3 * 64 + 16 <= a.d; at += 4 * 64) {
        float4 xv[4], wv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            xv[j] = *reinterpret_cast<const float4 *>(xp + at + 64 * j);
            wv[j] = *reinterpret_cast<const float4 *>(wp + at + 64 * j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) step(xv[j], wv[j]);
    }
    for (; at < a.d; at += 64) {
        float4 xv = make_float4(0.f, 0.f, 0.f, 0.f), wv = xv;
        if (at + 4 * q < a.d) {
            xv = *reinterpret_cast<const float4 *>(xp + at);
            wv = *reinterpret_cast<const float4 *>(wp + at);
        }
        step(xv, wv);
    }
    if (wave) sums[wave - 1][lane] = acc;
    __syncthreads();
    if (wave) return;
    acc = (acc + sums[0][lane]) + (sums[1][lane] + sums[2][lane]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // lane r + 16 q: column (expert) r, rows (tokens) q + 4 i
        const int t = t0 + q + 4 * i, e = e0 + r;
        if (t < a.tokens && e < a.experts) a.logits[(size_t)t * a.experts + e] = acc[i];
    }
}

// The choice of one token by one wave: l [experts] (logits) and key [experts] in LDS, each place of both read and written by one lane only -
// but for the logits of the chosen.  Lane j < used gets the token's j-th expert and its weight.
__device__ __forceinline__ void choose_experts(const RouterArgs &a, const double *l, unsigned long long *key, int lane, int &id, float &weight) {
    double top = -INFINITY, sum = 0;
    if (!a.sigmoid && (a.bias || !a.normalise)) {
        for (int i = lane; i < a.experts; i += 64) top = fmax(top, l[i]);
        top = wave_max64(top);
        for (int i = lane; i < a.experts; i += 64) sum += exp(l[i] - top);
        sum = wave_sum64(sum);
    }
    auto share = [&](double v) { return a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - top) / sum; };
    for (int i = lane; i < a.experts; i += 64) key[i] = order_of(a.bias ? share(l[i]) + (double)a.bias[i] : l[i]);
    id = 0;
    for (int j = 0; j < a.used; ++j) {
        unsigned long long best = 0;
        for (int i = lane; i < a.experts; i += 64) best = key[i] > best ? key[i] : best;
        best = wave_maxu64(best);
        int at = 0;
        for (int i0 = 0;; i0 += 64) {  // (one of them has it)
            const unsigned long long have = __builtin_amdgcn_ballot_w64(i0 + lane < a.experts && key[min(i0 + lane, a.experts - 1)] == best);
            if (have || i0 + 64 >= a.experts) {
                at = i0 + (have ? __builtin_ctzll(have) : 0);
                break;
            }
        }
        if (lane == (at & 63)) key[at] = 0;
        if (lane == j) id = at;
    }
    const bool mine = lane < a.used;
    const double v = mine ? l[id] : -INFINITY;
    double w;
    if (a.normalise) {
        // (softmax: by the largest of the chosen, whose weight then is no quotient of two small numbers)
        const double m = a.sigmoid ? 0.0 : wave_max64(v);
        const double e = !mine ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - m);
        w = e / wave_sum64(e);
    } else {
        w = share(v);
    }
    weight = (float)(w * (double)a.scale);
}

__device__ __forceinline__ void store_choice(const RouterArgs &a, int t, int lane, int id, float weight) {
    if (lane < a.used) {
        a.ids[(size_t)t * a.used + lane] = id;
        a.weights[(size_t)t * a.used + lane] = weight;
    }
}

// The lists of each expert's slots and their chunks, by one workgroup of 1024 threads: counted, summed up, handed out.  (In what order a list holds its slots
// is no part of any result: each row of a product is computed by itself.)  hist: [MAX_EXPERTS] in LDS.
template <class Id>
__device__ __forceinline__ void make_lists(Id &&id_of, int slots, int experts, const ExpertLists &lists, int *hist) {
    const int tid = threadIdx.x, lane = tid & 63;
    for (int e = tid; e < experts; e += 1024) hist[e] = 0;
    __syncthreads();
    for (int i = tid; i < slots; i += 1024) {
        const int e = id_of(i);
        if ((unsigned)e < (unsigned)experts) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    if (tid < 64) {
        int run = 0, made = 0;
        for (int e0 = 0; e0 < experts; e0 += 64) {
            const int e = e0 + lane, mine = e < experts ? hist[e] : 0, chunks = (mine + lists.chunk_rows - 1) / lists.chunk_rows;
            int sum = mine, chunk_sum = chunks;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int below = __shfl_up(sum, o), chunk_below = __shfl_up(chunk_sum, o);
                sum += lane >= o ? below : 0;
                chunk_sum += lane >= o ? chunk_below : 0;
            }
            const int first = run + sum - mine;
            if (e < experts) hist[e] = first;
            for (int i = 0; i < chunks; ++i) {  // (as even as whole rows allow)
                const int from = (int)((long long)mine * i / chunks), to = (int)((long long)mine * (i + 1) / chunks);
                lists.chunks[1 + made + chunk_sum - chunks + i] = int4{e, first + from, to - from, 0};
            }
            run += __shfl(sum, 63);
            made += __shfl(chunk_sum, 63);
        }
        if (lane == 0) lists.chunks[0] = int4{made, 0, 0, 0};
    }
    __syncthreads();
    for (int i = tid; i < slots; i += 1024) {
        const int e = id_of(i);
        if ((unsigned)e < (unsigned)experts) lists.list[atomicAdd(&hist[e], 1)] = i;
    }
}

// A wave per token.  ceil(tokens / 4) workgroups of 256 threads, 64 bytes of LDS per expert.
static __global__ void __launch_bounds__(256) choose_kernel(const RouterArgs a) {
    extern __shared__ __align__(16) double choose_smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), t = (int)blockIdx.x * 4 + wave;
    if (t >= a.tokens) return;
    double *l = choose_smem + (size_t)wave * 2 * a.experts;
    for (int i = lane; i < a.experts; i += 64) l[i] = a.logits[(size_t)t * a.experts + i];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    int id;
    float weight;
    choose_experts(a, l, reinterpret_cast<unsigned long long *>(l + a.experts), lane, id, weight);
    store_choice(a, t, lane, id, weight);
}

// Few tokens, one workgroup: the choices of all of them and the experts' lists.  LDS: 16 bytes per expert for each of `waves` waves.
constexpr int CHOOSE_FEW = 64;
static __global__ void __launch_bounds__(1024) choose_few_kernel(const RouterArgs a, int waves) {
    extern __shared__ __align__(16) double choose_smem[];
    __shared__ int ids[CHOOSE_FEW * MAX_USED], hist[MAX_EXPERTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    double *l = choose_smem + (size_t)wave * 2 * a.experts;
    for (int t = wave; wave < waves && t < a.tokens; t += waves) {
        for (int i = lane; i < a.experts; i += 64) l[i] = a.logits[(size_t)t * a.experts + i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        int id;
        float weight;
        choose_experts(a, l, reinterpret_cast<unsigned long long *>(l + a.experts), lane, id, weight);
        store_choice(a, t, lane, id, weight);
        if (lane < a.used) ids[t * a.used + lane] = id;
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    make_lists([&](int i) { return ids[i]; }, a.tokens * a.used, a.experts, a.lists, hist);
}

static __global__ void __launch_bounds__(1024) expert_lists_kernel(const int *__restrict__ ids, int slots, int experts, const ExpertLists lists) {
    __shared__ int hist[MAX_EXPERTS];
    make_lists([&](int i) { return ids[i]; }, slots, experts, lists, hist);
}

// A router whose weights one workgroup reads in about the time that a second launch would take: logits and choice of a token, 1024 threads.
static __global__ void __launch_bounds__(1024) router_one_kernel(const RouterArgs a) {
    __shared__ double l[MAX_EXPERTS];
    __shared__ unsigned long long key[MAX_EXPERTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), t = (int)blockIdx.x;
    for (int e = wave; e < a.experts; e += 16) {
        const double v = router_dot(a.x + (size_t)t * a.d, a.w + (size_t)e * a.d, a.d, lane);
        if (lane == 0) l[e] = v;
    }
    __syncthreads();
    if (wave) return;
    int id;
    float weight;
    choose_experts(a, l, key, lane, id, weight);
    store_choice(a, t, lane, id, weight);
}

}  // namespace jitnn
