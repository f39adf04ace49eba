// The router of a mixture of experts: its logits, the choices of a batch and the lists of what each expert gets.
#include "experts_rows.h"
#include "router.h"

#include <algorithm>
#include <type_traits>

namespace jitnn {

typedef double f64x4 __attribute__((ext_vector_type(4)));

// The share of one wave in a logit: quads first, first + step, ... of a row.
__device__ __forceinline__ double router_dot(const float *__restrict__ x, const float *__restrict__ w, int d, int first, int step) {
    double acc[4] = {0, 0, 0, 0};
    int i = 4 * first;
    step *= 4;
    for (; i + 3 * step < d; i += 4 * step) {
        float4 xv[4], wv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            xv[j] = *reinterpret_cast<const float4 *>(x + i + step * j);
            wv[j] = *reinterpret_cast<const float4 *>(w + i + step * j);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            acc[j] = fma((double)xv[j].w, (double)wv[j].w, fma((double)xv[j].z, (double)wv[j].z, fma((double)xv[j].y, (double)wv[j].y, fma((double)xv[j].x, (double)wv[j].x, acc[j]))));
    }
    for (; i < d; i += step) {
        const float4 xv = *reinterpret_cast<const float4 *>(x + i), wv = *reinterpret_cast<const float4 *>(w + i);
        acc[0] = fma((double)xv.w, (double)wv.w, fma((double)xv.z, (double)wv.z, fma((double)xv.y, (double)wv.y, fma((double)xv.x, (double)wv.x, acc[0]))));
    }
    return wave_sum64((acc[0] + acc[1]) + (acc[2] + acc[3]));
}

// Few tokens: a workgroup per logit, whose four waves share out the row.  grid (experts, tokens), 256 threads.
__global__ void __launch_bounds__(256) router_logits_kernel(const RouterArgs a) {
    __shared__ double sums[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), e = (int)blockIdx.x;
    const double l = router_dot(a.x + (size_t)blockIdx.y * a.d, a.w + (size_t)e * a.d, a.d, (int)threadIdx.x, 256);
    if (lane == 0) sums[wave] = l;
    __syncthreads();
    if (threadIdx.x == 0) a.logits[(size_t)blockIdx.y * a.experts + e] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// Many tokens: a workgroup's tile is 16 P tokens x 16 P experts, its four waves share out the values of its share of a row (a.splits of them along blockIdx.z, each with logits
// of its own), sixteen at a time: lane r + 16 q holds four consecutive values of row r, and product i of a step takes value i of each - the same four places of x and W, in
// whatever order.  What the L2s give bounds it, and a tile of 32 x 32 asks for half of what four of 16 x 16 do: 1000 tokens x 128 experts x 2048 values 16 us against 19 (17 with twice the splits).
// grid (ceil(tokens / 16 P), ceil(experts / 16 P), a.splits), 256 threads.
template <int P>
__global__ void __launch_bounds__(256) router_tiles_kernel(const RouterArgs a) {
    constexpr int AT_ONCE = 4; // steps whose loads are under way
    __shared__ f64x4 sums[3][P * P][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int t0 = (int)blockIdx.x * 16 * P, e0 = (int)blockIdx.y * 16 * P, steps = (a.d + 15) >> 4;
    const int from = (int)((long long)steps * blockIdx.z / a.splits) * 16, to = min((int)((long long)steps * (blockIdx.z + 1) / a.splits) * 16, a.d);
    const float *xp[P], *wp[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        xp[i] = a.x + (size_t)min(t0 + 16 * i + r, a.tokens - 1) * a.d + 4 * q;
        wp[i] = a.w + (size_t)min(e0 + 16 * i + r, a.experts - 1) * a.d + 4 * q;
    }
    f64x4 acc[P][P];
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < P; ++j) acc[i][j] = f64x4{0, 0, 0, 0};
    auto step = [&](const float4 (&xv)[P], const float4 (&wv)[P]) {
        auto products = [&](auto part) {
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int j = 0; j < P; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)part(xv[i]), (double)part(wv[j]), acc[i][j], 0, 0, 0);
        };
        products([](const float4 &v) { return v.x; });
        products([](const float4 &v) { return v.y; });
        products([](const float4 &v) { return v.z; });
        products([](const float4 &v) { return v.w; });
    };
    int at = from + 16 * wave;
    for (; at + (AT_ONCE - 1) * 64 + 16 <= to; at += AT_ONCE * 64) {
        float4 xv[AT_ONCE][P], wv[AT_ONCE][P];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                xv[j][i] = *reinterpret_cast<const float4 *>(xp[i] + at + 64 * j);
                wv[j][i] = *reinterpret_cast<const float4 *>(wp[i] + at + 64 * j);
            }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) step(xv[j], wv[j]);
    }
    for (; at < to; at += 64) {
        float4 xv[P], wv[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            xv[i] = wv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at + 4 * q < to) {
                xv[i] = *reinterpret_cast<const float4 *>(xp[i] + at);
                wv[i] = *reinterpret_cast<const float4 *>(wp[i] + at);
            }
        }
        step(xv, wv);
    }
#pragma unroll
    for (int i = 0; i < P * P; ++i)
        if (wave) sums[wave - 1][i][lane] = acc[i / P][i % P];
    __syncthreads();
    double *const logits = a.logits + (size_t)blockIdx.z * a.tokens * a.experts;
#pragma unroll
    for (int n = 0; n < P * P; ++n) {
        if (wave) continue;
        const f64x4 sum = (acc[n / P][n % P] + sums[0][n][lane]) + (sums[1][n][lane] + sums[2][n][lane]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // lane r + 16 q: column (expert) r, rows (tokens) q + 4 i
            const int t = t0 + 16 * (n / P) + q + 4 * i, e = e0 + 16 * (n % P) + r;
            if (t < a.tokens && e < a.experts) logits[(size_t)t * a.experts + e] = sum[i];
        }
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
            const int each = chunks > 1 ? mine / chunks : mine, more = mine - each * chunks;  // (as even as whole rows allow)
            for (int i = 0; i < chunks; ++i) lists.chunks[1 + made + chunk_sum - chunks + i] = int4{e, first + i * each + min(i, more), each + (i < more), 0};
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

// A wave per token.  ceil(tokens / 4) workgroups of 256 threads; L: see choose_experts.
template <int L>
__global__ void __launch_bounds__(256) choose_kernel(const RouterArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), t = (int)blockIdx.x * 4 + wave;
    if (t >= a.tokens) return;
    double l[L];
    load_logits(a, t, lane, l);
    int id;
    float weight;
    choose_experts(a, l, lane, id, weight);
    store_choice(a, t, lane, id, weight);
}

// The workgroups behind the one that makes the lists: sixteen units each, which wait for nothing.
__device__ __forceinline__ void prepare_beside(const ExpertPrepare &p, int wave, int lane) {
    const int unit = ((int)blockIdx.x - 1) * 16 + wave;
    if (unit < p.units()) experts_prepare_unit(p, unit, lane);
}
static unsigned beside(const ExpertPrepare &p) { return (unsigned)((p.units() + 15) / 16); }

// Few tokens, one workgroup: the choices of all of them and the experts' lists.
constexpr int CHOOSE_FEW = 64;
template <int L>
__global__ void __launch_bounds__(1024) choose_few_kernel(const RouterArgs a) {
    __shared__ int ids[CHOOSE_FEW * MAX_USED], hist[MAX_EXPERTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (blockIdx.x > 0) return prepare_beside(a.prepare, wave, lane);
    for (int t = wave; t < a.tokens; t += 16) {
        double l[L];
        load_logits(a, t, lane, l);
        int id;
        float weight;
        choose_experts(a, l, lane, id, weight);
        store_choice(a, t, lane, id, weight);
        if (lane < a.used) ids[t * a.used + lane] = id;
    }
    __syncthreads();
    make_lists([&](int i) { return ids[i]; }, a.tokens * a.used, a.experts, a.lists, hist);
}

__global__ void __launch_bounds__(1024) expert_lists_kernel(const int *__restrict__ ids, int slots, int experts, const ExpertLists lists, const ExpertPrepare prepare) {
    __shared__ int hist[MAX_EXPERTS];
    if (blockIdx.x > 0) return prepare_beside(prepare, __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), threadIdx.x & 63);
    make_lists([&](int i) { return ids[i]; }, slots, experts, lists, hist);
}

// A router whose weights one workgroup reads in about the time that a second launch would take: logits and choice of a token, 1024 threads.
template <int L>
__global__ void __launch_bounds__(1024) router_one_kernel(const RouterArgs a) {
    __shared__ double logits[MAX_EXPERTS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), t = (int)blockIdx.x;
    for (int e = wave; e < a.experts; e += 16) {
        const double v = router_dot(a.x + (size_t)t * a.d, a.w + (size_t)e * a.d, a.d, lane, 64);
        if (lane == 0) logits[e] = v;
    }
    __syncthreads();
    if (wave) return;
    double l[L];
#pragma unroll
    for (int i = 0; i < L; ++i) l[i] = logits[min(64 * i + lane, a.experts - 1)];
    int id;
    float weight;
    choose_experts(a, l, lane, id, weight);
    store_choice(a, t, lane, id, weight);
}

// f(the experts of a lane, as a type): what a lane does for each is most of a choice's instructions (32 tokens, 8 of 128 experts: 22 us with eight places a lane)
template <class F>
static void with_lanes(int experts, F &&f) {
    if (experts <= 64) f(std::integral_constant<int, 1>{});
    else if (experts <= 128) f(std::integral_constant<int, 2>{});
    else if (experts <= 256) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 8>{});
}
static_assert(MAX_EXPERTS <= 8 * 64, "every expert has a lane");

// One launch for logits and choice: so few weights that a token's one workgroup has read them when a second launch would start.  One / two launches, us: 8 experts of 4096 values, 1
// token 4.2 / 5.9, 64 tokens 4.7 / 6.2; 16 of 4096 6.1 / 5.9; 128 of 512 8.9 / 6.2; 64 of 2048 10.1 / 5.9.
static bool one_launch(int tokens, int experts, int d) { return (long long)experts * d <= 49152 && tokens <= 64; }

// A workgroup per logit, while all of them together read no more than 64 MiB of rows through the L2s, 136 for up to 128 tokens, where tiles are few; tiles beyond.  At 128 tokens the
// two are about level (64 experts of 2048 values 9.7 a workgroup per logit, 129 tokens in tiles 10.9; 128 of 1024 12.2, 129 tokens 10.3).  Logits and choice, tiles / a workgroup per logit, us: 64 tokens x 64 experts x 4096 values 13.4 / 9.3, 26 x 194 x 3040 13.6 / 10.5, 64 x 128 x 2048 11.6 / 10.4, 40 x 256 x 2048 12.0 / 12.1;
// 344 x 63 x 832 10.4 / 14.8, 512 x 8 x 4096 9.3 / 14.4.
static bool logit_each(int tokens, int experts, int d) { return (long long)tokens * experts * d <= (tokens <= 128 ? 17 : 8) << 20; }
static int tile_side(int tokens, int experts) { return tokens > 16 && experts > 16 ? 32 : 16; }
static int tile_splits(int tokens, int experts, int d) {
    const int side = tile_side(tokens, experts), tiles = ((tokens + side - 1) / side) * ((experts + side - 1) / side);
    return std::max(1, std::min({(side > 16 ? 512 : 1024) / tiles, 8, d / 256}));
}

size_t router_logits_bytes(int tokens, int experts, int d, bool choice_follows) {
    if (choice_follows && one_launch(tokens, experts, d)) return 0;
    return (size_t)tokens * experts * sizeof(double) * (logit_each(tokens, experts, d) ? 1 : tile_splits(tokens, experts, d));
}

void router_logits_launch(RouterArgs &a, hipStream_t s) {
    if (logit_each(a.tokens, a.experts, a.d)) {
        a.splits = 1;
        hipLaunchKernelGGL(router_logits_kernel, dim3(a.experts, a.tokens), dim3(256), 0, s, a);
    } else {
        a.splits = tile_splits(a.tokens, a.experts, a.d);
        const int side = tile_side(a.tokens, a.experts);
        const dim3 grid((a.tokens + side - 1) / side, (a.experts + side - 1) / side, a.splits);
        if (side > 16) hipLaunchKernelGGL(router_tiles_kernel<2>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(router_tiles_kernel<1>, grid, dim3(256), 0, s, a);
    }
}

void router_launch(RouterArgs a, hipStream_t s) {
    const bool lists = a.lists.list != nullptr;
    if (!lists && one_launch(a.tokens, a.experts, a.d)) {
        with_lanes(a.experts, [&](auto n) { hipLaunchKernelGGL(router_one_kernel<n()>, dim3(a.tokens), dim3(1024), 0, s, a); });
        return;
    }
    router_logits_launch(a, s);
    if (lists && a.tokens <= CHOOSE_FEW) {
        with_lanes(a.experts, [&](auto n) { hipLaunchKernelGGL(choose_few_kernel<n()>, dim3(1 + beside(a.prepare)), dim3(1024), 0, s, a); });
        return;
    }
    with_lanes(a.experts, [&](auto n) { hipLaunchKernelGGL(choose_kernel<n()>, dim3((a.tokens + 3) / 4), dim3(256), 0, s, a); });
    if (lists) expert_lists_launch(a.ids, a.tokens * a.used, a.experts, a.lists, a.prepare, s);
}

void expert_lists_launch(const int *ids, int slots, int experts, const ExpertLists &lists, const ExpertPrepare &prepare, hipStream_t s) {
    hipLaunchKernelGGL(expert_lists_kernel, dim3(1 + beside(prepare)), dim3(1024), 0, s, ids, slots, experts, lists, prepare);
}

}  // namespace jitnn
