// Verification of drafted tokens against the target's probabilities p = softmax(logits / T), from given random numbers.
//
// Row r of a sequence judges the token after it, x: kept while u0 q(x) < p(x), q the probability it was drafted with.  At the first that is
// not kept a token is drawn from max(p - q, 0), behind the last kept one from p, by the inverse of the distribution: the first index whose
// cumulative sum exceeds u1 times the total.  Such a draw is a whole number that another summation must reproduce, so weights and sums are held
// in FP64: a cumulative sum of 128256 FP32 weights is off by 1e-5 of a token's share, one of FP64 weights by 1e-14.
//   verify_stats_kernel   chunks of a row: largest logit (lowest index among equals), sum of exp((l - largest) / T)
//   verify_rest_kernel    (with draft probabilities) the refused row's sum of max(p - q, 0) per chunk
//   verify_draw_kernel    one workgroup per sequence: which tokens are kept, the chunk the draw falls in, the index in it
// All rows are judged whether or not an earlier one is refused: they are read once, side by side.
#pragma once
#include "common.h"
#include "rope.h"
#include "serving.h"

namespace jitnn {

constexpr int VERIFY_THREADS = 256, VERIFY_VALUES = 32, VERIFY_CHUNK = VERIFY_THREADS * VERIFY_VALUES;

struct VerifyStat {
    double sum;  // of exp((l - largest) / T); T <= 0: unused
    float largest;
    int index;
};

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));  // (rows of an odd vocabulary start anywhere)

// 2^y for y <= 0: the Taylor series of exp(f ln 2), |f| <= 1/2, to the twelfth power (the next term is 2e-16)
__device__ __forceinline__ double verify_exp2(double y) {
    y = fmax(y, -1100.);  // (-inf too)
    const double n = rint(y), x = (y - n) * 0.69314718055994530942;
    double p = 1. / 479001600.;
    p = fma(p, x, 1. / 39916800.);
    p = fma(p, x, 1. / 3628800.);
    p = fma(p, x, 1. / 362880.);
    p = fma(p, x, 1. / 40320.);
    p = fma(p, x, 1. / 5040.);
    p = fma(p, x, 1. / 720.);
    p = fma(p, x, 1. / 120.);
    p = fma(p, x, 1. / 24.);
    p = fma(p, x, 1. / 6.);
    p = fma(p, x, .5);
    p = fma(p, x, 1.);
    p = fma(p, x, 1.);
    return ldexp(p, (int)n);
}
// exp((l - largest) / T), rate = log2(e) / T; NaN has no weight, equal infinities have 1
__device__ __forceinline__ double verify_weight(float l, float largest, double rate) {
    return l == largest ? 1. : l < largest ? verify_exp2(((double)l - (double)largest) * rate) : 0.;
}
__device__ __forceinline__ double verify_wave_sum(double v) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ void verify_take(float v, int i, float &best, int &index) {
    if (v > best || (v == best && i < index)) {
        best = v;
        index = i;
    }
}
__device__ __forceinline__ void verify_wave_best(float &best, int &index) {
    for (int off = 32; off > 0; off >>= 1) {
        const float v = __shfl_xor(best, off);
        const int i = __shfl_xor(index, off);
        verify_take(v, i, best, index);
    }
}
__device__ __forceinline__ double verify_rate(float temperature) { return temperature > 0.f ? 1.44269504088896340736 / (double)temperature : 0.; }

// grid (chunks, rows)
__global__ void __launch_bounds__(VERIFY_THREADS) verify_stats_kernel(const VerifyArgs a) {
    __shared__ float best_of[VERIFY_THREADS / 64];
    __shared__ int index_of[VERIFY_THREADS / 64];
    __shared__ double sum_of[VERIFY_THREADS / 64];
    const int r = blockIdx.y, c0 = blockIdx.x * VERIFY_CHUNK, tid = threadIdx.x, wave = tid >> 6;
    const float *row = a.logits + (size_t)r * a.logits_stride;
    float v[VERIFY_VALUES];
#pragma unroll
    for (int u = 0; u < VERIFY_VALUES / 4; ++u) {
        const int i = c0 + 4 * (u * VERIFY_THREADS + tid);
        if (i + 4 <= a.vocab) {
            const f32x4_a4 x = *reinterpret_cast<const f32x4_a4 *>(row + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = x[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = i + e < a.vocab ? row[i + e] : -INFINITY;
        }
    }
    const int s = batch_sequence(a.starts, a.sequences, r);
    if (s >= a.sequences || r < a.starts[0]) return;  // a row of no sequence
    const float temperature = a.temperatures[s];
    float best = -INFINITY;
    int index = 0x7fffffff;
#pragma unroll
    for (int u = 0; u < VERIFY_VALUES; ++u) {
        const int i = c0 + 4 * ((u >> 2) * VERIFY_THREADS + tid) + (u & 3);
        if (i < a.vocab) verify_take(v[u], i, best, index);
    }
    verify_wave_best(best, index);
    if ((tid & 63) == 0) {
        best_of[wave] = best;
        index_of[wave] = index;
    }
    __syncthreads();
    best = best_of[0];
    index = index_of[0];
#pragma unroll
    for (int w = 1; w < VERIFY_THREADS / 64; ++w) verify_take(best_of[w], index_of[w], best, index);
    double sum = 0.;
    if (temperature > 0.f && best > -INFINITY) {
        const double rate = verify_rate(temperature);
#pragma unroll 4
        for (int u = 0; u < VERIFY_VALUES; ++u) sum += verify_weight(v[u], best, rate);
    }
    sum = verify_wave_sum(sum);
    if ((tid & 63) == 0) sum_of[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        VerifyStat *st = (VerifyStat *)a.part + (size_t)r * a.chunks + blockIdx.x;
        st->sum = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
        st->largest = best;
        st->index = index;
    }
}

// A row's largest logit, its index and the sum of its weights, from the chunks'; one wave, every lane receives them.
__device__ __forceinline__ VerifyStat verify_row(const VerifyStat *__restrict__ st, int chunks, double rate) {
    const int lane = threadIdx.x & 63;
    VerifyStat t{0., -INFINITY, 0x7fffffff};
    for (int c = lane; c < chunks; c += 64) verify_take(st[c].largest, st[c].index, t.largest, t.index);
    verify_wave_best(t.largest, t.index);
    for (int c = lane; c < chunks; c += 64)
        if (st[c].largest > -INFINITY) t.sum += st[c].sum * verify_weight(st[c].largest, t.largest, rate);
    t.sum = verify_wave_sum(t.sum);
    if (t.index == 0x7fffffff) t.index = 0;  // (nothing but -inf and NaN)
    return t;
}

// Where a sequence's drafts end.  A workgroup of WAVES waves, a row to each of them at a time.
struct VerifyEnd {
    int first, kept, row;  // the sequence's first row, the drafts kept, the row that draws
    bool refused;          // ... from what its draft left, and not behind the last draft
    float temperature;
    VerifyStat stat;       // of that row
};
template <int WAVES>
__device__ __forceinline__ VerifyEnd verify_end(const VerifyArgs &a, int s, int *first_refused, VerifyStat *stat) {
    const int begin = min(max(a.starts[s], 0), a.rows), end = min(max(a.starts[s + 1], begin), a.rows), tid = threadIdx.x, wave = tid >> 6;
    const float temperature = a.temperatures[s];
    const double rate = verify_rate(temperature);
    if (tid == 0) *first_refused = end - begin - 1;
    __syncthreads();
    for (int j = wave; j < end - begin - 1; j += WAVES) {
        const int r = begin + j, x = a.tokens[r + 1];
        const bool known = x >= 0 && x < a.vocab;  // (a draft that is no token is never kept)
        const float lx = known ? a.logits[(size_t)r * a.logits_stride + x] : 0.f, qx = known && a.draft_probs ? a.draft_probs[(size_t)r * a.draft_stride + x] : 1.f,
                    u = a.uniforms[2 * (size_t)r];
        const VerifyStat t = verify_row((const VerifyStat *)a.part + (size_t)r * a.chunks, a.chunks, rate);
        const bool keep = known && (temperature > 0.f ? t.largest > -INFINITY && (double)u * (double)qx < verify_weight(lx, t.largest, rate) / t.sum : x == t.index);
        if (!keep && (tid & 63) == 0) atomicMin(first_refused, j);
    }
    __syncthreads();
    VerifyEnd e;
    e.first = begin;
    e.kept = max(*first_refused, 0);
    e.row = begin + e.kept;
    e.refused = e.kept < end - begin - 1;
    e.temperature = temperature;
    if (wave == 0 && end > begin) {
        const VerifyStat t = verify_row((const VerifyStat *)a.part + (size_t)e.row * a.chunks, a.chunks, rate);
        if (tid == 0) *stat = t;
    }
    __syncthreads();
    if (end == begin) e.row = -1;
    else e.stat = *stat;
    return e;
}

// The weight of index i in the row that draws, over the row's sum.
__device__ __forceinline__ double verify_share(float l, float q, const VerifyEnd &e, double rate) {
    return fmax(verify_weight(l, e.stat.largest, rate) / e.stat.sum - (double)q, 0.);
}

// grid (chunks, sequences)
__global__ void __launch_bounds__(VERIFY_THREADS) verify_rest_kernel(const VerifyArgs a) {
    __shared__ int first_refused;
    __shared__ VerifyStat stat;
    __shared__ double sum_of[VERIFY_THREADS / 64];
    const int s = blockIdx.y, c0 = blockIdx.x * VERIFY_CHUNK, tid = threadIdx.x;
    const VerifyEnd e = verify_end<VERIFY_THREADS / 64>(a, s, &first_refused, &stat);
    if (e.row < 0 || !e.refused || !(e.temperature > 0.f)) return;
    const double rate = verify_rate(e.temperature);
    const float *row = a.logits + (size_t)e.row * a.logits_stride, *q = a.draft_probs + (size_t)e.row * a.draft_stride;
    float l[VERIFY_VALUES], d[VERIFY_VALUES];
#pragma unroll
    for (int u = 0; u < VERIFY_VALUES; ++u) {
        const int i = min(c0 + u * VERIFY_THREADS + tid, a.vocab - 1);
        l[u] = row[i];
        d[u] = q[i];
    }
    double sum = 0.;
#pragma unroll 4
    for (int u = 0; u < VERIFY_VALUES; ++u)
        if (c0 + u * VERIFY_THREADS + tid < a.vocab) sum += verify_share(l[u], d[u], e, rate);
    sum = verify_wave_sum(sum);
    if ((tid & 63) == 0) sum_of[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) ((double *)((VerifyStat *)a.part + (size_t)a.rows * a.chunks))[(size_t)s * a.chunks + blockIdx.x] = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
}

// grid (sequences)
constexpr int VERIFY_DRAW_THREADS = 1024, VERIFY_DRAW_VALUES = VERIFY_CHUNK / VERIFY_DRAW_THREADS;
__global__ void __launch_bounds__(VERIFY_DRAW_THREADS) verify_draw_kernel(const VerifyArgs a) {
    constexpr int WAVES = VERIFY_DRAW_THREADS / 64;
    __shared__ int first_refused, chosen_chunk;
    __shared__ VerifyStat stat;
    __shared__ double left, sum_of[WAVES];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const VerifyEnd e = verify_end<WAVES>(a, s, &first_refused, &stat);
    if (tid == 0) a.accepted[s] = e.row < 0 ? 0 : e.kept;
    if (e.row < 0) return;
    const int end = min(max(a.starts[s + 1], e.first), a.rows);
    for (int r = e.first + tid; r < end; r += VERIFY_DRAW_THREADS)
        if (r != e.row) a.out[r] = r < e.row ? a.tokens[r + 1] : -1;
    const double rate = verify_rate(e.temperature);
    if (!(e.temperature > 0.f) || !(e.stat.largest > -INFINITY)) {
        if (tid == 0) a.out[e.row] = e.stat.index;
        return;
    }
    const bool certain = e.refused && !a.draft_probs;  // drafted with probability 1: the rest is p without it
    const int x = certain ? a.tokens[e.row + 1] : -1;
    const float *row = a.logits + (size_t)e.row * a.logits_stride, *q = e.refused && a.draft_probs ? a.draft_probs + (size_t)e.row * a.draft_stride : nullptr;
    // ---- the chunk: one wave, 64 chunks at a time
    if (wave == 0) {
        const VerifyStat *st = (const VerifyStat *)a.part + (size_t)e.row * a.chunks;
        const double *rest = (const double *)((const VerifyStat *)a.part + (size_t)a.rows * a.chunks) + (size_t)s * a.chunks;
        auto weight_of = [&](int c) {
            if (c >= a.chunks) return 0.;
            if (q) return rest[c];
            double w = st[c].largest > -INFINITY ? st[c].sum * verify_weight(st[c].largest, e.stat.largest, rate) : 0.;
            if (x >= 0 && x < a.vocab && x / VERIFY_CHUNK == c) w = fmax(w - verify_weight(row[x], e.stat.largest, rate), 0.);
            return w / e.stat.sum;
        };
        double total = 0.;
        for (int c0 = 0; c0 < a.chunks; c0 += 64) total += verify_wave_sum(weight_of(c0 + lane));
        const double target = (double)a.uniforms[2 * (size_t)e.row + 1] * total;
        double before = 0., before_chunk = 0.;
        int chunk = -1, last = 0;
        for (int c0 = 0; c0 < a.chunks && chunk < 0; c0 += 64) {
            const double w = weight_of(c0 + lane);
            double upto = w;
            for (int off = 1; off < 64; off <<= 1) {
                const double o = __shfl_up(upto, off);
                if (lane >= off) upto += o;
            }
            const unsigned long long past = __ballot(before + upto > target), some = __ballot(w > 0.);
            if (past) {
                const int at = __ffsll((long long)past) - 1;
                chunk = c0 + at;
                before_chunk = before + (__shfl(upto, at) - __shfl(w, at));
            } else if (some) {
                last = c0 + 63 - __clzll((long long)some);
            }
            before += __shfl(upto, 63);
        }
        if (lane == 0) {
            chosen_chunk = chunk >= 0 ? chunk : last;
            left = chunk >= 0 ? target - before_chunk : INFINITY;
        }
    }
    __syncthreads();
    // ---- the index in it: every thread eight neighbours
    const int i0 = chosen_chunk * VERIFY_CHUNK + tid * VERIFY_DRAW_VALUES;
    double w[VERIFY_DRAW_VALUES], sum = 0.;
#pragma unroll
    for (int u = 0; u < VERIFY_DRAW_VALUES; ++u) {
        const int i = min(i0 + u, a.vocab - 1);
        const float l = row[i], d = q ? q[i] : 0.f;
        w[u] = i0 + u < a.vocab && i0 + u != x ? verify_share(l, d, e, rate) : 0.;
        sum += w[u];
    }
    double upto = sum;
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(upto, off);
        if (lane >= off) upto += o;
    }
    if (lane == 63) sum_of[wave] = upto;
    __syncthreads();
    double before = 0.;
    for (int v = 0; v < wave; ++v) before += sum_of[v];
    before += upto - sum;
    // the first index whose cumulative sum is past what is left; where rounding or a number of 1 leaves none, the last with any weight
    int mine = -1;
    double c = before;
#pragma unroll
    for (int u = 0; u < VERIFY_DRAW_VALUES; ++u) {
        c += w[u];
        if (mine < 0 && w[u] > 0. && c > left) mine = i0 + u;
    }
    __shared__ int first_at[WAVES], last_at[WAVES];
    int last = -1;
#pragma unroll
    for (int u = 0; u < VERIFY_DRAW_VALUES; ++u)
        if (w[u] > 0.) last = i0 + u;
    const unsigned long long hit = __ballot(mine >= 0), any = __ballot(last >= 0);
    const int hit_at = hit ? __shfl(mine, __ffsll((long long)hit) - 1) : -1, any_at = any ? __shfl(last, 63 - __clzll((long long)any)) : -1;
    if (lane == 0) {
        first_at[wave] = hit_at;
        last_at[wave] = any_at;
    }
    __syncthreads();
    if (tid == 0) {
        int found = -1, end_at = -1;
        for (int v = 0; v < WAVES; ++v) {
            if (found < 0 && first_at[v] >= 0) found = first_at[v];
            if (last_at[v] >= 0) end_at = last_at[v];
        }
        a.out[e.row] = found >= 0 ? found : end_at >= 0 ? end_at : e.stat.index;
    }
}

}  // namespace jitnn
