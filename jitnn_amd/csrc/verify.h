// Verification of drafted tokens against the target's probabilities p = softmax(logits / T), from given random numbers.
//
// Row r of a sequence judges the token after it, x: kept while u0 q(x) < p(x), q the probability it was drafted with.  At the first that is
// not kept a token is drawn from max(p - q, 0), behind the last kept one from p, by the inverse of the distribution: the first index whose
// cumulative sum exceeds u1 times the total.  Such a draw is a whole number that another summation must reproduce, so weights and sums are held
// in FP64: a cumulative sum of 128256 FP32 weights is off by 1e-5 of a token's share, one of FP64 weights by 1e-14.  A number that close to a border may fall on either side of it.
//   verify_stats_kernel   chunks of a row: largest logit (lowest index among equals), sum of exp((l - largest) / T) over all but the row's draft
//   verify_rest_kernel    (with draft probabilities, more than VERIFY_FEW chunks) the refused row's sum of max(p - q, 0) per chunk
//   verify_draw_kernel    one workgroup per sequence: which tokens are kept, the chunk the draw falls in, the index in it
// Measured, us per kernel: 16 x 9 ragged rows of 128256, a draft with certainty, stats 16.3 and draw 6.5; 32 x 5 rows with draft probabilities, stats 24.9, rest 10.1, draw
// 6.4; 5 rows of 32000, 5.0 and 5.5.  The stats read 82 MB in 18.3 us where the temperature is 0 (4.5 TB/s); the FP64 weights of 20 million logits
// are the other 6.  The rest and the draw are chains of dependent reads - starts, drafts and chunks' sums, the draft's logit, the chunk - of about 1 us each.
// All rows are judged whether or not an earlier one is refused: they are read once, side by side.
#pragma once
#include "common.h"
#include "rope.h"
#include "serving.h"

namespace jitnn {

constexpr int VERIFY_THREADS = 256, VERIFY_VALUES = 16, VERIFY_CHUNK = VERIFY_THREADS * VERIFY_VALUES;

struct VerifyStat {
    double sum;  // of exp((l - largest) / T) without the row's draft (of a row: with it); T <= 0: unused
    float largest;
    int index;
};

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));  // (rows of an odd vocabulary start anywhere)

__constant__ const double VERIFY_ROOTS[32] = {  // 2^(i / 32)
    1, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};

// exp((l - largest) / T) in FP64 as 2^(n / 32) 2^(f / 32), n whole and |f| <= 1/2: a table and the Taylor series to the fifth power (the next term is 2e-15).
// With the series alone, to the twelfth power over |f| <= 1/2 of a whole octave, the weights of 160 rows of 128256 took 17 us on top of the 17 that
// reading them takes.
struct VerifyWeight {
    const double *table;  // [32]: 2^(i / 32), in LDS
    double rate;  // 32 log2(e) / T
    float largest;
    // (a barrier behind it)
    static __device__ __forceinline__ void fill(double *table) {
        if (threadIdx.x < 32) table[threadIdx.x] = VERIFY_ROOTS[threadIdx.x];
    }
    __device__ __forceinline__ VerifyWeight(const double *table, float temperature, float largest)
        : table(table), rate(temperature > 0.f ? 32. * 1.44269504088896340736 / (double)temperature : 0.), largest(largest) {}
    // of a logit at or below the largest, which is finite; NaN and -inf have none
    __device__ __forceinline__ double operator()(float l) const {
        constexpr double whole = 6755399441055744.;  // 1.5 2^52: whole numbers end in the last bit
        constexpr double c1 = 0.02166084939249829, c2 = 0.00023459619820224677, c3 = 1.6938509724371819e-06, c4 = 9.172562701824643e-09, c5 = 3.9737099845494154e-11;  // (ln 2 / 32)^k / k!
        const double y = fmax(((double)l - (double)largest) * rate, -40000.), t = y + whole, f = y - (t - whole);
        const int n = (int)(unsigned)__double2loint(t);
        const double p = fma(f, fma(f, fma(f, fma(f, fma(f, c5, c4), c3), c2), c1), 1.);
        return ldexp(p * table[n & 31], n >> 5);
    }
    // the same where the largest may be infinite: equal infinities share all the weight
    __device__ __forceinline__ double any(float l) const { return fabsf(largest) < INFINITY ? (*this)(l) : l == largest ? 1. : 0.; }
};
// Across a wave without the trip through LDS that a shuffle takes (half a dozen of them in a row were 1.5 us of the draw's 7): within rows of 16 lanes from the lanes
// 1, 2, 4 and 8 before, then the last lane of a row to the next row, then that of the first half to the second.  What no lane sends is `none`.
template <int CTRL, int ROWS>
__device__ __forceinline__ int verify_from(int v, int none) {
    return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double verify_from(double v) {
    return __hiloint2double(verify_from<CTRL, ROWS>(__double2hiint(v), 0), verify_from<CTRL, ROWS>(__double2loint(v), 0));
}
__device__ __forceinline__ double verify_lane(double v, int lane) {  // the same lane for all
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double verify_wave_scan(double v) {  // the sum up to this lane
    v += verify_from<0x111, 0xf>(v);
    v += verify_from<0x112, 0xf>(v);
    v += verify_from<0x114, 0xf>(v);
    v += verify_from<0x118, 0xf>(v);
    v += verify_from<0x142, 0xa>(v);
    v += verify_from<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double verify_wave_sum(double v) {
    v = verify_wave_scan(v);
    return verify_lane(v, 63);
}
__device__ __forceinline__ void verify_take(float v, int i, float &best, int &index) {
    if (v > best || (v == best && i < index)) {
        best = v;
        index = i;
    }
}
template <int CTRL, int ROWS>
__device__ __forceinline__ void verify_best_from(float &best, int &index) {
    const float v = __int_as_float(verify_from<CTRL, ROWS>(__float_as_int(best), __float_as_int(-INFINITY)));
    verify_take(v, verify_from<CTRL, ROWS>(index, 0x7fffffff), best, index);
}
__device__ __forceinline__ void verify_wave_best(float &best, int &index) {
    verify_best_from<0x111, 0xf>(best, index);
    verify_best_from<0x112, 0xf>(best, index);
    verify_best_from<0x114, 0xf>(best, index);
    verify_best_from<0x118, 0xf>(best, index);
    verify_best_from<0x142, 0xa>(best, index);
    verify_best_from<0x143, 0xc>(best, index);
    best = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(best), 63));
    index = __builtin_amdgcn_readlane(index, 63);
}
// VERIFY_VALUES values of a chunk per thread, four neighbours at a time; behind the row's end -inf
__device__ __forceinline__ void verify_load(const float *__restrict__ row, int c0, int vocab, float (&v)[VERIFY_VALUES]) {
#pragma unroll
    for (int u = 0; u < VERIFY_VALUES / 4; ++u) {
        const int i = c0 + 4 * (u * VERIFY_THREADS + (int)threadIdx.x);
        if (i + 4 <= vocab) {
            const f32x4_a4 x = *reinterpret_cast<const f32x4_a4 *>(row + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = x[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * u + e] = i + e < vocab ? row[i + e] : -INFINITY;
        }
    }
}

// grid (chunks, rows).  A draft is left out of its chunk's sum and joined where it is judged: what is left when it is refused is so a sum and not a difference.  (Of a token with
// all but 6e-8 of the weight, the largest share that can be refused, a difference has the error of the whole, 2e-9 of what is left, and nothing of what is
// below 1e-16.)
__global__ void __launch_bounds__(VERIFY_THREADS) verify_stats_kernel(const VerifyArgs a) {
    __shared__ float best_of[VERIFY_THREADS / 64];
    __shared__ int index_of[VERIFY_THREADS / 64];
    __shared__ double sum_of[VERIFY_THREADS / 64], table[32];
    const int r = blockIdx.y, c0 = blockIdx.x * VERIFY_CHUNK, tid = threadIdx.x, wave = tid >> 6;
    float v[VERIFY_VALUES];
    verify_load(a.logits + (size_t)r * a.logits_stride, c0, a.vocab, v);
    VerifyWeight::fill(table);
    const int s = __builtin_amdgcn_readfirstlane(batch_sequence(a.starts, a.sequences, r));
    if (s >= a.sequences || r < a.starts[0]) return;  // a row of no sequence
    const float temperature = a.temperatures[s];
    const int end = min(a.starts[s + 1], a.rows), next = a.tokens[min(r + 1, a.rows - 1)];
    const int draft = r + 1 < end ? next - c0 : -1;  // as a place of the chunk
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
        const VerifyWeight weight(table, temperature, best);
        if (draft >= 0 && draft < VERIFY_CHUNK) {
#pragma unroll
            for (int u = 0; u < VERIFY_VALUES; ++u) v[u] = draft == 4 * ((u >> 2) * VERIFY_THREADS + tid) + (u & 3) ? -INFINITY : v[u];
        }
        if (best < INFINITY) {
#pragma unroll
            for (int u = 0; u < VERIFY_VALUES; ++u) sum += weight(v[u]);
        } else {
#pragma unroll
            for (int u = 0; u < VERIFY_VALUES; ++u) sum += weight.any(v[u]);
        }
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

// A row's largest logit, its index and the sum of its weights but for its draft's, from the chunks'; one wave, every lane receives them.  first: chunk `lane`'s part of the sum.
__device__ __forceinline__ VerifyStat verify_row(const VerifyStat *__restrict__ st, int chunks, const double *table, float temperature, double &first) {
    const int lane = threadIdx.x & 63;
    VerifyStat t{0., -INFINITY, 0x7fffffff}, mine{0., -INFINITY, 0x7fffffff};
    if (lane < chunks) mine = st[lane];
    verify_take(mine.largest, mine.index, t.largest, t.index);
    for (int c = lane + 64; c < chunks; c += 64) verify_take(st[c].largest, st[c].index, t.largest, t.index);
    verify_wave_best(t.largest, t.index);
    const VerifyWeight weight(table, temperature, t.largest);
    first = mine.largest > -INFINITY ? mine.sum * weight.any(mine.largest) : 0.;
    t.sum = first;
    for (int c = lane + 64; c < chunks; c += 64)
        if (st[c].largest > -INFINITY) t.sum += st[c].sum * weight.any(st[c].largest);
    t.sum = verify_wave_sum(t.sum);
    if (t.index == 0x7fffffff) t.index = 0;  // (nothing but NaN)
    return t;
}

// Where a sequence's drafts end.  A wave to each of its rows at a time; the last one has no draft to judge but may be the one that draws.
struct VerifyEnd {
    int first, end, kept, row;  // the sequence's first row, the one behind its last, the drafts kept, the row that draws (-1: the sequence has none)
    bool refused;               // it draws from what its draft left, and is not behind the last draft
    float temperature;
    VerifyStat stat;            // of that row
    int draft;                  // the token it refused, -1 where that is none
    float number;               // its random number
    const double *parts;
};
constexpr int VERIFY_ROWS = 32;  // rows whose sums are kept
struct VerifyRow {
    VerifyStat stat;
    int draft;
    float number;
};
struct VerifyShared {
    int first_refused;
    VerifyRow row[VERIFY_ROWS + 1];
    double table[32];
};
// parts [VERIFY_ROWS + 1][64] (or nullptr): what the first 64 chunks of each row hold of its sum, its draft left out; e.parts is the drawing row's, which has refused
// its draft or has none.
template <int WAVES>
__device__ __forceinline__ VerifyEnd verify_end(const VerifyArgs &a, int s, VerifyShared &sh, double *parts) {
    VerifyEnd e;
    e.first = min(max(a.starts[s], 0), a.rows);
    e.end = min(max(a.starts[s + 1], e.first), a.rows);
    e.temperature = a.temperatures[s];
    const int count = e.end - e.first, tid = threadIdx.x, wave = tid >> 6;
    if (tid == 0) sh.first_refused = count - 1;
    VerifyWeight::fill(sh.table);
    __syncthreads();
    auto judge = [&](const int j, const int slot) {
        const int r = e.first + j;
        const bool drafted = j + 1 < count;
        const int x = drafted ? a.tokens[r + 1] : -1;
        const bool known = x >= 0 && x < a.vocab;  // (a draft that is no token is never kept)
        const float u = a.uniforms[2 * (size_t)r], number = a.uniforms[2 * (size_t)r + 1], lx = known ? a.logits[(size_t)r * a.logits_stride + x] : 0.f,
                    qx = known && a.draft_probs ? a.draft_probs[(size_t)r * a.draft_stride + x] : 1.f;
        double first;
        VerifyStat t = verify_row((const VerifyStat *)a.part + (size_t)r * a.chunks, a.chunks, sh.table, e.temperature, first);
        if (parts && slot <= VERIFY_ROWS) parts[64 * slot + (tid & 63)] = first;
        const VerifyWeight weight(sh.table, e.temperature, t.largest);
        const double wx = known ? weight.any(lx) : 0.;
        t.sum += wx;
        const bool keep = known && (e.temperature > 0.f ? t.largest > -INFINITY && (double)u * (double)qx < wx / t.sum : x == t.index);
        if ((tid & 63) == 0) {
            if (slot <= VERIFY_ROWS) sh.row[slot] = VerifyRow{t, known ? x : -1, number};
            if (drafted && !keep) atomicMin(&sh.first_refused, j);
        }
    };
    for (int j = wave; j < count; j += WAVES) judge(j, j < VERIFY_ROWS ? j : VERIFY_ROWS + 1);
    __syncthreads();
    e.kept = max(sh.first_refused, 0);
    e.row = count > 0 ? e.first + e.kept : -1;
    e.refused = e.kept < count - 1;
    if (count <= 0) return e;
    if (e.kept >= VERIFY_ROWS) {
        if (wave == 0) judge(e.kept, VERIFY_ROWS);
        __syncthreads();
    }
    const int slot = min(e.kept, VERIFY_ROWS);
    const VerifyRow &at = sh.row[slot];
    e.parts = parts ? parts + 64 * slot : nullptr;
    e.stat = at.stat;
    e.draft = at.draft;
    e.number = at.number;
    return e;
}

// grid (chunks, sequences)
__global__ void __launch_bounds__(VERIFY_THREADS) verify_rest_kernel(const VerifyArgs a) {
    __shared__ VerifyShared sh;
    __shared__ double sum_of[VERIFY_THREADS / 64];
    const int s = blockIdx.y, c0 = blockIdx.x * VERIFY_CHUNK, tid = threadIdx.x;
    const VerifyEnd e = verify_end<VERIFY_THREADS / 64>(a, s, sh, nullptr);
    if (e.row < 0 || !e.refused || !(e.temperature > 0.f)) return;
    float l[VERIFY_VALUES], q[VERIFY_VALUES];
    verify_load(a.logits + (size_t)e.row * a.logits_stride, c0, a.vocab, l);
    verify_load(a.draft_probs + (size_t)e.row * a.draft_stride, c0, a.vocab, q);
    const VerifyWeight weight(sh.table, e.temperature, e.stat.largest);
    const double share = 1. / e.stat.sum;
    double sum = 0.;
    auto add = [&](double w, float q) {
        const double rest = fma(w, share, -(double)q);
        sum += rest > 0. && q > -INFINITY ? rest : 0.;  // (behind the row's end q is -inf)
    };
    if (fabsf(e.stat.largest) < INFINITY) {
#pragma unroll
        for (int u = 0; u < VERIFY_VALUES; ++u) add(weight(l[u]), q[u]);
    } else {
#pragma unroll
        for (int u = 0; u < VERIFY_VALUES; ++u) add(weight.any(l[u]), q[u]);
    }
    sum = verify_wave_sum(sum);
    if ((tid & 63) == 0) sum_of[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) ((double *)((VerifyStat *)a.part + (size_t)a.rows * a.chunks))[(size_t)s * a.chunks + blockIdx.x] = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
}

// grid (sequences).  Of few chunks it sums what the refused draft left by itself, 1 us each: all three kernels over 4 x 5 rows took 23 us at four
// chunks, 15 us so; at five 18 us.
constexpr int VERIFY_FEW = 4;
constexpr int VERIFY_DRAW_THREADS = VERIFY_CHUNK / 4;  // four neighbours each, in one load (eight in eight by half as many threads took 3 us longer)
// what the draw of a row leaves to each of four neighbours: p, without a draft's q or the draft x
__device__ __forceinline__ void verify_left(const VerifyArgs &a, const VerifyEnd &e, const VerifyWeight &weight, const double share, const float *q, const int x, const int i0,
                                            double (&w)[4]) {
    const float *row = a.logits + (size_t)e.row * a.logits_stride;
    f32x4_a4 l, d = {0.f, 0.f, 0.f, 0.f};
    if (i0 + 4 <= a.vocab) {
        l = *reinterpret_cast<const f32x4_a4 *>(row + i0);
        if (q) d = *reinterpret_cast<const f32x4_a4 *>(q + i0);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool there = i0 + u < a.vocab;
            l[u] = there ? row[i0 + u] : -INFINITY;
            if (q) d[u] = there ? q[i0 + u] : INFINITY;
        }
    }
    if (fabsf(e.stat.largest) < INFINITY) {
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = weight(l[u]);
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = weight.any(l[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = i0 + u != x ? fmax(fma(w[u], share, -(double)d[u]), 0.) : 0.;
}
__global__ void __launch_bounds__(VERIFY_DRAW_THREADS) verify_draw_kernel(const VerifyArgs a) {
    constexpr int WAVES = VERIFY_DRAW_THREADS / 64;
    __shared__ VerifyShared sh;
    __shared__ int chosen_chunk, first_at[WAVES], last_at[WAVES];
    __shared__ double left, sum_of[WAVES], rest_of[VERIFY_FEW][WAVES], parts[(VERIFY_ROWS + 1) * 64];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const double *rest = (const double *)((const VerifyStat *)a.part + (size_t)a.rows * a.chunks) + (size_t)s * a.chunks;
    // (asked for before it is known whether it is needed; without a refused draft nobody has written it)
    const double first_rest = a.draft_probs && a.chunks > VERIFY_FEW && lane < a.chunks ? rest[lane] : 0.;
    const VerifyEnd e = verify_end<WAVES>(a, s, sh, parts);
    if (tid == 0) a.accepted[s] = e.row < 0 ? 0 : e.kept;
    if (e.row < 0) return;
    for (int r = e.first + tid; r < e.end; r += VERIFY_DRAW_THREADS)
        if (r != e.row) a.out[r] = r < e.row ? a.tokens[r + 1] : -1;
    if (!(e.temperature > 0.f) || !(e.stat.largest > -INFINITY)) {
        if (tid == 0) a.out[e.row] = e.stat.index;
        return;
    }
    const VerifyWeight weight(sh.table, e.temperature, e.stat.largest);
    const double share = 1. / e.stat.sum;
    const int x = e.refused && !a.draft_probs ? e.draft : -1;  // drafted with probability 1: the rest is p without it
    const float *q = e.refused && a.draft_probs ? a.draft_probs + (size_t)e.row * a.draft_stride : nullptr;
    if (q && a.chunks <= VERIFY_FEW) {
#pragma unroll 1
        for (int c = 0; c < a.chunks; ++c) {
            double w[4];
            verify_left(a, e, weight, share, q, -1, c * VERIFY_CHUNK + 4 * tid, w);
            const double sum = verify_wave_sum((w[0] + w[1]) + (w[2] + w[3]));
            if (lane == 0) rest_of[c][wave] = sum;
        }
        __syncthreads();
    }
    // ---- the chunk: one wave, 64 chunks at a time
    if (wave == 0) {
        const VerifyStat *st = (const VerifyStat *)a.part + (size_t)e.row * a.chunks;
        auto weight_of = [&](int c) {
            if (c >= a.chunks) return 0.;
            if (q && a.chunks <= VERIFY_FEW) {
                double w = 0.;
                for (int v = 0; v < WAVES; ++v) w += rest_of[c][v];
                return w;
            }
            if (q) return c < 64 ? first_rest : rest[c];
            return share * (c < 64 ? e.parts[c] : st[c].largest > -INFINITY ? st[c].sum * weight.any(st[c].largest) : 0.);
        };
        const double first = weight_of(lane);  // (a vocabulary of 262144 has 64 chunks)
        double total = verify_wave_sum(first);
        for (int c0 = 64; c0 < a.chunks; c0 += 64) total += verify_wave_sum(weight_of(c0 + lane));
        const double target = (double)e.number * total;
        double before = 0., before_chunk = 0.;
        int chunk = -1, last = 0;
        for (int c0 = 0; c0 < a.chunks && chunk < 0; c0 += 64) {
            const double w = c0 == 0 ? first : weight_of(c0 + lane), upto = verify_wave_scan(w);
            const unsigned long long past = __ballot(before + upto > target), some = __ballot(w > 0.);
            if (past) {
                const int at = __ffsll((long long)past) - 1;
                chunk = c0 + at;
                before_chunk = before + (verify_lane(upto, at) - verify_lane(w, at));
            } else if (some) {
                last = c0 + 63 - __clzll((long long)some);
            }
            before += verify_lane(upto, 63);
        }
        if (lane == 0) {
            chosen_chunk = chunk >= 0 ? chunk : last;
            left = chunk >= 0 ? target - before_chunk : INFINITY;
        }
    }
    __syncthreads();
    // ---- the index in it
    const int i0 = chosen_chunk * VERIFY_CHUNK + 4 * tid;
    double w[4];
    verify_left(a, e, weight, share, q, x, i0, w);
    const double sum = (w[0] + w[1]) + (w[2] + w[3]);
    const double upto = verify_wave_scan(sum);
    if (lane == 63) sum_of[wave] = upto;
    __syncthreads();
    double c = upto - sum;
    for (int v = 0; v < wave; ++v) c += sum_of[v];
    // the first index whose cumulative sum is past what is left; where rounding or a number of 1 leaves none, the last with any weight
    int mine = -1, last = -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        c += w[u];
        if (mine < 0 && w[u] > 0. && c > left) mine = i0 + u;
        if (w[u] > 0.) last = i0 + u;
    }
    const unsigned long long hit = __ballot(mine >= 0), any = __ballot(last >= 0);
    const int hit_at = hit ? __builtin_amdgcn_readlane(mine, __ffsll((long long)hit) - 1) : -1, any_at = any ? __builtin_amdgcn_readlane(last, 63 - __clzll((long long)any)) : -1;
    if (lane == 0) {
        first_at[wave] = hit_at;
        last_at[wave] = any_at;
    }
    __syncthreads();
    if (wave == 0) {
        const int f = lane < WAVES ? first_at[lane] : -1, l = lane < WAVES ? last_at[lane] : -1;
        const unsigned long long found = __ballot(f >= 0), some = __ballot(l >= 0);
        const int at = found ? __builtin_amdgcn_readlane(f, __ffsll((long long)found) - 1) : some ? __builtin_amdgcn_readlane(l, 63 - __clzll((long long)some)) : e.stat.index;
        if (lane == 0) a.out[e.row] = at;
    }
}

}  // namespace jitnn
