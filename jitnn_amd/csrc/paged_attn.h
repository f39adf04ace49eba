// Attention of a batch over a paged cache: token t of sequence s, at position p, attends to the positions 0 .. p of s, whose keys and values lie
// in pages that a table names.  The leading pages may be everybody's: the workgroups that take their positions take the rows - (token, query
// head) pairs of one key/value head - of the whole batch, so that they are read once and not once per sequence; the other positions go
// to workgroups of their sequence.  Every workgroup leaves, for its span of keys, what its weights count in, their sum and the weighted sum
// of the values, and paged_merge_kernel joins a row's spans; where there is one span in all, its workgroups write the outputs.
//
// The products run on the matrix cores, transposed, S^T = K Q^T and O^T = V^T P^T, and nothing but the last sums goes through LDS:
//   * lane n + 16 g holds for the scores key n of a tile of 16 (16 bytes of its row per load), receives the scores of ROW n against the keys
//     4 g + i, and those, as weights, are its slots of the P operand: its running maximum and sum are one row's.
//   * of the values the lane loads, for the very keys 4 g + i, the D / 16 neighbours from D / 16 n on: all a row of V, so that the loads of
//     16 lanes are one row in one piece, and the A operand of V^T needs no more than the lane's own registers - its tile e takes the e-th value
//     of each key, row n of that tile being value D / 16 n + e.
//   A wave so streams keys and values from memory at its own pace, without a barrier (pa_stream): for few rows, which memory bounds.  8 sequences of up to 2000
//   positions, 32 heads of 128 in FP16: 148 MB in 34.6 us, one launch (4.3 TB/s).  Where the rows fill several waves, each wave's own stream of the same keys
//   is what bounds: there the waves share them through LDS (pa_wide).  64 sequences behind 16384 shared positions, 32 heads of 128 over 8: 126 us with streams
//   alone, 59 so, and the merge 7.  34 GFLOP, each product in two parts: 0.58 PFLOP/s over those 59 us, their start and the sequences' own positions among them; behind 131072 it is
//   274 us with the merge, 1.13 PFLOP/s over the further positions.
// FP16 pages: keys and values are operands as they are; queries (scaled so that a row's largest is near 2^13) and weights (the largest 2^11 to 2^16) go in two FP16
// parts: each within 2^-22 of itself, or 2^-36 of the largest where that is more.  The result is as good as in FP32 but for keys of less weight than 2^-14, which may be off by 2^-36 each
// (one part of 11 bits would leave 2^-12 of every weight).  FP32 pages: the FP32 matrix instruction, an eighth of the rate; 24 sequences of up to 5 rows behind 992 shared positions, 35 us and the merge 6.7.
// Sums, maxima and outputs are FP32.
//
// What a row does not see: its scores are masked; values past the last key that any row of the tile sees are cleared, and of those that only some see
// the ones that are not finite, whose rows become NaN (badkey): nothing behind a token reaches it.  The same mark makes NaN of rows whose positions
// lie on a page that the cache does not have.
#pragma once
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.h"
#include "serving.h"

namespace jitnn {

constexpr int PA_THREADS = 256, PA_WAVES = 4;
// A row's largest weight is 2^11.5 to 2^15.5 (and 1/4 in the exponent): inside FP16, whose steps of 2^-24 at the lower end are then 2^-35 of it at most.  (At 2^6 to 2^14 they were 2^-30, and
// 16384 keys of 2^-31 each off by a quarter of their sum, 2.6e-6.)
constexpr float PA_WEIGHT = 11.5f, PA_LAG = 4.f;

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x4v_a4 __attribute__((ext_vector_type(4), aligned(4)));  // (rows of y start anywhere)

template <class T, int D>
struct PaTile;
template <int D>
struct PaTile<_Float16, D> {
    static constexpr int KEYS = 32, TILES = 2, E = D / 16;  // keys of a step, tiles of 16, neighbouring values of a lane
    f16x8 k[TILES][D / 32];
    _Float16 v[TILES][4][E] __attribute__((aligned(16)));
};
template <int D>
struct PaTile<float, D> {
    static constexpr int KEYS = 16, TILES = 1, E = D / 16;
    f32x4v k[D / 16];
    float v[1][4][E] __attribute__((aligned(16)));
};

// maximum / sum over the lanes 16, 32 and 48 away
__device__ __forceinline__ float pa_max4(float v) {
    float a = v, b = v;  // (the maxima in assembly too: of what comes out of one, the compiler first makes both operands quiet)
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1\n\tv_max_f32 %0, %0, %1" : "+v"(a), "+v"(b));
    b = a;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1\n\tv_max_f32 %0, %0, %1" : "+v"(a), "+v"(b));
    return a;
}
__device__ __forceinline__ float pa_sum4(float v) {
    float a = v, b = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    a = b = a + b;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}

__device__ __forceinline__ bool pa_finite(_Float16 x) { return (__builtin_bit_cast(unsigned short, x) & 0x7c00) != 0x7c00; }
__device__ __forceinline__ bool pa_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// n / by and what is left of it, m = reciprocal(by): less than one below 2^32 / by, so that the product is at most one too small.
__device__ __forceinline__ unsigned pa_div(unsigned n, unsigned by, unsigned m, unsigned &rest) {
    unsigned d = __umulhi(n, m);
    rest = n - d * by;
    if (rest >= by) {
        ++d;
        rest -= by;
    }
    return d;
}
__device__ __forceinline__ int pa_div(int n, int by, unsigned m) {  // n >= 0
    unsigned rest;
    return (int)pa_div((unsigned)n, (unsigned)by, m, rest);
}

// The sequence of token t, its length and the token behind its last; one wave (or every wave) with the same t.  Lengths come with the starts, in one
// round trip for each 64 sequences.
struct RowPlace {
    int sequence, len, end;
};
__device__ __forceinline__ RowPlace row_place(const int *__restrict__ starts, const int *__restrict__ lens, int sequences, int t) {
    const int lane = threadIdx.x & 63;
    RowPlace p{0, 0, 0};
    for (int i0 = 0; i0 < sequences; i0 += 64) {
        const int i = min(i0 + lane, sequences - 1), end = starts[i + 1], len = lens[i];
        const int below = __popcll(__ballot(i0 + lane < sequences && end <= t));
        p.sequence += below;
        if (below < 64) {
            p.len = __builtin_amdgcn_readlane(len, below);
            p.end = __builtin_amdgcn_readlane(end, below);
            break;
        }
    }
    return p;
}

// What a wave holds of its rows, R tiles of 16.
template <class T, int D, int R>
struct PaRows {
    static constexpr int E = D / 16;
    int rows, row0, t0;    // rows of the part, the wave's first, the part's first token
    int group, token0, rem0;  // query heads per key/value head; the wave's first row as a token behind t0 and a head of the group
    float per_group;
    int begins, ends, lens, base;  // sequence base + lane: its first token, the one behind its last, its length
    int lim[R];            // the last position of the span that row n sees
    bool over[R];          // ... of a sequence longer than it may be
    int first, last;       // the least and the largest lim
    int badkey;            // rows that see this position are NaN
    f16x8 qh[R][sizeof(T) == 2 ? D / 32 : 1], ql[R][sizeof(T) == 2 ? D / 32 : 1];
    f32x4v qf[R][D / 16];  // (FP16: until they are operands)
    float qs[R];
    f32x4v o[R][E];
    float l[R];
    float less[R];       // a weight is 2^(score + less): PA_WEIGHT minus about the largest score so far, FLT_MAX before the first
    float minus;         // -1, which the compiler does not know: it would take the FP16 part off the weight in two instructions and not in one
    u32x4 ph[R], pl[R];  // weights (FP16): slot 4 t + i
    float pf[R][4];      // (FP32)

    // In steps, so that what they wait for is asked for together: begin (false: the workgroup has nothing to do), fetch (queries), find (the rows'
    // positions), take (the queries as operands).
    __device__ __forceinline__ bool begin(const AttnArgs &a, const bool ahead, const int seq, const int row0_of_wave, const int row0_of_block, const int key0) {
        group = a.group;
        per_group = a.per_group;
        // (the first 64 sequences' ends and lengths, a lane each, for find)
        base = 0;
        if (ahead) sequences_at(a);
        t0 = max(a.starts[ahead ? 0 : seq], 0);
        rows = max(min(a.starts[ahead ? a.sequences : seq + 1], a.tokens) - t0, 0) * group;
        row0 = row0_of_wave;
        // (a span that no row of the sequence reaches; where there is one span in all, its rows are still to be written)
        return row0_of_block < rows && (ahead || key0 == 0 || a.lens[seq] > key0);
    }
    __device__ __forceinline__ void sequences_at(const AttnArgs &a) {
        const int i = min(base + (int)(threadIdx.x & 63), a.sequences - 1);
        begins = a.starts[i];
        ends = a.starts[i + 1];
        lens = a.lens[i];
    }
    // the row behind the wave's first by `in` < 32 as a token behind t0 and a head of the group: whole numbers below 2^17, for which the FP32 quotient of a
    // number and a half has the right whole part
    __device__ __forceinline__ int2 place(const int in) const {
        const int x = rem0 + in, q = (int)(((float)x + 0.5f) * per_group);
        return make_int2(token0 + q, x - q * group);
    }
    // queries: 8 g + j of each 32 values (FP16), 4 g + j of each 16 (FP32) of row n
    __device__ __forceinline__ void fetch(const AttnArgs &a, const int kvh) {
        const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
        token0 = __builtin_amdgcn_readfirstlane(pa_div(row0, group, a.by_group));
        rem0 = row0 - token0 * group;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int2 at = place(max(min(16 * r + n, rows - 1 - row0), 0));  // (a wave without rows reads behind them: of a token that exists)
            const float *q = a.q + (size_t)min(t0 + at.x, a.tokens - 1) * a.q_stride + (size_t)(kvh * group + at.y) * D;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) qf[r][s] = *reinterpret_cast<const f32x4v_a4 *>(q + (sizeof(T) == 2 ? 32 * (s >> 1) + 8 * g + 4 * (s & 1) : 16 * s + 4 * g));
        }
    }
    // The positions of the rows' tokens.  Of a sequence they follow one another.  Of the whole batch: where no sequence ends inside the span - a vote over
    // all of them -, all rows see all of it; otherwise token by token, in scalar registers: a token's sequence is how many ends are at or below it.
    __device__ __forceinline__ void find(const AttnArgs &a, const bool ahead, const int seq, const int key1) {
        const int n = threadIdx.x & 15, lane = threadIdx.x & 63;
        last = -1;
        first = badkey = 0x7fffffff;
        int token[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            lim[r] = -1;
            over[r] = false;
            token[r] = row0 + 16 * r + n < rows ? place(16 * r + n).x : -1;
        }
        const int count = min(16 * R, rows - row0);  // of the wave's rows
        if (count <= 0) return;
        const int end_token = place(count - 1).x;
        if (!ahead) {
            const int len = a.lens[seq], behind = len - a.starts[seq + 1] + t0;
            const bool long_one = len > a.max_len;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                over[r] = long_one && token[r] >= 0;
                if (!long_one && token[r] >= 0) lim[r] = min(behind + token[r], key1 - 1);
            }
            if (!long_one) {
                first = min(behind + token0, key1 - 1);
                last = min(behind + end_token, key1 - 1);
            }
            return;
        }
        bool all = true;
        for (;;) {
            const bool whole = lens <= a.max_len && lens - (ends - begins) >= key1 - 1;
            all = all && __ballot(base + lane < a.sequences && !whole) == 0;
            if (base + 64 >= a.sequences) break;
            base += 64;
            sequences_at(a);
        }
        if (all) {
            first = last = key1 - 1;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (token[r] >= 0) lim[r] = key1 - 1;
            return;
        }
        if (base > 0) {
            base = 0;
            sequences_at(a);
        }
        for (int k = token0; k <= end_token; ++k) {
            int below;
            while ((below = __popcll(__ballot(base + lane < a.sequences && ends <= t0 + k))) == 64 && base + 64 < a.sequences) {
                base += 64;  // (the tokens to come are not in front of these either)
                sequences_at(a);
            }
            const int len = __builtin_amdgcn_readlane(lens, min(below, 63)), end = __builtin_amdgcn_readlane(ends, min(below, 63));
            const bool long_one = len > a.max_len;
            const int pos = min(len - end + t0 + k, key1 - 1);
            if (!long_one) {
                last = max(last, pos);
                first = min(first, pos);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (token[r] == k) {
                    over[r] = long_one;
                    lim[r] = long_one ? -1 : pos;
                }
        }
        last = __builtin_amdgcn_readfirstlane(last);
        first = __builtin_amdgcn_readfirstlane(first);
    }
    __device__ __forceinline__ void take(const AttnArgs &a) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            qs[r] = 1.f;
            float amax = 0.f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    qf[r][s][j] *= a.scale;
                    if constexpr (sizeof(T) == 2) amax = fmaxf(amax, fabsf(qf[r][s][j]));
                }
            if constexpr (sizeof(T) == 2) {
                const float f = half_scale(pa_max4(amax));
                qs[r] = 1.f / f;
#pragma unroll
                for (int s = 0; s < D / 32; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float y = qf[r][2 * s + (j >> 2)][j & 3] * f;
                        qh[r][s][j] = (_Float16)y;
                        ql[r][s][j] = (_Float16)(y - (float)qh[r][s][j]);
                    }
            }
            less[r] = FLT_MAX;
            l[r] = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[r][e] = f32x4v{0.f, 0.f, 0.f, 0.f};
        }
        asm("v_mov_b32 %0, -1.0" : "=v"(minus));
    }

    // Scores sc[r][t][i] of row n (in units of 1 / qs), key base + 16 t + 4 g + i, to weights 2^(score + less).  Only where the largest would be above 2^(PA_WEIGHT + PA_LAG) does less
    // follow the scores: the rescaling of the output, which a wave of 32 rows would need in nearly every step of a short span, is left to the
    // first.  It need not be PA_WEIGHT minus the maximum to the bit, only the same for all of a row's weights here and, as their unit, for whoever joins them with others; where FP32 cannot hold
    // it within 1/4 (scores beyond 2^23), it does without PA_WEIGHT.
    template <int TILES>
    __device__ __forceinline__ void weigh(f32x4v (&sc)[R][TILES], const int base, const bool partial) {
        const int g = (threadIdx.x & 63) >> 4;
        if (partial) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[r][t][i] = base + 16 * t + 4 * g + i <= lim[r] ? sc[r][t][i] : -INFINITY;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[r][t][i]);
            top = pa_max4(top);
            if constexpr (sizeof(T) == 2) top *= qs[r];
            if (__ballot(top + less[r] > PA_WEIGHT + PA_LAG)) {
                const float full = PA_WEIGHT - top, now = fminf(less[r], fabsf(full + top - PA_WEIGHT) <= 0.25f ? full : -top);
                const float f = __builtin_amdgcn_exp2f(now - less[r]);
                l[r] *= f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[r][e] *= f;
                less[r] = now;
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    float p0, p1;
                    if constexpr (sizeof(T) == 2) {
                        p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][t][i], qs[r], less[r]));
                        p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][t][i + 1], qs[r], less[r]));
                    } else {
                        p0 = __builtin_amdgcn_exp2f(sc[r][t][i] + less[r]);
                        p1 = __builtin_amdgcn_exp2f(sc[r][t][i + 1] + less[r]);
                    }
                    l[r] += p0 + p1;
                    if constexpr (sizeof(T) == 2) {
                        const f16x2 hi = __builtin_convertvector((f32x2{p0, p1}), f16x2);
                        const f16x2 lo = __builtin_convertvector((f32x2{__builtin_fmaf((float)hi[0], minus, p0), __builtin_fmaf((float)hi[1], minus, p1)}), f16x2);
                        ph[r][2 * t + i / 2] = __builtin_bit_cast(uint32_t, hi);
                        pl[r][2 * t + i / 2] = __builtin_bit_cast(uint32_t, lo);
                    } else {
                        pf[r][i] = p0;
                        pf[r][i + 1] = p1;
                    }
                }
        }
    }

    // Of values that only some rows see, the ones that are not finite: cleared, and their first position kept.  v: keys base + 16 t + 4 g + i.
    template <int TILES>
    __device__ __forceinline__ void clean(T (&v)[TILES][4][E], const int base) {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool fine = true;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const bool f = pa_finite(v[t][i][e]);
                    fine = fine && f;
                    if (!f) v[t][i][e] = (T)0.f;
                }
                if (!fine) badkey = min(badkey, base + 16 * t + 4 * g + i);
            }
    }

    // o[r][e][i], value E (4 g + i) + e of row n, += weights times the e-th of the lane's values of each key
    template <int TILES>
    __device__ __forceinline__ void sum(T (&v)[TILES][4][E], const int e) {
        if constexpr (sizeof(T) == 2) {
            f16x8 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = v[0][i][e];
                x[4 + i] = v[TILES - 1][i][e];
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                o[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(f16x8, pl[r]), o[r][e], 0, 0, 0);
                o[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(f16x8, ph[r]), o[r][e], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0][i][e], pf[r][i], o[r][e], 0, 0, 0);
        }
    }

    // the score of a weight of 1; -inf where there are no weights
    __device__ __forceinline__ float unit(const int r) const { return less[r] < FLT_MAX ? -less[r] : -INFINITY; }
    // the sum of row n's weights over the four lanes that hold it; NaN for a row that is to be NaN
    __device__ __forceinline__ float total(const int r) const { return over[r] || lim[r] >= badkey ? NAN : pa_sum4(l[r]); }
    __device__ __forceinline__ void spread_badkey() {
        if (!__ballot(badkey != 0x7fffffff)) return;
        for (int off = 1; off < 64; off <<= 1) badkey = min(badkey, __shfl_xor(badkey, off));
    }
};

// Where the tiles of 16 keys of the steps of a wave or workgroup lie, looked up and laid out for 64 steps at a time, a lane to each: in the loop a
// tile's descriptors are two lane reads and a few scalar additions (worked out there from the page's number they were a quarter of its instructions).
// A descriptor's extent ends behind the last key: what lies behind reads as zero without a branch or a mask, and a tile that does not exist
// (behind the last key, on a page that the cache does not have) costs nothing.
template <int TILES, int KEYS, int ROW>
struct PaPages {
    int lo[TILES], hi[TILES];  // lane u: bytes from the pool's start (48 bits) and, in the top bits, keys; first the pages' numbers in lo
    // the pages of the steps step0 + stride * lane, of keys below `end` (which may be asked for before it is known how many of them are seen: then settle)
    __device__ __forceinline__ void fetch(const AttnArgs &a, const int *table, const int key0, const int end, const int step0, const int stride) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int key = key0 + (step0 + lane * stride) * KEYS + 16 * t;
            lo[t] = key < end ? table[key >> a.page_shift] : -1;
        }
    }
    __device__ __forceinline__ void settle(const AttnArgs &a, const int key0, const int kend, const int step0, const int stride, int &badkey) {
        const int lane = threadIdx.x & 63;
        const size_t page_bytes = ((size_t)a.kv << a.page_shift) * ROW;
        int bad = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int key = key0 + (step0 + lane * stride) * KEYS + 16 * t;
            const bool seen = key < kend, there = (unsigned)lo[t] < (unsigned)a.pages;
            if (seen && !there) bad = min(bad, key);
            const size_t at = seen && there ? (size_t)lo[t] * page_bytes + (size_t)((key & ((1 << a.page_shift) - 1)) * ROW) : 0;
            lo[t] = (int)(unsigned)at;
            hi[t] = (int)(unsigned)(at >> 32) | (seen && there ? min(kend - key, 16) << 16 : 0);
        }
        if (__ballot(bad != 0x7fffffff)) {
            for (int off = 1; off < 64; off <<= 1) bad = min(bad, __shfl_xor(bad, off));
            badkey = min(badkey, bad);
        }
    }
    __device__ __forceinline__ void look_up(const AttnArgs &a, const int *table, const int key0, const int kend, const int step0, const int stride, int &badkey) {
        fetch(a, table, key0, kend, step0, stride);
        settle(a, key0, kend, step0, stride, badkey);
    }
    struct Place {
        size_t at;
        int extent;
    };
    __device__ __forceinline__ Place tile(const int u, const int t) const {
        unsigned l = __builtin_amdgcn_readlane(lo[0], u), h = __builtin_amdgcn_readlane(hi[0], u);
#pragma unroll
        for (int i = 1; i < TILES; ++i)
            if (t == i) {
                l = __builtin_amdgcn_readlane(lo[i], u);
                h = __builtin_amdgcn_readlane(hi[i], u);
            }
        return Place{((size_t)(h & 0xffffu) << 32) | l, (int)(h >> 16) * ROW};
    }
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(const uint8_t *pages, const Place &p) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)(pages + p.at), 0, p.extent, 0x00020000);
    }
};

// ---- few rows: every wave streams keys of its own

// LDS of a workgroup: outputs [wave][16 R][D + 4], maxima and sums [wave][16 R]
template <int D, int R>
constexpr size_t pa_stream_floats() {
    return (size_t)PA_WAVES * 16 * R * (D + 4) + 2 * PA_WAVES * 16 * R;
}

// The waves take rows in 4 / key_waves shares and, of each share, every key_waves-th step of the span.
template <class T, int D, int R>
__device__ __forceinline__ void pa_stream(const AttnArgs &a, const AttnPart &part, const bool ahead, const int seq, const int block, const int kvh, const int key0,
                                          const int key1, const int slot, const int slots, float *lds) {
    using Tile = PaTile<T, D>;
    constexpr int KEYS = Tile::KEYS, TILES = Tile::TILES, E = Tile::E, ROW = D * (int)sizeof(T);
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int key_waves = part.key_waves, row_waves = key_waves == PA_WAVES ? 1 : 2;  // (4 or 2 of the four)
    const int wr = wave & (row_waves - 1), wk = row_waves == 1 ? wave : wave >> 1;
    const int *table = a.tables + (size_t)(ahead ? 0 : seq) * a.table_stride;
    PaRows<T, D, R> w;
    PaPages<TILES, KEYS, ROW> pages;
    pages.fetch(a, table, key0, key1, wk, key_waves);
    if (!w.begin(a, ahead, seq, (block * row_waves + wr) * 16 * R, block * row_waves * 16 * R, key0)) return;
    w.fetch(a, kvh);
    w.find(a, ahead, seq, key1);
    const int kend = w.last + 1;  // keys key0 .. kend - 1
    const int steps = kend > key0 ? (kend - key0 + KEYS - 1) / KEYS : 0;
    const uint8_t *const kbase = (const uint8_t *)a.k + ((size_t)kvh << a.page_shift) * ROW, *const vbase = (const uint8_t *)a.v + ((size_t)kvh << a.page_shift) * ROW;
    const int koff = n * ROW + 16 * g, voff = 4 * g * ROW + E * n * (int)sizeof(T);
    Tile x;
    auto load_k = [&](int u) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const auto p = pages.source(kbase, pages.tile(u, t));
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int s = 0; s < D / 32; ++s) x.k[t][s] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(p, koff + 64 * s, 0, 0));
            } else {
#pragma unroll
                for (int s = 0; s < D / 16; ++s) x.k[s] = __builtin_bit_cast(f32x4v, __builtin_amdgcn_raw_buffer_load_b128(p, koff + 64 * s, 0, 0));
            }
        }
    };
    auto load_v = [&](int u) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const auto p = pages.source(vbase, pages.tile(u, t));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                constexpr int W = E * sizeof(T) % 16 == 0 ? 16 : 8;  // bytes of a load
#pragma unroll
                for (int b = 0; b < E * (int)sizeof(T) / W; ++b) {
                    if constexpr (W == 16)
                        *reinterpret_cast<u32x4 *>(&x.v[t][i][b * W / sizeof(T)]) = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(p, voff + i * ROW + b * W, 0, 0));
                    else
                        *reinterpret_cast<u32x2 *>(&x.v[t][i][b * W / sizeof(T)]) = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(p, voff + i * ROW + b * W, 0, 0));
                }
            }
        }
    };

    int step = wk, u = 0;  // u: the lane that holds the places of `step`
    if (step < steps) {
        pages.settle(a, key0, kend, step, key_waves, w.badkey);
        load_k(0);
        load_v(0);
    }
    w.take(a);
    while (step < steps) {
        const int base = key0 + step * KEYS;
        f32x4v sc[R][TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                f32x4v c = {0.f, 0.f, 0.f, 0.f};
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int s = 0; s < D / 32; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[t][s], w.ql[r][s], c, 0, 0, 0);
#pragma unroll
                    for (int s = 0; s < D / 32; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[t][s], w.qh[r][s], c, 0, 0, 0);
                } else {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[s][j], w.qf[r][s][j], c, 0, 0, 0);
                }
                sc[r][t] = c;
            }
        // the keys of the next step, into the registers that the products have read.  (Without a branch: one around these loads, in FP32 with heads of 192 values, left the products' first
        // use without the wait it needs.  Behind the other branches between the two, here and in pa_wide, the compiler puts it on every way there, as the listing shows: to be looked at
        // again with any change to what stands between.)
        const int next = step + key_waves;
        load_k((u + 1) & 63);
        const bool partial = base + KEYS - 1 > w.first;  // some row does not see all of them
        if (partial && w.first < w.last) w.clean(x.v, base);  // ... and others see more
        w.weigh(sc, base, partial);
#pragma unroll
        for (int e = 0; e < E; ++e) w.sum(x.v, e);
        u = (u + 1) & 63;
        load_v(u);
        step = next;
        if (u == 63) pages.look_up(a, table, key0, kend, step + key_waves, key_waves, w.badkey);  // (what is under way has its places)
    }

    // ---- the waves' sums meet in LDS
    w.spread_badkey();
    float *const lo = lds, *const lm = lds + (size_t)PA_WAVES * 16 * R * (D + 4), *const ll = lm + PA_WAVES * 16 * R;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float *p = lo + (size_t)(wave * 16 * R + 16 * r + n) * (D + 4) + 4 * E * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<f32x4v *>(p + E * i + e) = f32x4v{w.o[r][e][i], w.o[r][e + 1][i], w.o[r][e + 2][i], w.o[r][e + 3][i]};
        const float sum = w.total(r);
        if (g == 0) {
            lm[wave * 16 * R + 16 * r + n] = w.unit(r);
            ll[wave * 16 * R + 16 * r + n] = sum;
        }
    }
    __syncthreads();
    const int first_row = block * row_waves * 16 * R, token_of_first = pa_div(first_row, a.group, a.by_group), rem_of_first = first_row - token_of_first * w.group;
    for (int at = tid; at < row_waves * 16 * R * (D / 4); at += PA_THREADS) {
        const int rr = at / (D / 4), e = 4 * (at - rr * (D / 4)), wv = rr / (16 * R), in = rr - wv * 16 * R;  // wave wv + row_waves j holds row `in` of the keys' share j
        if (first_row + rr >= w.rows) break;  // (rr grows with at)
        float top = -INFINITY, sum = 0.f;
        f32x4v acc = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < key_waves; ++j) top = fmaxf(top, lm[(wv + row_waves * j) * 16 * R + in]);
        for (int j = 0; j < key_waves; ++j) {
            const int src = (wv + row_waves * j) * 16 * R + in;
            const float mm = lm[src], f = mm > -INFINITY ? __builtin_amdgcn_exp2f(mm - top) : 0.f;
            // (a wave without a key has no weight; one whose rows are to be NaN has, whatever its unit)
            sum += ll[src] == ll[src] ? ll[src] * f : NAN;
            acc += *reinterpret_cast<const f32x4v *>(lo + (size_t)src * (D + 4) + e) * f;
        }
        if (slots == 1) {
            const int q = (int)(((float)(rem_of_first + rr) + 0.5f) * w.per_group), t = w.t0 + token_of_first + q, h = kvh * w.group + rem_of_first + rr - q * w.group;
            // (a row that sees nothing is zero)
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<f32x4v_a4 *>(a.y + (size_t)t * a.y_stride + (size_t)h * D + e) = acc * f;
        } else {
            const size_t at_slot = (((size_t)kvh * a.tokens + w.t0) * w.group + first_row + rr) * slots + slot;
            *reinterpret_cast<f32x4v *>(a.part + at_slot * D + e) = acc;
            if (e == 0) *reinterpret_cast<float2 *>(a.stat + 2 * at_slot) = make_float2(top, sum);
        }
    }
}

// ---- many rows: the workgroup's waves take rows of their own and the same keys, through LDS

// A step's keys and values lie in LDS as rows of 16-byte pieces.  A lane reads piece c of key n, sixteen keys side by side: the pieces of a
// key's row trade places by its number, so that the sixteen are in sixteen different quads of banks.
template <int PIECES>
__device__ __forceinline__ int pa_piece(int c, int n) { return PIECES % 16 == 0 ? c ^ (n & 15) : c ^ ((n >> 1) & 7); }

template <class T, int D>
struct PaWide {
    using Tile = PaTile<T, D>;
    static constexpr int PIECES = D * (int)sizeof(T) / 16;                 // of a row
    static constexpr int STEP = Tile::KEYS * PIECES;                       // of a step's keys, and of its values
    static constexpr int COPIES = STEP / PA_THREADS;                       // of each per thread
    static constexpr int AHEAD = 2;                                        // steps in registers on their way to LDS
    static constexpr size_t LDS = (size_t)2 * 2 * STEP * 16;               // two steps
    static_assert(STEP % PA_THREADS == 0 && 16 * PIECES % 64 == 0, "whole copies, whole waves to a tile");
};

// All waves on the same keys, 16 R rows each.  What the waves need of a step is requested two steps before, each wave a quarter of it (a wave that
// requested all of it for itself waited 5000 cycles a step where the products take 1000), goes to LDS a step before, and one barrier a step says
// that it is there and that the step before has been read.
template <class T, int D, int R>
__device__ __forceinline__ void pa_wide(const AttnArgs &a, const bool ahead, const int seq, const int block, const int kvh, const int key0, const int key1, const int slot,
                                        const int slots, float *lds) {
    using W = PaWide<T, D>;
    using Tile = typename W::Tile;
    constexpr int KEYS = Tile::KEYS, TILES = Tile::TILES, E = Tile::E, ROW = D * (int)sizeof(T), PIECES = W::PIECES, COPIES = W::COPIES;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int *table = a.tables + (size_t)(ahead ? 0 : seq) * a.table_stride;
    PaRows<T, D, R> w;
    PaPages<TILES, KEYS, ROW> pages;
    pages.fetch(a, table, key0, key1, 0, 1);
    if (!w.begin(a, ahead, seq, (block * PA_WAVES + wave) * 16 * R, block * PA_WAVES * 16 * R, key0)) return;
    w.fetch(a, kvh);
    w.find(a, ahead, seq, key1);
    // keys key0 .. kend - 1: what any row of the workgroup may see, and some of the shared ones perhaps that none does
    int kend = key1;
    if (!ahead) {
        const int len = a.lens[seq], last_token = pa_div(min((block + 1) * PA_WAVES * 16 * R, w.rows), a.group, a.by_group);  // ... or the one behind it
        kend = min(key1, len - (a.starts[seq + 1] - w.t0) + min(last_token + 1, pa_div(w.rows, a.group, a.by_group)));
        if (slots > 1 && kend <= key0) return;  // (a span that begins behind a row's position is not read)
    }
    const int steps = kend > key0 ? (kend - key0 + KEYS - 1) / KEYS : 0;
    const uint8_t *const kbase = (const uint8_t *)a.k + ((size_t)kvh << a.page_shift) * ROW, *const vbase = (const uint8_t *)a.v + ((size_t)kvh << a.page_shift) * ROW;
    // copy i of this thread: LDS piece tid + 256 i of the step, i.e. piece (..) % PIECES of row (..) / PIECES; all of a wave's are in one tile
    int koff[COPIES], voff[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const int j = tid + PA_THREADS * i, row = j / PIECES, c = j - row * PIECES;
        koff[i] = (row & 15) * ROW + 16 * pa_piece<PIECES>(c, row & 15);
        voff[i] = (row & 15) * ROW + 16 * c;
    }
    u32x4 kr[W::AHEAD][COPIES], vr[W::AHEAD][COPIES];
    uint8_t *const sm = reinterpret_cast<uint8_t *>(lds);  // [2][keys, values][STEP][16]
    auto request = [&](auto slot_c, int u) {
        constexpr int S = decltype(slot_c)::value;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            constexpr int TILE = 16 * PIECES;
            const auto p = pages.tile(u, TILES == 1 ? 0 : TILE % PA_THREADS == 0 ? i * PA_THREADS / TILE : (wave + PA_WAVES * i) * 64 / TILE);
            kr[S][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(pages.source(kbase, p), koff[i], 0, 0));
            vr[S][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(pages.source(vbase, p), voff[i], 0, 0));
        }
    };
    auto store = [&](auto slot_c, int buffer) {
        constexpr int S = decltype(slot_c)::value;
        u32x4 *p = reinterpret_cast<u32x4 *>(sm + (size_t)buffer * 2 * W::STEP * 16);
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            p[tid + PA_THREADS * i] = kr[S][i];
            p[W::STEP + tid + PA_THREADS * i] = vr[S][i];
        }
    };
    auto product = [&](int step) {
        const int base = key0 + step * KEYS;
        if (base > w.last) return;  // (none of the wave's rows sees any of them)
        const uint8_t *ks = sm + (size_t)(step & 1) * 2 * W::STEP * 16, *vs = ks + (size_t)W::STEP * 16;
        f32x4v sc[R][TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < R; ++r) sc[r][t] = f32x4v{0.f, 0.f, 0.f, 0.f};
        u32x4 keys[PIECES / 4][TILES];  // (all requested before the first is used, in the registers that the values take afterwards)
#pragma unroll
        for (int s = 0; s < PIECES / 4; ++s)
#pragma unroll
            for (int t = 0; t < TILES; ++t) keys[s][t] = *reinterpret_cast<const u32x4 *>(ks + (size_t)(16 * t + n) * ROW + 16 * pa_piece<PIECES>(4 * s + g, n));
        __builtin_amdgcn_sched_barrier(0);
        // (a wave with operands for the matrix cores goes before one that works on weights: 64 sequences of 32 heads of 128 behind 131072 positions 274 us with the merge, 283 without)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < PIECES / 4; ++s) {
            const u32x4(&k)[TILES] = keys[s];
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int r = 0; r < R; ++r) sc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[t]), w.ql[r][s], sc[r][t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int r = 0; r < R; ++r) sc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[t]), w.qh[r][s], sc[r][t], 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < R; ++r) sc[r][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4v, k[0])[j], w.qf[r][s][j], sc[r][0], 0, 0, 0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        const bool partial = base + KEYS - 1 > w.first;
        w.weigh(sc, base, partial);
        T v[TILES][4][E] __attribute__((aligned(16)));
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                constexpr int V = E * sizeof(T) % 16 == 0 ? 16 : 8;
                const uint8_t *p = vs + (size_t)(16 * t + 4 * g + i) * ROW + E * n * (int)sizeof(T);
#pragma unroll
                for (int b = 0; b < E * (int)sizeof(T) / V; ++b) {
                    if constexpr (V == 16) *reinterpret_cast<u32x4 *>(&v[t][i][b * V / sizeof(T)]) = *reinterpret_cast<const u32x4 *>(p + b * V);
                    else *reinterpret_cast<u32x2 *>(&v[t][i][b * V / sizeof(T)]) = *reinterpret_cast<const u32x2 *>(p + b * V);
                }
            }
        if (partial) w.clean(v, base);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int e = 0; e < E; ++e) w.sum(v, e);
        __builtin_amdgcn_s_setprio(0);
    };
    // steps s and s + 1 are requested, s is stored, from then on: barrier, request s + 2, store s + 1, product s
    constexpr std::integral_constant<int, 0> c0{};
    constexpr std::integral_constant<int, 1> c1{};
    if (steps > 0) {
        pages.settle(a, key0, kend, 0, 1, w.badkey);
        request(c0, 0);
        request(c1, 1);
    }
    w.take(a);
    if (steps > 0) store(c0, 0);
    auto turn = [&](auto mine, auto other, int step) {  // step's registers were `mine`
        if ((step & 63) == 62) pages.look_up(a, table, key0, kend, step + 2, 1, w.badkey);
        request(mine, (step + 2) & 63);
        __syncthreads();
        product(step);
        store(other, (step + 1) & 1);
    };
    for (int step = 0; step < steps; step += 2) {
        turn(c0, c1, step);
        if (step + 1 < steps) turn(c1, c0, step + 1);
    }

    // ---- the outputs, turned in LDS so that a row goes out in one piece (a lane holds E values of it at four places)
    w.spread_badkey();
    __syncthreads();
    float *const mine = lds + (size_t)wave * 16 * (D + 4);
    const size_t first_slot = (((size_t)kvh * a.tokens + w.t0) * w.group + w.row0) * slots + slot;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = w.total(r), f = slots > 1 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;  // (a row that sees nothing is zero)
        float *p = mine + n * (D + 4) + 4 * E * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<f32x4v *>(p + E * i + e) = f32x4v{w.o[r][e][i], w.o[r][e + 1][i], w.o[r][e + 2][i], w.o[r][e + 3][i]} * f;
        const int row_n = w.row0 + 16 * r + n;
        if (slots > 1 && g == 0 && row_n < w.rows) {
            *reinterpret_cast<float2 *>(a.stat + 2 * (first_slot + (size_t)(16 * r + n) * slots)) = make_float2(w.unit(r), sum);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 16 * (D / 4) / 64; ++i) {
            const int piece = lane + 64 * i, in = piece / (D / 4), e = 4 * (piece - in * (D / 4));
            const f32x4v v = *reinterpret_cast<const f32x4v *>(mine + in * (D + 4) + e);
            if (w.row0 + 16 * r + in < w.rows) {
                float *to = a.part + (first_slot + (size_t)(16 * r + in) * slots) * D;
                if (slots == 1) {
                    const int2 at = w.place(16 * r + in);
                    to = a.y + (size_t)(w.t0 + at.x) * a.y_stride + (size_t)(kvh * w.group + at.y) * D;
                }
                *reinterpret_cast<f32x4v_a4 *>(to + e) = v;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

template <class T, int D, int R>
__device__ __forceinline__ void pa_attend(const AttnArgs &a, const AttnPart &part, const bool ahead, const int seq, const int block, const int kvh, const int key0,
                                          const int key1, const int slot, const int slots, float *lds) {
    if (part.key_waves == 1) {
        pa_wide<T, D, R>(a, ahead, seq, block, kvh, key0, key1, slot, slots, lds);
        return;
    }
    if constexpr (R == 2) {
        // (of a ragged batch: a sequence whose rows fill one tile takes no product for the other)
        if (!ahead && part.key_waves == PA_WAVES && (a.starts[seq + 1] - a.starts[seq]) * a.group <= 16) {
            pa_stream<T, D, 1>(a, part, ahead, seq, block, kvh, key0, key1, slot, slots, lds);
            return;
        }
    }
    pa_stream<T, D, R>(a, part, ahead, seq, block, kvh, key0, key1, slot, slots, lds);
}

// The workgroups: `chunk` of the shared positions, as many of the sequences' own, and so on until one kind is used up - the first are bound by the matrix
// cores, the others by memory, and a CU that holds one of each has use for both.  Of one kind, `beside` units (span, sequence, key/value head) are taken
// together, and workgroup b of them takes row block b / beside of unit b % beside: the row blocks of a unit, which read the same keys, run on one
// XCD (workgroups go round the eight).  Of the sequences' own positions the last rows, which see most of a prompt's, go first, of as many units
// as run at once (three prompts of 332 tokens, 56 heads of 128, FP32: 87 us with 8 units together, 77 so).
template <class T, int D, int RA, int RO>
__global__ void __launch_bounds__(PA_THREADS, D <= 128 ? 2 : 1) paged_attn_kernel(const AttnArgs a) {
    extern __shared__ __align__(16) float pa_lds[];
    const unsigned kv = (unsigned)a.kv, seqs = (unsigned)a.sequences, chunk = (unsigned)a.chunk;
    unsigned in, of, side, kvh;
    const unsigned c = pa_div(blockIdx.x, chunk, a.by_chunk, in);
    const bool own = c < 2 * (unsigned)a.pairs ? (c & 1) != 0 : a.chunks_own > a.chunks_ahead;
    const unsigned b = (c < 2 * (unsigned)a.pairs ? c / 2 : c - (unsigned)a.pairs) * chunk + in;
    const int slots = a.ahead.spans + a.own.spans;
    if (!own) {
        const unsigned beside = (unsigned)a.ahead.beside, first = pa_div(b, beside * (unsigned)a.ahead.blocks, a.by_ahead, of) * beside;
        const unsigned block = pa_div(of, beside, a.by_ahead_beside, side), u = first + side;
        if (u >= kv * (unsigned)a.ahead.spans) return;
        const int span = (int)pa_div(u, kv, a.by_kv, kvh);
        pa_attend<T, D, RA>(a, a.ahead, true, 0, (int)block, (int)kvh, span * a.ahead.span, min((span + 1) * a.ahead.span, a.shared), span, slots, pa_lds);
    } else {
        const unsigned beside = (unsigned)a.own.beside, first = pa_div(b, beside * (unsigned)a.own.blocks, a.by_own, of) * beside;
        const unsigned block = pa_div(of, beside, a.by_own_beside, side), u = first + side;
        if (u >= kv * seqs * (unsigned)a.own.spans) return;
        unsigned seq;
        const int span = (int)pa_div(pa_div(u, kv, a.by_kv, kvh), seqs, a.by_sequences, seq);
        const int key0 = a.shared + span * a.own.span;
        pa_attend<T, D, RO>(a, a.own, false, (int)seq, a.own.blocks - 1 - (int)block, (int)kvh, key0, min(key0 + a.own.span, a.max_len), a.ahead.spans + span, slots, pa_lds);
    }
}

// ---- y of every row (token, head) from its spans, y = sum_i 2^(u_i - u) o_i / sum_i 2^(u_i - u) l_i with u_i the units of their weights (PaRows::unit) and u the largest: bound by the latency of a chain (the
// token's sequence, the statistics, the sums) where rows are few, 4 us, and by memory where they are many.  Spans that begin behind the row's position were not written.
constexpr int PA_MERGE = 256;

// What token t's rows see: spans of the shared positions and of the sequence's own; false where y is already right or has been made so (`rows` rows of it from y
// on, this thread's four values of each group of D / 4 threads).
struct MergeRow {
    int ahead, count;
};
template <int D>
__device__ __forceinline__ bool merge_row(const AttnArgs &a, const int t, const bool writes, f32x4v_a4 *y, MergeRow &m) {
    const RowPlace at = row_place(a.starts, a.lens, a.sequences, t);
    if (at.sequence >= a.sequences || t < a.starts[0]) return false;  // behind the last sequence
    const int lim = at.len - at.end + t;
    if (lim < 0 || at.len > a.max_len) {
        const float f = at.len > a.max_len ? NAN : 0.f;
        if (writes) *y = f32x4v{f, f, f, f};
        return false;
    }
    m.ahead = min(a.ahead.spans, a.shared > 0 ? pa_div(lim, a.ahead.span, a.by_ahead_span) + 1 : 0);
    m.count = m.ahead + (lim >= a.shared ? pa_div(lim - a.shared, a.own.span, a.by_own_span) + 1 : 0);
    return true;
}

// Few spans: D / 4 threads take a row, a workgroup PA_MERGE / (D / 4) rows of a token.
constexpr int PA_FEW = 8;
template <int D>
__global__ void __launch_bounds__(PA_MERGE) paged_merge_few_kernel(const AttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = PA_MERGE / LANES;
    const int tid = threadIdx.x, grp = tid / LANES, in = tid - grp * LANES, t = blockIdx.x, h = blockIdx.y * GROUPS + grp;
    const bool mine = grp < GROUPS && h < a.heads;
    f32x4v_a4 *y = reinterpret_cast<f32x4v_a4 *>(a.y + (size_t)t * a.y_stride + (size_t)h * D) + in;
    MergeRow m;
    if (!merge_row<D>(a, t, mine, y, m) || !mine) return;
    const int group = a.group, kvh = pa_div(h, group, a.by_group);
    const size_t first_slot = (((size_t)kvh * a.tokens + t) * group + h - kvh * group) * (a.ahead.spans + a.own.spans);
    f32x4v x[PA_FEW];
    float2 st[PA_FEW];
#pragma unroll
    for (int u = 0; u < PA_FEW; ++u)
        if (u < m.count) {
            const size_t slot = first_slot + (u < m.ahead ? u : a.ahead.spans + u - m.ahead);
            st[u] = *reinterpret_cast<const float2 *>(a.stat + 2 * slot);
            x[u] = *reinterpret_cast<const f32x4v *>(a.part + slot * D + 4 * in);
        }
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int u = 0; u < PA_FEW; ++u)
        if (u < m.count) top = fmaxf(top, st[u].x);
    f32x4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < PA_FEW; ++u)
        if (u < m.count) {
            const float f = st[u].x > -INFINITY ? __builtin_amdgcn_exp2f(st[u].x - top) : 0.f;
            sum += st[u].y == st[u].y ? st[u].y * f : NAN;
            acc += x[u] * f;
        }
    *y = acc * (sum == 0.f ? 0.f : 1.f / sum);
}

// Many: a workgroup per row, groups of D / 4 threads take a span each, all of a group's requested before the first is used.
template <int D>
__global__ void __launch_bounds__(PA_MERGE) paged_merge_kernel(const AttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = PA_MERGE / LANES, U = 8;
    __shared__ float weight[PA_MERGE], top_of[PA_MERGE / 64], sum_of[PA_MERGE / 64];
    __shared__ f32x4v part_of[GROUPS][LANES];
    const int tid = threadIdx.x, wave = tid >> 6, grp = tid / LANES, in = tid - grp * LANES;
    const int t = blockIdx.x, h = blockIdx.y, slots = a.ahead.spans + a.own.spans;
    f32x4v_a4 *y = reinterpret_cast<f32x4v_a4 *>(a.y + (size_t)t * a.y_stride + (size_t)h * D);
    MergeRow m;
    if (!merge_row<D>(a, t, grp == 0, y + in, m)) return;
    const int first_own = a.ahead.spans, ahead = m.ahead, count = m.count;  // at most PA_MERGE (paged_attn_plan)
    const int group = a.group, kvh = pa_div(h, group, a.by_group);
    const size_t first_slot = (((size_t)kvh * a.tokens + t) * group + h - kvh * group) * slots;
    auto slot_of = [&](int i) { return first_slot + (i < ahead ? i : first_own + i - ahead); };
    f32x4v acc = {0.f, 0.f, 0.f, 0.f}, x[U];
    auto request = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const f32x4v *>(a.part + slot_of(min(i0 + u * GROUPS, count - 1)) * D + 4 * in);
    };
    const bool mine = grp < GROUPS;
    if (mine) request(grp);
    float2 st = tid < count ? *reinterpret_cast<const float2 *>(a.stat + 2 * slot_of(tid)) : make_float2(-INFINITY, 0.f);
    const float best = wave_max(st.x);
    if ((tid & 63) == 0) top_of[wave] = best;
    __syncthreads();
    const float top = fmaxf(fmaxf(top_of[0], top_of[1]), fmaxf(top_of[2], top_of[3]));
    const float f = st.x > -INFINITY ? __builtin_amdgcn_exp2f(st.x - top) : 0.f;
    weight[tid] = f;
    const float sum = wave_sum(st.y == st.y ? st.y * f : NAN);
    if ((tid & 63) == 0) sum_of[wave] = sum;
    __syncthreads();
    if (mine)
        for (int i0 = grp; i0 < count; i0 += U * GROUPS) {
            if (i0 != grp) request(i0);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * GROUPS < count) acc += x[u] * weight[i0 + u * GROUPS];
        }
    if (mine) part_of[grp][in] = acc;
    __syncthreads();
    if (grp == 0) {
        for (int j = 1; j < GROUPS; ++j) acc += part_of[j][in];
        const float all = (sum_of[0] + sum_of[1]) + (sum_of[2] + sum_of[3]);
        y[in] = acc * (all == 0.f ? 0.f : 1.f / all);
    }
}

// ---- launch

template <class T, int D, int R>
constexpr size_t pa_lds_bytes() {
    return std::max(pa_stream_floats<D, R>() * sizeof(float), PaWide<T, D>::LDS);
}
template <class T, int D, int RA, int RO>
static void paged_attn_run(unsigned blocks, hipStream_t s, const AttnArgs &a) {
    constexpr size_t lds = pa_lds_bytes<T, D, (RA > RO ? RA : RO)>();
    // (more than 64 KiB must be asked for, once; a refusal shows at the launch)
    static const hipError_t asked = hipFuncSetAttribute((const void *)paged_attn_kernel<T, D, RA, RO>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    (void)asked;
    hipLaunchKernelGGL((paged_attn_kernel<T, D, RA, RO>), dim3(blocks), dim3(PA_THREADS), lds, s, a);
}
template <class T>
static void paged_attn_pick(int D, unsigned blocks, hipStream_t s, const AttnArgs &a) {
    auto tiles = [&](auto d) {
        constexpr int DD = decltype(d)::value;
        if (a.own.tiles == 2) paged_attn_run<T, DD, 2, 2>(blocks, s, a);
        else if (a.ahead.tiles == 2) paged_attn_run<T, DD, 2, 1>(blocks, s, a);
        else paged_attn_run<T, DD, 1, 1>(blocks, s, a);
    };
    switch (D) {
    case 64: tiles(std::integral_constant<int, 64>{}); break;
    case 128: tiles(std::integral_constant<int, 128>{}); break;
    case 192: paged_attn_run<T, 192, 1, 1>(blocks, s, a); break;
    default: paged_attn_run<T, 256, 1, 1>(blocks, s, a); break;
    }
}

}  // namespace jitnn
