// Attention of a batch over a paged cache: token t of sequence s, at position p, attends to the positions 0 .. p of s, whose keys and values lie
// in pages that a table names.  The leading pages may be everybody's: the workgroups that take their positions take the rows - (token, query
// head) pairs of one key/value head - of the whole batch, so that they are read once and not once per sequence; the other positions go
// to workgroups of their sequence.  Every workgroup leaves, for its span of keys, the largest score, the sum of the weights and the weighted sum
// of the values, and paged_merge_kernel joins a row's spans.
//
// The products run on the matrix cores, transposed, S^T = K Q^T and O^T = V^T P^T, and nothing but the last sums goes through LDS:
//   * lane n + 16 g holds for the scores key n of a tile of 16 (16 bytes of its row per load), receives the scores of ROW n against the keys
//     4 g + i, and those, as weights, are its slots of the P operand: its running maximum and sum are one row's.
//   * of the values the lane loads, for the very keys 4 g + i, the D / 16 neighbours from D / 16 n on: all a row of V, so that the loads of
//     16 lanes are one row in one piece, and the A operand of V^T needs no more than the lane's own registers - its tile e takes the e-th value
//     of each key, row n of that tile being value D / 16 n + e.
//   A wave so streams keys and values from memory at its own pace, without a barrier.
// FP16 pages: keys and values are operands as they are; queries (scaled so that a row's largest is near 2^13) and weights (times 2^6 to 2^14) go in two FP16
// parts, 22 bits together, so that the result is as good as in FP32.  FP32 pages: the FP32 matrix instruction.
// Sums, maxima and outputs are FP32.
//
// What a row does not see: its scores are masked; values past the last key that any row of the tile sees are cleared, and of those that only some see
// the ones that are not finite, whose rows become NaN (badkey): nothing behind a token reaches it.  The same mark makes NaN of rows whose positions
// lie on a page that the cache does not have.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "serving.h"

namespace jitnn {

constexpr int PA_THREADS = 256, PA_WAVES = 4;
constexpr int PA_SEARCH = 1024;  // sequences whose starts a workgroup keeps in LDS
constexpr float PA_WEIGHT = 6.f, PA_LAG = 8.f;  // weights are 2^(score - m + 6), m at most 8 below the maximum: up to 2^14, inside FP16

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
    float a = v, b = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    a = b = fmaxf(a, b);
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return fmaxf(a, b);
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

// The sequence of token t in ascending starts[0 .. sequences]
__device__ __forceinline__ int pa_sequence(const int *starts, int sequences, int t) {
    int lo = 0, hi = sequences;  // the first s with starts[s + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
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
            p.len = __shfl(len, below);
            p.end = __shfl(end, below);
            break;
        }
    }
    return p;
}

// What a wave holds of its rows, R tiles of 16.
template <class T, int D, int R>
struct PaRows {
    static constexpr int E = D / 16;
    int rows, row0, t0;    // rows of the part, the wave's first, the first row's token
    int lim[R];            // the last position of the span that row n sees
    bool over[R];          // ... of a sequence longer than it may be
    int first, last;       // the least and the largest lim
    int badkey;            // rows that see this position are NaN
    f16x8 qh[R][sizeof(T) == 2 ? D / 32 : 1], ql[R][sizeof(T) == 2 ? D / 32 : 1];
    f32x4v qf[R][D / 16];  // (FP16: until they are operands)
    float qs[R];
    f32x4v o[R][E];
    float m[R], l[R];
    float less[R];       // PA_WEIGHT - m
    float minus;         // -1, which the compiler does not know: it would take the FP16 part off the weight in two instructions and not in one
    u32x4 ph[R], pl[R];  // weights (FP16): slot 4 t + i
    float pf[R][4];      // (FP32)

    // Four steps, so that what they wait for is asked for together: begin (false: the workgroup has nothing to do), fetch (queries, and the starts and
    // lens to LDS), a barrier, find (the rows' positions), take (the queries as operands).
    __device__ __forceinline__ bool begin(const AttnArgs &a, const bool ahead, const int seq, const int row0_of_wave, const int row0_of_block, const int key0) {
        t0 = max(a.starts[ahead ? 0 : seq], 0);
        rows = max(min(a.starts[ahead ? a.sequences : seq + 1], a.tokens) - t0, 0) * (a.heads / a.kv);
        row0 = row0_of_wave;
        // (a span that no row of the sequence reaches; where there is one span in all, its rows are still to be written)
        return row0_of_block < rows && (ahead || key0 == 0 || a.lens[seq] > key0);
    }
    // queries: 8 g + j of each 32 values (FP16), 4 g + j of each 16 (FP32) of row n
    __device__ __forceinline__ void fetch(const AttnArgs &a, const bool ahead, const int kvh, int *search) {
        const int tid = threadIdx.x, n = tid & 15, g = (tid & 63) >> 4, group = a.heads / a.kv;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = min(row0 + 16 * r + n, rows - 1), t = t0 + row / group, h = kvh * group + row % group;
            const float *q = a.q + (size_t)t * a.q_stride + (size_t)h * D;
#pragma unroll
            for (int s = 0; s < D / 16; ++s) qf[r][s] = *reinterpret_cast<const f32x4v_a4 *>(q + (sizeof(T) == 2 ? 32 * (s >> 1) + 8 * g + 4 * (s & 1) : 16 * s + 4 * g));
        }
        if (ahead && a.sequences <= PA_SEARCH) {
            for (int i = tid; i <= a.sequences; i += PA_THREADS) search[i] = a.starts[i];
            for (int i = tid; i < a.sequences; i += PA_THREADS) search[a.sequences + 1 + i] = a.lens[i];
        }
    }
    __device__ __forceinline__ void find(const AttnArgs &a, const bool ahead, const int seq, const int key1, const int *search) {
        const bool near = ahead && a.sequences <= PA_SEARCH;
        const int *starts = near ? search : a.starts, *lens = near ? search + a.sequences + 1 : a.lens;
        const int n = threadIdx.x & 15, group = a.heads / a.kv;
        last = -1;
        first = badkey = 0x7fffffff;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = row0 + 16 * r + n, t = t0 + row / group;
            lim[r] = -1;
            over[r] = false;
            if (row < rows) {
                const int s = ahead ? min(pa_sequence(starts, a.sequences, t), a.sequences - 1) : seq;
                over[r] = lens[s] > a.max_len;
                if (!over[r]) {
                    lim[r] = min(lens[s] - starts[s + 1] + t, key1 - 1);
                    last = max(last, lim[r]);
                    first = min(first, lim[r]);
                }
            }
        }
        for (int off = 1; off < 16; off <<= 1) {
            last = max(last, __shfl_xor(last, off));
            first = min(first, __shfl_xor(first, off));
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
            m[r] = -INFINITY;
            l[r] = less[r] = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[r][e] = f32x4v{0.f, 0.f, 0.f, 0.f};
        }
        asm("v_mov_b32 %0, -1.0" : "=v"(minus));
    }

    // Scores sc[r][t][i] of row n (in units of 1 / qs), key base + 16 t + 4 g + i, to weights 2^(score - m + PA_WEIGHT).  m follows the maximum only when that
    // is more than PA_LAG above it: the rescaling of the output, which a wave of 32 rows would need in nearly every step of a short span, is left to the
    // first.
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
            if (__ballot(top > m[r] + PA_LAG)) {
                top = fmaxf(m[r], top);
                const float f = top > -INFINITY ? __builtin_amdgcn_exp2f(m[r] - top) : 1.f;
                l[r] *= f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[r][e] *= f;
                m[r] = top;
                less[r] = top > -INFINITY ? PA_WEIGHT - top : 0.f;
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

    // the sum of row n's weights over the four lanes that hold it; NaN for a row that is to be NaN
    __device__ __forceinline__ float total(const int r) const { return over[r] || lim[r] >= badkey ? NAN : pa_sum4(l[r]); }
    __device__ __forceinline__ void spread_badkey() {
        for (int off = 1; off < 64; off <<= 1) badkey = min(badkey, __shfl_xor(badkey, off));
    }
};

// Pages of the steps of a wave or workgroup, looked up 64 steps at a time, and the tiles of 16 keys in them, as descriptors whose extent ends behind the
// last key: what lies behind reads as zero without a branch or a mask, and a tile that does not exist (behind the last key, behind the last
// step, on a page that the cache does not have) costs nothing.
template <int TILES, int KEYS, int ROW>
struct PaPages {
    int ids[TILES];  // lane u: the pages of step `first of the 64` + u, -1: none
    // the pages of the steps step0 + stride * lane, of keys below `end` (which may be asked for before it is known how many of them are seen: then check)
    __device__ __forceinline__ void fetch(const AttnArgs &a, const int *table, const int key0, const int end, const int step0, const int stride) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int key = key0 + (step0 + lane * stride) * KEYS + 16 * t;
            ids[t] = key < end ? table[key >> a.page_shift] : -1;
        }
    }
    __device__ __forceinline__ void check(const AttnArgs &a, const int key0, const int kend, const int step0, const int stride, int &badkey) {
        const int lane = threadIdx.x & 63;
        int bad = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int key = key0 + (step0 + lane * stride) * KEYS + 16 * t;
            if ((unsigned)ids[t] >= (unsigned)a.pages) {
                if (key < kend) bad = min(bad, key);
                ids[t] = -1;
            }
        }
        if (__ballot(bad != 0x7fffffff)) {
            for (int off = 1; off < 64; off <<= 1) bad = min(bad, __shfl_xor(bad, off));
            badkey = min(badkey, bad);
        }
    }
    __device__ __forceinline__ void look_up(const AttnArgs &a, const int *table, const int key0, const int kend, const int step0, const int stride, int &badkey) {
        fetch(a, table, key0, kend, step0, stride);
        check(a, key0, kend, step0, stride, badkey);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t tile(const AttnArgs &a, const uint8_t *pages, const int key0, const int kend, const int step, const int u, const int t) const {
        const int key = key0 + step * KEYS + 16 * t;
        int id = __builtin_amdgcn_readlane(ids[0], u);
#pragma unroll
        for (int i = 1; i < TILES; ++i)
            if (t == i) id = __builtin_amdgcn_readlane(ids[i], u);
        const size_t at = (size_t)(id < 0 ? 0 : id) * (((size_t)a.kv << a.page_shift) * ROW) + (size_t)(key & ((1 << a.page_shift) - 1)) * ROW;
        // (in a scalar register by force: of the clamp the compiler makes a vector instruction, and of a descriptor in vector registers a loop)
        const int extent = __builtin_amdgcn_readfirstlane(id < 0 ? 0 : max(min(kend - key, 16), 0) * ROW);
        return __builtin_amdgcn_make_buffer_rsrc((void *)(pages + at), 0, extent, 0x00020000);
    }
};

// ---- few rows: every wave streams keys of its own

// LDS of a workgroup: outputs [wave][16 R][D + 4], maxima and sums [wave][16 R], then starts and lens
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
    const int group = a.heads / a.kv, key_waves = part.key_waves, row_waves = PA_WAVES / key_waves;
    const int wr = wave & (row_waves - 1), wk = wave / row_waves;
    const int *table = a.tables + (size_t)(ahead ? 0 : seq) * a.table_stride;
    int *const search = reinterpret_cast<int *>(lds + pa_stream_floats<D, R>());
    PaRows<T, D, R> w;
    PaPages<TILES, KEYS, ROW> pages;
    if (!w.begin(a, ahead, seq, (block * row_waves + wr) * 16 * R, block * row_waves * 16 * R, key0)) return;
    pages.fetch(a, table, key0, key1, wk, key_waves);
    w.fetch(a, ahead, kvh, search);
    if (ahead) __syncthreads();
    w.find(a, ahead, seq, key1, search);
    const int kend = w.last + 1;  // keys key0 .. kend - 1
    const int steps = kend > key0 ? (kend - key0 + KEYS - 1) / KEYS : 0;
    const uint8_t *const kbase = (const uint8_t *)a.k + ((size_t)kvh << a.page_shift) * ROW, *const vbase = (const uint8_t *)a.v + ((size_t)kvh << a.page_shift) * ROW;
    const int koff = n * ROW + 16 * g, voff = 4 * g * ROW + E * n * (int)sizeof(T);
    Tile x;
    auto load_k = [&](int step, int u) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const auto p = pages.tile(a, kbase, key0, kend, step, u, t);
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int s = 0; s < D / 32; ++s) x.k[t][s] = __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(p, koff + 64 * s, 0, 0));
            } else {
#pragma unroll
                for (int s = 0; s < D / 16; ++s) x.k[s] = __builtin_bit_cast(f32x4v, __builtin_amdgcn_raw_buffer_load_b128(p, koff + 64 * s, 0, 0));
            }
        }
    };
    auto load_v = [&](int step, int u) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const auto p = pages.tile(a, vbase, key0, kend, step, u, t);
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

    int step = wk, u = 0;  // u: lane of the ids that holds the pages of `step`
    if (step < steps) {
        pages.check(a, key0, kend, step, key_waves, w.badkey);
        load_k(step, 0);
        load_v(step, 0);
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
        // the keys of the next step, into the registers that the products have read (no branch may stand between the products and the first use of their
        // result: the compiler has been seen to leave out the wait it needs there)
        const int next = step + key_waves;
        load_k(next, (u + 1) & 63);
        const bool partial = base + KEYS - 1 > w.first;  // some row does not see all of them
        if (partial && w.first < w.last) w.clean(x.v, base);  // ... and others see more
        w.weigh(sc, base, partial);
#pragma unroll
        for (int e = 0; e < E; ++e) w.sum(x.v, e);
        u = (u + 1) & 63;
        load_v(next, u);
        step = next;
        if (u == 63 && step + key_waves < steps) pages.look_up(a, table, key0, kend, step + key_waves, key_waves, w.badkey);  // (what is under way has its pages)
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
            lm[wave * 16 * R + 16 * r + n] = w.m[r];
            ll[wave * 16 * R + 16 * r + n] = sum;
        }
    }
    __syncthreads();
    for (int at = tid; at < row_waves * 16 * R * (D / 4); at += PA_THREADS) {
        const int rr = at / (D / 4), e = 4 * (at - rr * (D / 4)), wv = rr / (16 * R), in = rr - wv * 16 * R;  // wave wv + row_waves j holds row `in` of the keys' share j
        const int row = block * row_waves * 16 * R + rr;
        if (row >= w.rows) break;  // (rr grows with at)
        float top = -INFINITY, sum = 0.f;
        f32x4v acc = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < key_waves; ++j) top = fmaxf(top, lm[(wv + row_waves * j) * 16 * R + in]);
        for (int j = 0; j < key_waves; ++j) {
            const int src = (wv + row_waves * j) * 16 * R + in;
            const float mm = lm[src], f = mm > -INFINITY ? __builtin_amdgcn_exp2f(mm - top) : 0.f;
            // (a wave without a key has no weight; one whose rows are to be NaN has, wherever its maximum stands)
            sum += ll[src] == ll[src] ? ll[src] * f : NAN;
            acc += *reinterpret_cast<const f32x4v *>(lo + (size_t)src * (D + 4) + e) * f;
        }
        const int t = w.t0 + row / group, h = kvh * group + row % group;
        if (slots == 1) {
            // (a row that sees nothing is zero)
            const float f = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<f32x4v_a4 *>(a.y + (size_t)t * a.y_stride + (size_t)h * D + e) = acc * f;
        } else {
            const size_t at_slot = ((size_t)t * a.heads + h) * slots + slot;
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
    const int group = a.heads / a.kv;
    __shared__ int last_of[PA_WAVES];
    const int *table = a.tables + (size_t)(ahead ? 0 : seq) * a.table_stride;
    int *const search = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(lds) + W::LDS);
    PaRows<T, D, R> w;
    PaPages<TILES, KEYS, ROW> pages;
    if (!w.begin(a, ahead, seq, (block * PA_WAVES + wave) * 16 * R, block * PA_WAVES * 16 * R, key0)) return;
    pages.fetch(a, table, key0, key1, 0, 1);
    w.fetch(a, ahead, kvh, search);
    if (ahead) __syncthreads();
    w.find(a, ahead, seq, key1, search);
    if (lane == 0) last_of[wave] = w.last;
    __syncthreads();
    int kend = 0;  // keys key0 .. kend - 1: what any row of the workgroup sees
#pragma unroll
    for (int i = 0; i < PA_WAVES; ++i) kend = max(kend, last_of[i] + 1);
    kend = __builtin_amdgcn_readfirstlane(kend);
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
    auto request = [&](auto slot_c, int step, int u) {
        constexpr int S = decltype(slot_c)::value;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int t = TILES == 1 ? 0 : (wave + PA_WAVES * i) * 64 / (16 * PIECES);
            kr[S][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(pages.tile(a, kbase, key0, kend, step, u, t), koff[i], 0, 0));
        }
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
            const int t = TILES == 1 ? 0 : (wave + PA_WAVES * i) * 64 / (16 * PIECES);
            vr[S][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(pages.tile(a, vbase, key0, kend, step, u, t), voff[i], 0, 0));
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
#pragma unroll
        for (int s = 0; s < PIECES / 4; ++s) {
            u32x4 k[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) k[t] = *reinterpret_cast<const u32x4 *>(ks + (size_t)(16 * t + n) * ROW + 16 * pa_piece<PIECES>(4 * s + g, n));
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
#pragma unroll
        for (int e = 0; e < E; ++e) w.sum(v, e);
    };
    // steps s and s + 1 are requested, s is stored, from then on: barrier, request s + 2, store s + 1, product s
    constexpr std::integral_constant<int, 0> c0{};
    constexpr std::integral_constant<int, 1> c1{};
    if (steps > 0) {
        pages.check(a, key0, kend, 0, 1, w.badkey);
        request(c0, 0, 0);
        request(c1, 1, 1);
    }
    w.take(a);
    if (steps > 0) store(c0, 0);
    auto turn = [&](auto mine, auto other, int step) {  // step's registers were `mine`
        if ((step & 63) == 62 && step + 2 < steps) pages.look_up(a, table, key0, kend, step + 2, 1, w.badkey);
        request(mine, step + 2, (step + 2) & 63);
        __syncthreads();
        product(step);
        store(other, (step + 1) & 1);
    };
    for (int step = 0; step < steps; step += 2) {
        turn(c0, c1, step);
        if (step + 1 < steps) turn(c1, c0, step + 1);
    }

    w.spread_badkey();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = w.total(r);
        const int row = w.row0 + 16 * r + n;
        if (row < w.rows) {
            const int t = w.t0 + row / group, h = kvh * group + row % group;
            const size_t at_slot = ((size_t)t * a.heads + h) * slots + slot;
            const float f = slots > 1 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            float *p = (slots > 1 ? a.part + at_slot * D : a.y + (size_t)t * a.y_stride + (size_t)h * D) + 4 * E * g;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < E; e += 4)
                    *reinterpret_cast<f32x4v_a4 *>(p + E * i + e) = f32x4v{w.o[r][e][i], w.o[r][e + 1][i], w.o[r][e + 2][i], w.o[r][e + 3][i]} * f;
            if (slots > 1 && g == 0) *reinterpret_cast<float2 *>(a.stat + 2 * at_slot) = make_float2(w.m[r], sum);
        }
    }
}

template <class T, int D, int R>
__device__ __forceinline__ void pa_attend(const AttnArgs &a, const AttnPart &part, const bool ahead, const int seq, const int block, const int kvh, const int key0,
                                          const int key1, const int slot, const int slots, float *lds) {
    if (part.key_waves == 1) pa_wide<T, D, R>(a, ahead, seq, block, kvh, key0, key1, slot, slots, lds);
    else pa_stream<T, D, R>(a, part, ahead, seq, block, kvh, key0, key1, slot, slots, lds);
}

// The workgroups: `chunk` of the shared positions, as many of the sequences' own, and so on until one kind is used up - the first are bound by the matrix
// cores, the others by memory, and a CU that holds one of each has use for both.  Of one kind, workgroup b takes of unit u = (span, sequence,
// key/value head) the row block b / 8 % blocks, u = b / (8 blocks) * 8 + b % 8: the row blocks of a unit, which read the same keys, run on one XCD
// (workgroups go round the eight) one after the other.
template <class T, int D, int RA, int RO>
__global__ void __launch_bounds__(PA_THREADS, D <= 128 ? 2 : 1) paged_attn_kernel(const AttnArgs a) {
    extern __shared__ __align__(16) float pa_lds[];
    const unsigned kv = (unsigned)a.kv, seqs = (unsigned)a.sequences, chunk = (unsigned)a.chunk, c = blockIdx.x / chunk, in = blockIdx.x - c * chunk;
    const bool own = c < 2 * (unsigned)a.pairs ? (c & 1) != 0 : a.chunks_own > a.chunks_ahead;
    const unsigned b = (c < 2 * (unsigned)a.pairs ? c / 2 : c - (unsigned)a.pairs) * chunk + in;
    const int slots = a.ahead.spans + a.own.spans;
    if (!own) {
        const unsigned per = 8u * (unsigned)a.ahead.blocks, u = b / per * 8 + b % 8;
        if (u >= kv * (unsigned)a.ahead.spans) return;
        const int span = (int)(u / kv), kvh = (int)(u % kv);
        pa_attend<T, D, RA>(a, a.ahead, true, 0, (int)(b % per / 8), kvh, span * a.ahead.span, min((span + 1) * a.ahead.span, a.shared), span, slots, pa_lds);
    } else {
        const unsigned per = 8u * (unsigned)a.own.blocks, u = b / per * 8 + b % 8;
        if (u >= kv * seqs * (unsigned)a.own.spans) return;
        const int kvh = (int)(u % kv), seq = (int)(u / kv % seqs), span = (int)(u / kv / seqs);
        const int key0 = a.shared + span * a.own.span;
        pa_attend<T, D, RO>(a, a.own, false, seq, (int)(b % per / 8), kvh, key0, min(key0 + a.own.span, a.max_len), a.ahead.spans + span, slots, pa_lds);
    }
}

// y of every row (token, head) from its spans, a workgroup per row: groups of D / 4 threads take a span each, all of a group's requested before the
// first is used.  Spans that begin behind the row's position were not written.
constexpr int PA_MERGE = 256;
template <int D>
__global__ void __launch_bounds__(PA_MERGE) paged_merge_kernel(const AttnArgs a) {
    constexpr int LANES = D / 4, GROUPS = PA_MERGE / LANES, U = 8;
    __shared__ float weight[PA_MERGE], top_of[PA_MERGE / 64], sum_of[PA_MERGE / 64];
    __shared__ f32x4v part_of[GROUPS][LANES];
    const int tid = threadIdx.x, wave = tid >> 6, grp = tid / LANES, in = tid - grp * LANES;
    const long long row = blockIdx.x;
    const int t = (int)(row / a.heads), h = (int)(row - (long long)t * a.heads), slots = a.ahead.spans + a.own.spans;
    const RowPlace at = row_place(a.starts, a.lens, a.sequences, t);
    if (at.sequence >= a.sequences || t < a.starts[0]) return;  // behind the last sequence
    const int lim = at.len - at.end + t;
    f32x4v_a4 *y = reinterpret_cast<f32x4v_a4 *>(a.y + (size_t)t * a.y_stride + (size_t)h * D);
    if (lim < 0 || at.len > a.max_len) {
        const float f = at.len > a.max_len ? NAN : 0.f;
        if (grp == 0) y[in] = f32x4v{f, f, f, f};
        return;
    }
    const int first_own = a.ahead.spans;
    const int ahead = min(first_own, a.shared > 0 ? lim / a.ahead.span + 1 : 0), own = lim >= a.shared ? (lim - a.shared) / a.own.span + 1 : 0;
    const int count = ahead + own;  // at most PA_MERGE (paged_attn_plan)
    auto slot_of = [&](int i) { return (size_t)row * slots + (i < ahead ? i : first_own + i - ahead); };
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
    constexpr int R = RA > RO ? RA : RO;
    // (more than 64 KiB must be asked for, once; a refusal shows at the launch)
    static const hipError_t asked = hipFuncSetAttribute((const void *)paged_attn_kernel<T, D, RA, RO>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                        (int)(pa_lds_bytes<T, D, R>() + (2 * PA_SEARCH + 1) * sizeof(int)));
    (void)asked;
    const size_t lds = pa_lds_bytes<T, D, R>() + (a.ahead.spans > 0 && a.sequences <= PA_SEARCH ? (size_t)(2 * a.sequences + 1) * sizeof(int) : 0);
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
