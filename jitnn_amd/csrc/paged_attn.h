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
// FP16 pages: keys and values are operands as they are; queries (scaled so that a row's largest is near 2^13) and weights (times 2^14) go in two FP16
// parts, 22 bits together, so that the result is as good as in FP32.  FP32 pages: the FP32 matrix instruction.
// Sums, maxima and outputs are FP32.
//
// What a row does not see: its scores are masked; values past the last key that any row of the tile sees are cleared, and of those that only some see
// the ones that are not finite, whose rows become NaN (badkey): nothing behind a token reaches it.  The same mark makes NaN of rows whose positions
// lie on a page that the cache does not have.
#pragma once
#include <type_traits>

#include "common.h"
#include "serving.h"

namespace jitnn {

constexpr int PA_THREADS = 256, PA_WAVES = 4;
constexpr int PA_SEARCH = 1024;  // sequences whose starts a workgroup keeps in LDS
constexpr float PA_WEIGHT = 14.f;  // weights are 2^(score - maximum + 14)

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

// LDS of a workgroup: outputs [wave][16 R][D + 4], maxima and sums [wave][16 R], then starts and lens
template <int D, int R>
constexpr size_t pa_lds_floats() {
    return (size_t)PA_WAVES * 16 * R * (D + 4) + 2 * PA_WAVES * 16 * R;
}

template <class T, int D, int R>
__device__ __forceinline__ void pa_attend(const AttnArgs &a, const AttnPart &part, const bool ahead, const int seq, const int block, const int kvh, const int key0,
                                          const int key1, const int slot, const int slots, float *lds) {
    using Tile = PaTile<T, D>;
    constexpr int KEYS = Tile::KEYS, TILES = Tile::TILES, E = Tile::E;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = a.heads / a.kv, key_waves = part.key_waves, row_waves = PA_WAVES / key_waves;
    const int wr = wave & (row_waves - 1), wk = wave / row_waves;
    // ---- this workgroup's rows
    const int *starts = a.starts, *lens = a.lens;
    if (ahead && a.sequences <= PA_SEARCH) {
        int *s = reinterpret_cast<int *>(lds + pa_lds_floats<D, R>());
        for (int i = tid; i <= a.sequences; i += PA_THREADS) s[i] = a.starts[i];
        for (int i = tid; i < a.sequences; i += PA_THREADS) s[a.sequences + 1 + i] = a.lens[i];
        __syncthreads();
        starts = s;
        lens = s + a.sequences + 1;
    }
    const int t0 = ahead ? max(starts[0], 0) : max(starts[seq], 0), t1 = min(ahead ? starts[a.sequences] : starts[seq + 1], a.tokens);
    const int rows = max(t1 - t0, 0) * group, row0 = (block * row_waves + wr) * 16 * R;
    if ((long long)block * row_waves * 16 * R >= rows) return;
    // (the workgroups of a span that no row of the sequence reaches; where there is one span in all, its rows are still to be written)
    if (!ahead && key0 > 0 && lens[seq] <= key0) return;
    int lim[R];  // the last position of the span that a row sees
    bool over[R];
    int last = -1, first = 0x7fffffff;  // of the wave's rows
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
    const int kend = last + 1;  // keys key0 .. kend - 1

    // ---- queries: 8 g + j of each 32 values (FP16), 4 g + j of each 16 (FP32) of row n
    f16x8 qh[R][sizeof(T) == 2 ? D / 32 : 1], ql[R][sizeof(T) == 2 ? D / 32 : 1];
    f32x4v qf[R][sizeof(T) == 4 ? D / 16 : 1];
    float qs[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = min(row0 + 16 * r + n, rows - 1), t = t0 + row / group, h = kvh * group + row % group;
        const float *q = a.q + (size_t)t * a.q_stride + (size_t)h * D;
        if constexpr (sizeof(T) == 2) {
            float x[D / 4];
            float amax = 0.f;
#pragma unroll
            for (int s = 0; s < D / 32; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[8 * s + j] = q[32 * s + 8 * g + j] * a.scale;
                    amax = fmaxf(amax, fabsf(x[8 * s + j]));
                }
            const float f = half_scale(pa_max4(amax));
            qs[r] = 1.f / f;
#pragma unroll
            for (int s = 0; s < D / 32; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = x[8 * s + j] * f;
                    qh[r][s][j] = (_Float16)y;
                    ql[r][s][j] = (_Float16)(y - (float)qh[r][s][j]);
                }
        } else {
            qs[r] = 1.f;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) qf[r][s][j] = q[16 * s + 4 * g + j] * a.scale;
        }
    }

    f32x4v o[R][E];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
    int badkey = 0x7fffffff;  // rows that see this position are NaN

    // ---- the wave's steps: KEYS keys each, every key_waves-th of the span.  Loads are in buffer form, a descriptor per tile of 16 keys: its extent
    // ends behind the last key, so that what lies behind reads as zero without a branch or a mask, and a tile that does not exist (behind the last key,
    // behind the last step, on a page that the cache does not have) costs nothing.
    const int steps = kend > key0 ? (kend - key0 + KEYS - 1) / KEYS : 0;
    const int *table = a.tables + (size_t)(ahead ? 0 : seq) * a.table_stride;
    constexpr int ROW = D * (int)sizeof(T);  // bytes of a key
    const size_t page_bytes = ((size_t)a.kv << a.page_shift) * ROW;
    const int in_page = (1 << a.page_shift) - 1;
    const uint8_t *const kbase = (const uint8_t *)a.k + ((size_t)kvh << a.page_shift) * ROW, *const vbase = (const uint8_t *)a.v + ((size_t)kvh << a.page_shift) * ROW;
    const int koff = n * ROW + 16 * g, voff = 4 * g * ROW + E * n * (int)sizeof(T);
    int ids[TILES];  // lane u: the pages of step `first of the 64` + u, -1: none
    auto look_up = [&](int step0) {
        int bad = 0x7fffffff;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int key = key0 + (step0 + lane * key_waves) * KEYS + 16 * t;
            ids[t] = -1;
            if (step0 + lane * key_waves < steps && key < kend) {
                ids[t] = table[key >> a.page_shift];
                if ((unsigned)ids[t] >= (unsigned)a.pages) {
                    bad = min(bad, key);
                    ids[t] = -1;
                }
            }
        }
        if (__ballot(bad != 0x7fffffff)) {
            for (int off = 1; off < 64; off <<= 1) bad = min(bad, __shfl_xor(bad, off));
            badkey = min(badkey, bad);
        }
    };
    Tile x;
    auto source = [&](const uint8_t *pages, int step, int u, int t) {
        const int key = key0 + step * KEYS + 16 * t, id = __builtin_amdgcn_readlane(ids[t], u);
        const size_t at = (size_t)(id < 0 ? 0 : id) * page_bytes + (size_t)(key & in_page) * ROW;
        return __builtin_amdgcn_make_buffer_rsrc((void *)(pages + at), 0, id < 0 ? 0 : max(min(kend - key, 16), 0) * ROW, 0x00020000);
    };
    auto load_k = [&](int step, int u) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const auto p = source(kbase, step, u, t);
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
            const auto p = source(vbase, step, u, t);
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

    int step = wk, u = 0;  // u: lane of ids that holds the pages of `step`
    if (step < steps) {
        look_up(step);
        load_k(step, 0);
        load_v(step, 0);
    }
    while (step < steps) {
        const int base = key0 + step * KEYS;
        // ---- scores: sc[r][t][i] of row n, key base + 16 t + 4 g + i
        f32x4v sc[R][TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                f32x4v c = {0.f, 0.f, 0.f, 0.f};
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int s = 0; s < D / 32; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[t][s], ql[r][s], c, 0, 0, 0);
#pragma unroll
                    for (int s = 0; s < D / 32; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[t][s], qh[r][s], c, 0, 0, 0);
                } else {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[s][j], qf[r][s][j], c, 0, 0, 0);
                }
                sc[r][t] = c;
            }
        // the keys of the next step, into the registers that the products have read
        const int next = step + key_waves;
        load_k(next, (u + 1) & 63);
        const bool partial = base + KEYS - 1 > first;  // some row does not see all of them
        if (partial && first < last) {                 // ... and others see more
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bool fine = true;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const bool f = pa_finite(x.v[t][i][e]);
                        fine = fine && f;
                        if (!f) x.v[t][i][e] = (T)0.f;
                    }
                    if (!fine) badkey = min(badkey, base + 16 * t + 4 * g + i);
                }
        }
        f16x8 ph[R], pl[R];  // (FP16) slot 4 t + i
        float pf[R][4];      // (FP32)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float s = sc[r][t][i];
                    if constexpr (sizeof(T) == 2) s *= qs[r];
                    if (partial) s = base + 16 * t + 4 * g + i <= lim[r] ? s : -INFINITY;
                    sc[r][t][i] = s;
                    top = fmaxf(top, s);
                }
            top = fmaxf(m[r], pa_max4(top));
            if (__ballot(top > m[r])) {  // the sums so far are in units of an older maximum
                const float f = top > -INFINITY ? __builtin_amdgcn_exp2f(m[r] - top) : 1.f;
                l[r] *= f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[r][e] *= f;
                m[r] = top;
            }
            const float less = top > -INFINITY ? PA_WEIGHT - top : 0.f;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(sc[r][t][i] + less);
                    l[r] += p;
                    if constexpr (sizeof(T) == 2) {
                        ph[r][4 * t + i] = (_Float16)p;
                        pl[r][4 * t + i] = (_Float16)(p - (float)ph[r][4 * t + i]);
                    } else {
                        pf[r][i] = p;
                    }
                }
        }
        // ---- o[r][e][i]: value E (4 g + i) + e of row n
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (sizeof(T) == 2) {
                f16x8 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = x.v[0][i][e];
                    v[4 + i] = x.v[TILES - 1][i][e];
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    o[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[r], o[r][e], 0, 0, 0);
                    o[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[r], o[r][e], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[0][i][e], pf[r][i], o[r][e], 0, 0, 0);
            }
        }
        u = (u + 1) & 63;
        load_v(next, u);
        step = next;
        if (u == 63 && step + key_waves < steps) look_up(step + key_waves);  // (what is under way has its pages)
    }

    // ---- the waves' sums meet in LDS
    for (int off = 1; off < 64; off <<= 1) badkey = min(badkey, __shfl_xor(badkey, off));
    float *const lo = lds, *const lm = lds + (size_t)PA_WAVES * 16 * R * (D + 4), *const ll = lm + PA_WAVES * 16 * R;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float *p = lo + (size_t)(wave * 16 * R + 16 * r + n) * (D + 4) + 4 * E * g;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < E; e += 4) *reinterpret_cast<f32x4v *>(p + E * i + e) = f32x4v{o[r][e][i], o[r][e + 1][i], o[r][e + 2][i], o[r][e + 3][i]};
        float sum = pa_sum4(l[r]);
        if (over[r] || lim[r] >= badkey) sum = NAN;
        if (g == 0) {
            lm[wave * 16 * R + 16 * r + n] = m[r];
            ll[wave * 16 * R + 16 * r + n] = sum;
        }
    }
    __syncthreads();
    for (int at = tid; at < row_waves * 16 * R * (D / 4); at += PA_THREADS) {
        const int rr = at / (D / 4), e = 4 * (at - rr * (D / 4)), w = rr / (16 * R), in = rr - w * 16 * R;  // wave w + row_waves j holds row `in` of the keys' share j
        const int row = block * row_waves * 16 * R + rr;
        if (row >= rows) break;  // (rr grows with at)
        float top = -INFINITY, sum = 0.f;
        f32x4v acc = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < key_waves; ++j) top = fmaxf(top, lm[(w + row_waves * j) * 16 * R + in]);
        for (int j = 0; j < key_waves; ++j) {
            const int src = (w + row_waves * j) * 16 * R + in;
            const float mm = lm[src], f = mm > -INFINITY ? __builtin_amdgcn_exp2f(mm - top) : 0.f;
            // (a wave without a key has no weight; one whose rows are to be NaN has, wherever its maximum stands)
            sum += ll[src] == ll[src] ? ll[src] * f : NAN;
            acc += *reinterpret_cast<const f32x4v *>(lo + (size_t)src * (D + 4) + e) * f;
        }
        const int t = t0 + row / group, h = kvh * group + row % group;
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

// The workgroups: first those of the shared positions, then the sequences' own.  Of one part, workgroup b takes of unit u = (span, sequence, key/value
// head) the row block b / 8 % blocks, u = b / (8 blocks) * 8 + b % 8: the row blocks of a unit, which read the same keys, run on one XCD
// (workgroups go round the eight) one after the other.
template <class T, int D, int RA, int RO>
__global__ void __launch_bounds__(PA_THREADS, D <= 128 ? 2 : 1) paged_attn_kernel(const AttnArgs a) {
    extern __shared__ __align__(16) float pa_lds[];
    unsigned b = blockIdx.x;
    const unsigned units_ahead = (unsigned)(a.ahead.spans * a.kv), blocks_ahead = (units_ahead + 7) / 8 * 8 * (unsigned)a.ahead.blocks;
    const int slots = a.ahead.spans + a.own.spans;
    if (b < blocks_ahead) {
        const unsigned per = 8u * (unsigned)a.ahead.blocks, u = b / per * 8 + b % 8;
        if (u >= units_ahead) return;
        const int span = (int)(u / (unsigned)a.kv), kvh = (int)(u % (unsigned)a.kv);
        pa_attend<T, D, RA>(a, a.ahead, true, 0, (int)(b % per / 8), kvh, span * a.ahead.span, min((span + 1) * a.ahead.span, a.shared), span, slots, pa_lds);
    } else {
        b -= blocks_ahead;
        const unsigned per = 8u * (unsigned)a.own.blocks, u = b / per * 8 + b % 8, kv = (unsigned)a.kv, seqs = (unsigned)a.sequences;
        if (u >= kv * seqs * (unsigned)a.own.spans) return;
        const int kvh = (int)(u % kv), seq = (int)(u / kv % seqs), span = (int)(u / kv / seqs);
        const int key0 = a.shared + span * a.own.span;
        pa_attend<T, D, RO>(a, a.own, false, seq, (int)(b % per / 8), kvh, key0, min(key0 + a.own.span, a.max_len), a.ahead.spans + span, slots, pa_lds);
    }
}

// y of every row from its spans: a wave per row (token, head), D / 64 values a lane.  Spans that begin behind the row's position were not written.
template <int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const AttnArgs a) {
    constexpr int V = D / 64, U = 8;
    const int lane = threadIdx.x & 63;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (long long)a.tokens * a.heads) return;
    const int t = (int)(row / a.heads), h = (int)(row - (long long)t * a.heads), slots = a.ahead.spans + a.own.spans;
    int s = 0;
    for (int i = lane; i < ((a.sequences + 63) & ~63); i += 64) s += __popcll(__ballot(i < a.sequences && a.starts[i + 1] <= t));
    if (s >= a.sequences || t < a.starts[0]) return;  // behind the last sequence
    const int len = a.lens[s], lim = len - a.starts[s + 1] + t;
    float *y = a.y + (size_t)t * a.y_stride + (size_t)h * D + V * lane;
    if (lim < 0 || len > a.max_len) {
        const float f = len > a.max_len ? NAN : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = f;
        return;
    }
    const int first_own = a.ahead.spans;
    const int ahead = min(first_own, a.shared > 0 ? lim / a.ahead.span + 1 : 0), own = lim >= a.shared ? (lim - a.shared) / a.own.span + 1 : 0;
    const int count = ahead + own;
    auto slot_of = [&](int i) { return (size_t)row * slots + (i < ahead ? i : first_own + i - ahead); };
    float m = -INFINITY;
    for (int i = lane; i < count; i += 64) m = fmaxf(m, a.stat[2 * slot_of(i)]);
    m = wave_max(m);
    float sum = 0.f, acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
    for (int i0 = 0; i0 < count; i0 += U) {
        float mm[U], ss[U], x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t at = slot_of(min(i0 + u, count - 1));
            mm[u] = a.stat[2 * at];
            ss[u] = a.stat[2 * at + 1];
#pragma unroll
            for (int v = 0; v < V; ++v) x[u][v] = a.part[at * D + V * lane + v];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u < count) {
                const float f = mm[u] > -INFINITY ? __builtin_amdgcn_exp2f(mm[u] - m) : 0.f;
                sum += ss[u] == ss[u] ? ss[u] * f : NAN;
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf(x[u][v], f, acc[v]);
            }
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = acc[v] * f;
}

// ---- launch

template <class T, int D, int RA, int RO>
static void paged_attn_run(unsigned blocks, hipStream_t s, const AttnArgs &a) {
    constexpr int R = RA > RO ? RA : RO;
    // (more than 64 KiB must be asked for, once; a refusal shows at the launch)
    static const hipError_t asked = hipFuncSetAttribute((const void *)paged_attn_kernel<T, D, RA, RO>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                        (int)(pa_lds_floats<D, R>() * sizeof(float) + (2 * PA_SEARCH + 1) * sizeof(int)));
    (void)asked;
    const size_t lds = pa_lds_floats<D, R>() * sizeof(float) + (a.ahead.spans > 0 && a.sequences <= PA_SEARCH ? (size_t)(2 * a.sequences + 1) * sizeof(int) : 0);
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
