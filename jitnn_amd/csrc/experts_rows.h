// The experts' products of many (token, expert) pairs on the matrix cores, at FP32-grade accuracy: gemv_rows_kernel's operands and decoders (gemv_rows.h), for
// rows that a list gathers.
//
// The operands of an activation row are prepared once, row by row (experts_prepare_unit: FP16 hi and lo parts of the row scaled per 256 values, and the sums of
// its blocks), whoever it will meet: which eight rows stand in one matrix operand, the lists of the experts say when the operand is put together in LDS.
// A workgroup takes one expert, up to eight times `groups` of its rows and 8 waves x T tiles of 16 weight rows; all its waves are at the same 256 values of K, so that
// the operands cross from L2 to LDS once for the eight of them, while every weight byte is read by one wave only, decoded once and kept in registers for all
// the groups.  Nothing is added up across waves or workgroups but shares of K (a.splits), which whoever reads
// them adds up in order, and a row's result does not depend on the rows beside it.
// Bound by what turns quants into operands - vector units 53 (Q4_K) to 66 % (Q5_K, Q6_K) busy for chunks of up to sixteen rows: with every expert's weights in the caches
// 32 tokens over 128 experts took 122 us instead of 139, 24 over eight 227 instead of 274 (260 since) -, by operands and products in turn for more (see the shapes).
#pragma once
#include <utility>

#include "act.h"
#include "common.h"
#include "experts.h"
#include "gemv_rows.h"
#include "row_end.h"

namespace jitnn {

constexpr int ER_OP_CHUNKS = 72;                      // 16-byte pieces of a row's operands of one column: [8 blocks and the sums][hi, lo][lane group]
constexpr int ER_OP_BYTES = ER_OP_CHUNKS * 16;

// A workgroup's shape: its waves, the groups of eight rows whose operands are in LDS at a time, how many such sets a chunk has at most, and waves per SIMD that the registers
// are to leave room for.
template <int WAVES, int GS, int SETS, int PER_SIMD>
struct RowsShape {
    static constexpr int waves = WAVES, threads = 64 * WAVES, gs = GS, sets = SETS, groups = GS * SETS, per_simd = PER_SIMD;
    static constexpr int set_rows = 8 * GS, all_rows = 8 * groups, set_chunks = GS * 9 * 64;  // (set_chunks: pieces of a set's operands)
};
// Tiles of 16 weight rows that a wave holds: two share the operands that cross LDS; one of Q6_K, which has sixteen operands a tile where the others have eight, and where 128
// registers have to do.
template <int FMT, class S>
__host__ __device__ constexpr int er_tiles() { return RTile<FMT>::NOPS > 8 || S::per_simd > 2 ? 1 : 2; }
template <int FMT, class S>
__host__ __device__ constexpr size_t experts_rows_lds() {
    constexpr size_t ops = (size_t)2 * (S::set_chunks * 16 + S::set_rows * sizeof(float)), gated = er_tiles<FMT, S>() == 1 ? (size_t)S::waves / 2 * S::groups * 64 * sizeof(float2) : 0;
    return (ops > gated ? ops : gated) + (size_t)S::all_rows * 2 * sizeof(int) + (size_t)S::waves * er_tiles<FMT, S>() * RTile<FMT>::STAGE_BYTES;
}

__device__ __forceinline__ f32x4 mfma(const f16x8 &x, const f16x8 &w, const f32x4 &c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w, c, 0, 0, 0); }
// Sum v of a lane's two: the hi and lo parts' side by side
__device__ __forceinline__ float joined(const f32x4 &c, int v) { return c[2 * v] + c[2 * v + 1]; }
template <class F, int... I>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F &&f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F &&f) { each_of(std::make_integer_sequence<int, N>{}, f); }

// Column c of eight rows, as rows_prepare_column, in pieces of a row: operand s (block s of the column; 8: the sums), part and lane group kq at
// 16-byte piece 8 s + 4 part + kq.  v: the lane's quads (zeros behind the row's last value).
template <int GS, bool HALVES>
__device__ __forceinline__ void experts_prepare_column(const float4 (&v)[8], uint8_t *__restrict__ op, float *__restrict__ inv, bool have, int part) {
    float amax = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v[t].x), fabsf(v[t].y)), fmaxf(fabsf(v[t].z), fabsf(v[t].w))));
    amax = group_max8(amax);
    const float scale = half_scale(amax);
    const int kq = HALVES ? part & 3 : part >> 1, h = HALVES ? part >> 2 : part & 1;
    float sm = 0.f, sm2 = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const float a0 = v[t].x * scale, a1 = v[t].z * scale, a2 = v[t].y * scale, a3 = v[t].w * scale;  // (the decoders' order of a dword's bytes)
        const float qs = (a0 + a1) + (a2 + a3);
        if constexpr (GS == 32) {
            const float bs = group_sum<8>(qs);
            sm = part == t ? bs : sm;
        } else {
            const float lo = group_sum<8>(part < 4 ? qs : 0.f), hi = group_sum<8>(part < 4 ? 0.f : qs);
            const float mine = (part & 1) ? hi : lo;
            sm = (part >> 1) == t ? mine : sm;
            sm2 = 4 + (part >> 1) == t ? mine : sm2;
        }
        const h2raw h01 = __builtin_amdgcn_cvt_pkrtz(a0, a1), h23 = __builtin_amdgcn_cvt_pkrtz(a2, a3);
        const h2raw l01 = __builtin_amdgcn_cvt_pkrtz(a0 - (float)h01.x, a1 - (float)h01.y);
        const h2raw l23 = __builtin_amdgcn_cvt_pkrtz(a2 - (float)h23.x, a3 - (float)h23.y);
        if (have) {
            *reinterpret_cast<u32x2 *>(op + t * 128 + kq * 16 + 8 * h) = u32x2{__builtin_bit_cast(uint32_t, h01), __builtin_bit_cast(uint32_t, h23)};
            *reinterpret_cast<u32x2 *>(op + t * 128 + 64 + kq * 16 + 8 * h) = u32x2{__builtin_bit_cast(uint32_t, l01), __builtin_bit_cast(uint32_t, l23)};
        }
    }
    // the sums of the blocks / 64 (a sum of 32 values below 2^14 stays below 2^13): lane `part` of the row has that of block `part`.  Blocks of 16 values:
    // the upper eight in lane group 1; HALVES: times 4 in lane groups 1 and 2 (RTile<F_Q4_1>); zeros elsewhere
    auto put = [&](int group, _Float16 hi, _Float16 lo) {
        reinterpret_cast<_Float16 *>(op + 8 * 128 + group * 16)[part] = hi;
        reinterpret_cast<_Float16 *>(op + 8 * 128 + 64 + group * 16)[part] = lo;
    };
    sm *= 0.015625f;
    sm2 *= 0.015625f;
    const _Float16 shi = (_Float16)sm, slo = (_Float16)(sm - (float)shi), thi = (_Float16)sm2, tlo = (_Float16)(sm2 - (float)thi), zero = (_Float16)0.f, four = (_Float16)4.f;
    if (have) {
        put(0, shi, slo);
        put(1, GS == 16 ? thi : HALVES ? shi * four : zero, GS == 16 ? tlo : HALVES ? slo * four : zero);
        put(2, HALVES ? shi * four : zero, HALVES ? slo * four : zero);
        put(3, zero, zero);
        if (part == 0) *inv = 1.f / scale;
    }
}

// One wave's unit: a column of eight rows.
__device__ __forceinline__ void experts_prepare_unit(const ExpertPrepare &p, int unit, int lane) {
    const int b = lane >> 3, part = lane & 7, ncol = (p.k + 255) >> 8, octet = unit / ncol, c = unit - octet * ncol, row = octet * 8 + b;
    const bool have = row < p.rows;
    const float *xr = p.x + (size_t)(have ? row : 0) * p.k;
    float4 v[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const int at = c * 256 + 32 * t + 4 * part;
        v[t] = at < p.k ? *reinterpret_cast<const float4 *>(xr + at) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const size_t at = (size_t)row * ncol + c;
    if (p.ops[0]) experts_prepare_column<32, false>(v, p.ops[0] + at * ER_OP_BYTES, p.inv[0] + at, have, part);
    if (p.ops[1]) experts_prepare_column<16, false>(v, p.ops[1] + at * ER_OP_BYTES, p.inv[1] + at, have, part);
    if (p.ops[2]) experts_prepare_column<32, true>(v, p.ops[2] + at * ER_OP_BYTES, p.inv[2] + at, have, part);
}

// Sixteen bytes of which those from `end` on are zero and not read: the sixteen in front of `end`, moved down (there are as many: a matrix is no smaller).
__device__ __forceinline__ u32x4 ld128_until(const uint8_t *p, const uint8_t *end) {
    const int behind = bytes_behind((long long)(p - end) + 16);
    const u32x4 v = ld128<2>(p - behind);
    const Halves h = moved_down({(unsigned long long)v.y << 32 | v.x, (unsigned long long)v.w << 32 | v.z}, behind);
    return u32x4{(uint32_t)h.lo, (uint32_t)(h.lo >> 32), (uint32_t)h.hi, (uint32_t)(h.hi >> 32)};
}

// The last column of rows that are no whole columns (32-value blocks): what lies behind a row's last block is the next row, behind the last row nobody's.
template <class R>
__device__ __forceinline__ void load_last_column(typename R::Raw &r, const typename R::Ptr &p, int c, const uint8_t *end) {
    const uint8_t *q = p.full + (size_t)c * R::BYTES;
#pragma unroll
    for (int i = 0; i < R::FULL; ++i) r.c[i] = ld128_until(q + 64 * i, end);
    if constexpr (R::REST > 0) r.c[R::FULL] = ld128_until(q + p.rest, end);
}

// grid: a.nblocks x a.splits x (at least as many as there are chunks); experts_rows_lds() of dynamic LDS, chunks of at most S::all_rows rows.
// DUAL: y = act(gate x) * (up x), a wave having a tile of each, or the one or the other, waves 2 i and 2 i + 1 the same rows of the two.  Otherwise a split takes its share
// of the columns and has a y of its own.
template <int FMT, class S, bool DUAL>
__global__ void __launch_bounds__(S::threads, S::per_simd) experts_rows_kernel(const ExpertRowsArgs a) {
    typedef RTile<FMT> R;
    constexpr int NOPS = R::NOPS, T = er_tiles<FMT, S>(), NI = S::set_chunks / S::threads + 1, V = 2;  // (V: sums that a lane has of a tile and a group)
    constexpr int CHAINS = R::BLOCK_SCALES ? 1 : NOPS / 8;  // sums of a tile and a group that products add to: two in turn where there are as many operands
    constexpr int AHEAD = S::sets > 1 ? 4 : 8;  // operands that come out of LDS ahead of their products (one set: a group's all at once)
    constexpr bool PARTIAL = R::BLOCK_SCALES;  // (only 32-value blocks have rows that are no whole columns)
    extern __shared__ __attribute__((aligned(16))) uint8_t er_smem[];
    uint8_t *stage = er_smem;                                                                    // per wave: T tiles' bytes of a column
    uint32_t *const where = reinterpret_cast<uint32_t *>(er_smem + (size_t)S::waves * T * R::STAGE_BYTES);  // [all_rows] a row's operands, in bytes from the first one's
    int *const slots = reinterpret_cast<int *>(where + S::all_rows);                             // [all_rows]
    u32x4 *const ops = reinterpret_cast<u32x4 *>(slots + S::all_rows);                           // [2][gs][9][64]
    float *const invs = reinterpret_cast<float *>(ops + (size_t)2 * S::set_chunks);              // [2][set_rows]
    const int tid = threadIdx.x, lane = tid & 63, kq = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    stage += (size_t)wave * T * R::STAGE_BYTES;
    const int per_chunk = a.nblocks * a.splits, u = (int)blockIdx.x / per_chunk, of_chunk = (int)blockIdx.x - u * per_chunk, split = of_chunk / a.nblocks,
              block = of_chunk - split * a.nblocks;
    if (u >= a.chunks->x) return;
    const int4 ch = a.chunks[1 + u];  // expert, place of its first row in the list, rows
    const int ncol = (a.k + 255) >> 8, groups = (ch.z + 7) >> 3, sets = (groups + S::gs - 1) / S::gs;
    const int c0 = (int)((long long)ncol * split / a.splits), c1 = (int)((long long)ncol * (split + 1) / a.splits);

    const int slot = a.list[ch.y + min(min(tid, S::all_rows - 1), ch.z - 1)];  // (a place without a row takes the last one again: computed, not stored)
    static_assert(S::all_rows <= S::threads, "a thread for each row");
    // the weights on their way: the first column of this wave's tiles
    const size_t rowbytes = (size_t)(a.k / block_values(FMT)) * block_bytes(FMT);
    const uint8_t *const w0 = a.w + (size_t)ch.x * a.expert_bytes, *const w1 = DUAL ? a.w2 + (size_t)ch.x * a.expert_bytes : w0;
    const int ntiles = a.n >> 4, first = block * S::waves + wave;
    const int tile = DUAL ? (T == 2 ? first : first >> 1) : first * T;  // of this wave (T 2 without DUAL: and the next one)
    const bool second = DUAL && T == 1 && (wave & 1);                   // a wave with a tile of up
    const uint8_t *const end0 = a.w + (size_t)a.experts * a.expert_bytes, *const end1 = DUAL ? a.w2 + (size_t)a.experts * a.expert_bytes : end0;
    typename R::Ptr ptr[T];
    typename R::Raw raw[T];
#pragma unroll
    for (int t = 0; t < T; ++t) ptr[t] = R::ptr(second || (DUAL && t) ? w1 : w0, min(DUAL ? tile : tile + t, ntiles - 1) * 16, rowbytes, lane);
    const int last_blocks = PARTIAL ? (a.k & 255) >> 5 : 0;  // of the last column, where it is none of eight
    auto fetch = [&](int c) {
        if (PARTIAL && last_blocks && c == ncol - 1) {
#pragma unroll
            for (int t = 0; t < T; ++t) load_last_column<R>(raw[t], ptr[t], c, second || (DUAL && t) ? end1 : end0);
            return;
        }
#pragma unroll
        for (int t = 0; t < T; ++t) R::load(raw[t], ptr[t], c);
    };
    fetch(c0);
    if (tid < S::all_rows) {
        slots[tid] = slot;
        where[tid] = (uint32_t)(slot / a.per_row) * (uint32_t)ncol * (uint32_t)ER_OP_BYTES;
    }
    __syncthreads();
    // Piece i of this thread: lane l of operand s of group g of a set, whose row is that of l's place.  What the whole rounds leave is shared out over the waves, a few
    // lanes each, the others doing what the last of those does; and a group that the chunk has not is the last row's again: no load stands behind a condition,
    // for at the end of one the compiler waits for what was asked for before it.
    constexpr int ROUNDS = NI - 1, SHARE = (S::set_chunks - ROUNDS * S::threads) / S::waves;
    static_assert(SHARE >= 1 && SHARE <= 64 && SHARE * S::waves == S::set_chunks - ROUNDS * S::threads, "whole lanes");
    uint32_t from[NI];   // one set: where it stands in column 0; several: of the row in its set | where in the row's operands << 16
    int to[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int idx = i < ROUNDS ? tid + i * S::threads : ROUNDS * S::threads + wave * SHARE + min(lane, SHARE - 1);
        const int g = idx / (9 * 64), rest = idx - g * (9 * 64), s = rest >> 6, l = rest & 63;
        const uint32_t row = (uint32_t)(g * 8 + ((l & 15) >> 1)), piece = (uint32_t)(s * 128 + (l & 1) * 64 + (l >> 4) * 16);
        from[i] = S::sets == 1 ? where[row] + piece : row | piece << 16;
        to[i] = idx;
    }
    const int inv_row = min(tid, S::set_rows - 1);
    const uint32_t inv_from = where[inv_row] / (uint32_t)(ER_OP_BYTES / 4);
    u32x4 next[NI];
    float next_inv;
    auto ask = [&](int c, int set) {
        const uint32_t column = (uint32_t)c * ER_OP_BYTES;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const uint32_t at = S::sets == 1 ? from[i] : where[set * S::set_rows + (from[i] & 0xffffu)] + (from[i] >> 16);
            next[i] = *reinterpret_cast<const u32x4 *>(a.ops + (at + column));
        }
        const uint32_t at = S::sets == 1 ? inv_from : where[set * S::set_rows + inv_row] / (uint32_t)(ER_OP_BYTES / 4);
        next_inv = *reinterpret_cast<const float *>(reinterpret_cast<const uint8_t *>(a.inv) + (at + 4u * (uint32_t)c));
    };
    ask(c0, 0);

    float acc[T][S::groups][V];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int g = 0; g < S::groups; ++g)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[t][g][v] = 0.f;
    int buffer = 0;
    // A set's operands into the buffer that nobody reads any more: every wave has passed the barrier of the set before, behind its products of the one before that.
    auto put = [&]() {
        u32x4 *const op = ops + (size_t)buffer * S::set_chunks;
#pragma unroll
        for (int i = 0; i < NI; ++i) op[to[i]] = next[i];
        if (tid < S::set_rows) invs[buffer * S::set_rows + tid] = next_inv;
        buffer ^= 1;
    };
    for (int c = c0; c < c1; ++c) {
        f16x8 B[T][NOPS], Bm[T];
        float d[T], dmin64[T], dblk[R::BLOCK_SCALES ? T : 1][8];
        const uint8_t *row[T];
        uint32_t tail[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            row[t] = R::park(raw[t], stage + t * R::STAGE_BYTES, lane);
            tail[t] = raw[t].tail;
        }
        put();  // (in front of the request for the next weights: loads come back in order, and a wait for these would be one for those)
        if (c + 1 < c1) fetch(c + 1);
        auto decode = [&](int t) {
            if constexpr (R::BLOCK_SCALES) {
                R::decode(row[t], tail[t], lane, B[t], Bm[t], dblk[t]);
                if (PARTIAL && last_blocks && c == ncol - 1) {  // (their operands are zero, what stands there need not be a number)
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        dblk[t][s] = s < last_blocks ? dblk[t][s] : 0.f;
                        Bm[t][s] = s < last_blocks ? Bm[t][s] : (_Float16)0.f;
                    }
                }
            } else {
                float dm;
                R::decode(row[t], tail[t], lane, B[t], Bm[t], d[t], dm);
                dmin64[t] = dm * 64.f;
            }
        };
#pragma unroll
        for (int t = 0; t < T; ++t) decode(t);
        // (sets and groups by their number at compile time: sums that a loop indexes are kept in memory)
        each<S::sets>([&](auto set_) {
            constexpr int set = decltype(set_)::value;
            if (set >= sets) return;
            if (set > 0) put();
            const u32x4 *const op = ops + (size_t)(buffer ^ 1) * S::set_chunks;
            const float *const iv = invs + (buffer ^ 1) * S::set_rows;
            const bool more = set + 1 < sets;
            ask(more ? c : min(c + 1, c1 - 1), more ? set + 1 : 0);  // (behind the last one: that one again)
            __syncthreads();
            constexpr int N = S::gs * 9;
            f16x8 A[AHEAD + 1];
#pragma unroll
            for (int i = 0; i < AHEAD && S::sets > 1; ++i) A[i] = __builtin_bit_cast(f16x8, op[i * 64 + lane]);
            each<S::gs>([&](auto gi_) {
                constexpr int gi = decltype(gi_)::value, g = set * S::gs + gi;
                if (g >= groups) return;
                const float2 w2 = *reinterpret_cast<const float2 *>(iv + gi * 8 + 2 * kq);
                const float w[V] = {w2.x, w2.y};
                f32x4 cs[T][CHAINS], cm[T];
                float u[T][V];
#pragma unroll
                for (int t = 0; t < T; ++t) {
#pragma unroll
                    for (int i = 0; i < CHAINS; ++i) cs[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int v = 0; v < V; ++v) u[t][v] = 0.f;
                }
                if constexpr (S::sets == 1) {
#pragma unroll
                    for (int s = 0; s < 9; ++s) A[s] = __builtin_bit_cast(f16x8, op[(gi * 9 + s) * 64 + lane]);
                }
                each<9>([&](auto s_) {
                    constexpr int s = decltype(s_)::value, at = gi * 9 + s;
                    if constexpr (S::sets > 1 && at + AHEAD < N) A[(at + AHEAD) % (AHEAD + 1)] = __builtin_bit_cast(f16x8, op[(at + AHEAD) * 64 + lane]);
                    const f16x8 x = A[S::sets > 1 ? at % (AHEAD + 1) : s];
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        if constexpr (s == 8) {
                            if constexpr (R::MINS || !R::BLOCK_SCALES) cm[t] = mfma16(x, Bm[t]);
                        } else if constexpr (R::BLOCK_SCALES) {
                            const f32x4 block = mfma16(x, B[t][s]);
#pragma unroll
                            for (int v = 0; v < V; ++v) u[t][v] = __builtin_fmaf(dblk[t][s], joined(block, v), u[t][v]);
                        } else {
                            each<NOPS / 8>([&](auto q) {
                                constexpr int i = decltype(q)::value, w = s * (NOPS / 8) + i;
                                static_assert(R::aidx(w) == s, "the weights' operands of one of the activations'");
                                cs[t][i] = mfma(x, B[t][w], cs[t][i]);
                            });
                        }
                    }
                    if constexpr (S::sets > 1) __builtin_amdgcn_sched_barrier(0);
                });
#pragma unroll
                for (int t = 0; t < T; ++t) {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        if constexpr (R::BLOCK_SCALES) {
                            if constexpr (R::MINS) u[t][v] = __builtin_fmaf(64.f, joined(cm[t], v), u[t][v]);
                        } else {
                            const f32x4 all = CHAINS > 1 ? cs[t][0] + cs[t][CHAINS - 1] : cs[t][0];
                            u[t][v] = __builtin_fmaf(d[t], joined(all, v), -dmin64[t] * joined(cm[t], v));
                        }
                        acc[t][g][v] = __builtin_fmaf(w[v], u[t][v], acc[t][g][v]);
                    }
                }
                // (the operands and products of one group at a time: of more than one there are no registers)
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int v = 0; v < V; ++v) asm volatile("" : "+v"(acc[t][g][v]));
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    }
    float *const y0 = a.y + (DUAL ? 0 : (size_t)split * a.split_floats);
    float *const other = reinterpret_cast<float *>(ops) + ((size_t)(wave >> 1) * S::groups * 64 + lane) * V;
    if constexpr (DUAL && T == 1) {
        __syncthreads();
        if (second) {
#pragma unroll
            for (int g = 0; g < S::groups; ++g)
#pragma unroll
                for (int v = 0; v < V; ++v) other[g * 64 * V + v] = acc[0][g][v];
        }
        __syncthreads();
        if (second) return;
    }
#pragma unroll
    for (int g = 0; g < S::groups; ++g) {
        if (g >= groups) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int b = g * 8 + V * kq + v;
            if (b >= ch.z) continue;
            float *const y = y0 + (size_t)slots[b] * a.n + (lane & 15);
            const float v0 = acc[0][g][v], v1 = DUAL && T == 1 ? other[g * 64 * V + v] : acc[T - 1][g][v];
            if (tile < ntiles) y[tile * 16] = DUAL ? activate(a.act, v0) * v1 : v0;
            if (!DUAL && T == 2 && tile + 1 < ntiles) y[tile * 16 + 16] = v1;
        }
    }
}

// The shapes, by the groups of a chunk.
// One: 32 tokens of which each meets eight of 128 experts, gate and up of 2048 x 768 / down: workgroups of eight waves 64 us in Q4_K and 62 in Q6_K, of four 82 and 62; formats of
// 32-value blocks, whose scales take registers, the other way round (five tokens, six of 64 experts of 2048 x 1408 in Q8_0 82 and 34 against 64 and 32).
// Two: with a tile a wave 128 registers do, and a CU has sixteen waves (24 tokens, two of eight experts of 4096 x 14336 in Q5_K 317 -> 266 us); where they do not - Q6_K, 32-value
// blocks but Q4_0 -, four waves of two tiles (of one of Q6_K) (24 tokens, two of eight of 4096 x 4096: Q8_0 140 us against 152 and 145 of eight waves, Q4_1 84 / 106 / 90, Q6_K
// 141 / 212 / 148, Q4_0 114 / 107 / 121, Q5_K 98 / - / 101).
// Three to twelve (to eight of 32-value blocks: registers): in sets of four, whose operands come out of LDS ahead of their products.  512 tokens, two of eight of 4096 x 14336 in Q4_K
// and Q6_K: 1380 us (1340 since the lists and the tokens' operands are made in one launch), with eight at most - more chunks where an expert has more rows than most - 1457; groups of sixteen rows, hi and lo parts as operands of their own, 1472; four
// waves and sets of two 1479; sixteen groups a chunk 1600 to 2243 (registers).  What bounds it there, of 1490: without its products it took 1009 us - operands on their way 215,
// to LDS 70, decoding 125, weights 130 -, without all of those 956; the products alone would be 490.
typedef RowsShape<8, 1, 1, 2> RowsShape1;
typedef RowsShape<4, 1, 1, 2> RowsShape1Short;
typedef RowsShape<8, 2, 1, 4> RowsShape2;
typedef RowsShape<4, 2, 1, 2> RowsShape2Short;
typedef RowsShape<8, 4, 2, 2> RowsShape8;
typedef RowsShape<8, 4, 3, 2> RowsShape12;

template <int FMT, class S>
static RowsKernelRef experts_rows_shape(bool dual) {
    const RowsKernel fn = dual ? experts_rows_kernel<FMT, S, true> : experts_rows_kernel<FMT, S, false>;
    // (weight rows of a workgroup: its waves' tiles; of a pair of matrices half as many of each)
    return {fn, experts_rows_lds<FMT, S>(), S::threads, S::waves * er_tiles<FMT, S>() / (dual ? 2 : 1), S::all_rows / 8};
}
// groups: of a chunk, at most 12, of 32-value blocks 8
template <int FMT>
static RowsKernelRef experts_rows_pick(int groups, bool dual) {
    if (groups <= 1) {
        if constexpr (RTile<FMT>::BLOCK_SCALES) return experts_rows_shape<FMT, RowsShape1Short>(dual);
        else return experts_rows_shape<FMT, RowsShape1>(dual);
    }
    if (groups <= 2) {
        if constexpr (FMT == F_Q6_K || (RTile<FMT>::BLOCK_SCALES && FMT != F_Q4_0)) return experts_rows_shape<FMT, RowsShape2Short>(dual);
        else return experts_rows_shape<FMT, RowsShape2>(dual);
    }
    if constexpr (!RTile<FMT>::BLOCK_SCALES) {
        if (groups > 8) return experts_rows_shape<FMT, RowsShape12>(dual);
    }
    return experts_rows_shape<FMT, RowsShape8>(dual);
}

}  // namespace jitnn
