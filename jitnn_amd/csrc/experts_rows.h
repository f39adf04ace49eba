// The experts' products of many (token, expert) pairs on the matrix cores, at FP32-grade accuracy: gemv_rows_kernel's operands and decoders (gemv_rows.h), for
// rows that a list gathers.
//
// The operands of an activation row are prepared once, row by row (experts_prepare_kernel: FP16 hi and lo parts of the row scaled per 256 values, and the sums of
// its blocks), whoever it will meet: which eight rows stand in one matrix operand, the lists of the experts say when the operand is put together in LDS.
// A workgroup takes one expert, up to eight times `groups` of its rows and 8 waves x T tiles of 16 weight rows; all its waves are at the same 256 values of K, so that
// the operands cross from L2 to LDS once for the eight of them, while every weight byte is read by one wave only, decoded once and kept in registers for all
// the groups.  Nothing is added up across waves or workgroups, and a row's result does not depend on the rows beside it.
#pragma once
#include "act.h"
#include "common.h"
#include "experts.h"
#include "gemv_rows.h"

namespace jitnn {

constexpr int ER_WAVES = 8, ER_THREADS = ER_WAVES * 64;
constexpr int ER_OP_CHUNKS = 72;                      // 16-byte pieces of a row's operands of one column: [8 blocks and the sums][hi, lo][lane group]
constexpr int ER_OP_BYTES = ER_OP_CHUNKS * 16;
constexpr int ER_T = 2;                               // tiles of 16 weight rows that a wave holds: of gate and up one each
constexpr int ER_GROUP_CHUNKS = 9 * 64;               // pieces of the operands of a group of eight rows

template <int FMT>
__host__ __device__ constexpr size_t experts_rows_lds(int groups) {
    return (size_t)2 * groups * (ER_GROUP_CHUNKS * 16 + 8 * sizeof(float)) + (size_t)groups * 8 * 2 * sizeof(int) + (size_t)ER_WAVES * ER_T * RTile<FMT>::STAGE_BYTES;
}

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

struct ExpertPrepareOut {
    uint8_t *ops[3];  // per layout (GR_LAYOUT_*): nullptr - not wanted
    float *inv[3];    // [rows, columns]
};
// One wave per (column, eight rows): x [rows, k], k a multiple of 4.  grid (ceil(k / 256), ceil(rows / 8))
static __global__ void __launch_bounds__(64) experts_prepare_kernel(const float *__restrict__ x, int rows, int k, const ExpertPrepareOut o) {
    const int lane = threadIdx.x, b = lane >> 3, part = lane & 7, c = (int)blockIdx.x, ncol = (k + 255) >> 8, row = (int)blockIdx.y * 8 + b;
    const bool have = row < rows;
    const float *xr = x + (size_t)(have ? row : 0) * k;
    float4 v[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const int at = c * 256 + 32 * t + 4 * part;
        v[t] = at < k ? *reinterpret_cast<const float4 *>(xr + at) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const size_t at = (size_t)row * ncol + c;
    if (o.ops[0]) experts_prepare_column<32, false>(v, o.ops[0] + at * ER_OP_BYTES, o.inv[0] + at, have, part);
    if (o.ops[1]) experts_prepare_column<16, false>(v, o.ops[1] + at * ER_OP_BYTES, o.inv[1] + at, have, part);
    if (o.ops[2]) experts_prepare_column<32, true>(v, o.ops[2] + at * ER_OP_BYTES, o.inv[2] + at, have, part);
}

// Sixteen bytes of which those from `end` on are zero and not read: the sixteen in front of `end`, moved down (there are as many: a matrix is no smaller).
__device__ __forceinline__ u32x4 ld128_until(const uint8_t *p, const uint8_t *end) {
    const int behind = max((int)(p + 16 - end), 0), by = 8 * min(behind, 16);  // (of a wave's columns, so never far behind)
    const u32x4 v = ld128<2>(p - behind);
    const unsigned long long lo = (unsigned long long)v.y << 32 | v.x, hi = (unsigned long long)v.w << 32 | v.z;
    const unsigned long long down = by == 0 ? lo : by < 64 ? lo >> by | hi << (64 - by) : by < 128 ? hi >> (by - 64) : 0;
    const unsigned long long up = by < 64 ? hi >> by : 0;
    return u32x4{(uint32_t)down, (uint32_t)(down >> 32), (uint32_t)up, (uint32_t)(up >> 32)};
}

// The last column of rows that are no whole columns (32-value blocks): what lies behind a row's last block is the next row, behind the last row nobody's.
template <class R>
__device__ __forceinline__ void load_last_column(typename R::Raw &r, const typename R::Ptr &p, int c, const uint8_t *end) {
    const uint8_t *q = p.full + (size_t)c * R::BYTES;
#pragma unroll
    for (int i = 0; i < R::FULL; ++i) r.c[i] = ld128_until(q + 64 * i, end);
    if constexpr (R::REST > 0) r.c[R::FULL] = ld128_until(q + p.rest, end);
}

// grid: a.nblocks x (at least as many as there are chunks); experts_rows_lds<FMT>(a.groups) of dynamic LDS, a.groups <= GM.
// DUAL: tile i of gate and of up, y = act(gate x) * (up x); otherwise tiles 2 i and 2 i + 1 of w.
template <int FMT, int GM, bool DUAL>
__global__ void __launch_bounds__(ER_THREADS) experts_rows_kernel(const ExpertRowsArgs a) {
    typedef RTile<FMT> R;
    constexpr int NOPS = R::NOPS, NI = (GM * ER_GROUP_CHUNKS + ER_THREADS - 1) / ER_THREADS;
    constexpr int HELD = NOPS > 8 && GM > 1 ? 1 : ER_T;  // tiles whose operands a wave has at a time: of Q6_K's sixteen a tile there is room for one beside the rest
    constexpr bool PARTIAL = R::BLOCK_SCALES;  // (only 32-value blocks have rows that are no whole columns)
    extern __shared__ __attribute__((aligned(16))) uint8_t er_smem[];
    const int G = a.groups;
    u32x4 *const ops = reinterpret_cast<u32x4 *>(er_smem);                            // [2][G][9][64]
    float *const invs = reinterpret_cast<float *>(ops + (size_t)2 * G * ER_GROUP_CHUNKS);  // [2][G * 8]
    uint32_t *const where = reinterpret_cast<uint32_t *>(invs + 2 * G * 8);           // [G * 8] a row's operands, in columns from the first one's
    int *const slots = reinterpret_cast<int *>(where + G * 8);                        // [G * 8]
    const int tid = threadIdx.x, lane = tid & 63, kq = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t *const stage = reinterpret_cast<uint8_t *>(slots + G * 8) + (size_t)wave * ER_T * R::STAGE_BYTES;
    const int u = (int)blockIdx.x / a.nblocks, block = (int)blockIdx.x - u * a.nblocks;
    if (u >= a.chunks->x) return;
    const int4 ch = a.chunks[1 + u];  // expert, place of its first row in the list, rows
    const int ncol = (a.k + 255) >> 8, groups = (ch.z + 7) >> 3, items = groups * ER_GROUP_CHUNKS;

    // the weights on their way first: column 0 of this wave's tiles
    const size_t rowbytes = (size_t)(a.k / block_values(FMT)) * block_bytes(FMT);
    const uint8_t *const w0 = a.w + (size_t)ch.x * a.expert_bytes, *const w1 = DUAL ? a.w2 + (size_t)ch.x * a.expert_bytes : w0;
    const int ntiles = a.n >> 4, tile = (block * ER_WAVES + wave) * (DUAL ? 1 : ER_T);
    const uint8_t *const end0 = a.w + (size_t)a.experts * a.expert_bytes, *const end1 = DUAL ? a.w2 + (size_t)a.experts * a.expert_bytes : end0;
    typename R::Ptr ptr[ER_T];
    typename R::Raw raw[ER_T];
    ptr[0] = R::ptr(w0, min(tile, ntiles - 1) * 16, rowbytes, lane);
    ptr[1] = R::ptr(w1, min(DUAL ? tile : tile + 1, ntiles - 1) * 16, rowbytes, lane);
    const int last_blocks = PARTIAL ? (a.k & 255) >> 5 : 0;  // of the last column, where it is none of eight
    auto fetch = [&](int c) {
        if (PARTIAL && last_blocks && c == ncol - 1) {
            load_last_column<R>(raw[0], ptr[0], c, end0);
            load_last_column<R>(raw[1], ptr[1], c, end1);
            return;
        }
        R::load(raw[0], ptr[0], c);
        R::load(raw[1], ptr[1], c);
    };
    fetch(0);
    if (tid < groups * 8) {  // (a place without a row takes the last one again: computed, not stored)
        const int slot = a.list[ch.y + min(tid, ch.z - 1)];
        slots[tid] = slot;
        where[tid] = (uint32_t)(slot / a.per_row) * (uint32_t)ncol;
    }
    __syncthreads();
    // piece i of this thread: lane l of operand s of group g, whose row is that of l's place
    uint32_t from[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int idx = min(tid + i * ER_THREADS, items - 1), g = idx / ER_GROUP_CHUNKS, rest = idx - g * ER_GROUP_CHUNKS, s = rest >> 6, l = rest & 63;
        from[i] = where[g * 8 + ((l & 15) >> 1)] * (uint32_t)ER_OP_BYTES + (uint32_t)(s * 128 + (l & 1) * 64 + (l >> 4) * 16);
    }
    const uint32_t inv_from = tid < groups * 8 ? where[tid] : 0u;
    u32x4 next[NI];
    float next_inv = 0.f;
    auto ask = [&](int c) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (i == 0 || wave * 64 + i * ER_THREADS < items) next[i] = *reinterpret_cast<const u32x4 *>(a.ops + from[i] + (size_t)c * ER_OP_BYTES);
        if (tid < groups * 8) next_inv = a.inv[inv_from + c];
    };
    ask(0);

    float2 acc[ER_T][GM];
#pragma unroll
    for (int t = 0; t < ER_T; ++t)
#pragma unroll
        for (int g = 0; g < GM; ++g) acc[t][g] = make_float2(0.f, 0.f);
    for (int c = 0; c < ncol; ++c) {
        // this column's operands into the buffer that nobody reads any more: every wave has passed the barrier of the column before, behind its products of the
        // one before that
        u32x4 *const op = ops + (size_t)(c & 1) * G * ER_GROUP_CHUNKS;
        float *const iv = invs + (c & 1) * G * 8;
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (wave * 64 + i * ER_THREADS < items) op[tid + i * ER_THREADS] = next[i];
        if (tid < groups * 8) iv[tid] = next_inv;
        const uint8_t *row[ER_T];
        uint32_t tail[ER_T];
#pragma unroll
        for (int t = 0; t < ER_T; ++t) {
            row[t] = R::park(raw[t], stage + t * R::STAGE_BYTES, lane);
            tail[t] = raw[t].tail;
        }
        if (c + 1 < ncol) {
            fetch(c + 1);
            ask(c + 1);
        }
        f16x8 B[HELD][NOPS], Bm[HELD];
        float d[HELD], dmin64[HELD], dblk[R::BLOCK_SCALES ? HELD : 1][8];
        auto decode = [&](int t, int h) {
            if constexpr (R::BLOCK_SCALES) {
                R::decode(row[t], tail[t], lane, B[h], Bm[h], dblk[h]);
                if (PARTIAL && last_blocks && c == ncol - 1) {  // (their operands are zero, what stands there need not be a number)
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        dblk[h][s] = s < last_blocks ? dblk[h][s] : 0.f;
                        Bm[h][s] = s < last_blocks ? Bm[h][s] : (_Float16)0.f;
                    }
                }
            } else {
                float dm;
                R::decode(row[t], tail[t], lane, B[h], Bm[h], d[h], dm);
                dmin64[h] = dm * 64.f;
            }
        };
        // the products of tiles t0 .. t0 + HELD - 1 with every group
        auto multiply = [&](int t0) {
#pragma unroll
            for (int g = 0; g < GM; ++g) {
                if (g >= groups) break;
                f16x8 A[9];
#pragma unroll
                for (int s = 0; s < 9; ++s) A[s] = __builtin_bit_cast(f16x8, op[(g * 9 + s) * 64 + lane]);
                const float2 w = *reinterpret_cast<const float2 *>(iv + g * 8 + 2 * kq);
#pragma unroll
                for (int h = 0; h < HELD; ++h) {
                    float u0, u1;
                    if constexpr (R::BLOCK_SCALES) {
                        u0 = u1 = 0.f;
#pragma unroll
                        for (int s = 0; s < 8; ++s) {
                            const f32x4 cs = mfma16(A[s], B[h][s]);
                            u0 = __builtin_fmaf(dblk[h][s], cs[0] + cs[1], u0);
                            u1 = __builtin_fmaf(dblk[h][s], cs[2] + cs[3], u1);
                        }
                        if constexpr (R::MINS) {
                            const f32x4 cm = mfma16(A[8], Bm[h]);
                            u0 = __builtin_fmaf(64.f, cm[0] + cm[1], u0);
                            u1 = __builtin_fmaf(64.f, cm[2] + cm[3], u1);
                        }
                    } else {
                        f32x4 cs = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int s = 0; s < NOPS; ++s) cs = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[R::aidx(s)], B[h][s], cs, 0, 0, 0);
                        const f32x4 cm = mfma16(A[8], Bm[h]);
                        const float s0 = cs[0] + cs[1], s1 = cs[2] + cs[3], m0 = cm[0] + cm[1], m1 = cm[2] + cm[3];
                        u0 = __builtin_fmaf(d[h], s0, -dmin64[h] * m0);
                        u1 = __builtin_fmaf(d[h], s1, -dmin64[h] * m1);
                    }
                    acc[t0 + h][g].x = __builtin_fmaf(w.x, u0, acc[t0 + h][g].x);
                    acc[t0 + h][g].y = __builtin_fmaf(w.y, u1, acc[t0 + h][g].y);
                }
                // (the operands and products of one group at a time: of more than one there are no registers)
#pragma unroll
                for (int h = 0; h < HELD; ++h) asm volatile("" : "+v"(acc[t0 + h][g].x), "+v"(acc[t0 + h][g].y));
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if constexpr (HELD == ER_T) {
#pragma unroll
            for (int t = 0; t < ER_T; ++t) decode(t, t);
            __syncthreads();
            multiply(0);
        } else {
            decode(0, 0);
            __syncthreads();
            multiply(0);
            decode(1, 0);
            multiply(1);
        }
    }
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        if (g >= groups) break;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int b = g * 8 + 2 * kq + r;
            if (b >= ch.z) continue;
            float *const y = a.y + (size_t)slots[b] * a.n + (lane & 15);
            const float v0 = r ? acc[0][g].y : acc[0][g].x, v1 = r ? acc[1][g].y : acc[1][g].x;
            if (DUAL) {
                if (tile < ntiles) y[tile * 16] = activate(a.act, v0) * v1;
            } else {
                if (tile < ntiles) y[tile * 16] = v0;
                if (tile + 1 < ntiles) y[tile * 16 + 16] = v1;
            }
        }
    }
}

// groups: the largest that the LDS of a workgroup holds two buffers of, at most 5
template <int FMT>
static KernelRef experts_rows_pick(int groups, bool dual) {
    const void *fn = groups == 1 ? (dual ? (const void *)experts_rows_kernel<FMT, 1, true> : (const void *)experts_rows_kernel<FMT, 1, false>)
                     : groups == 2 ? (dual ? (const void *)experts_rows_kernel<FMT, 2, true> : (const void *)experts_rows_kernel<FMT, 2, false>)
                                   : (dual ? (const void *)experts_rows_kernel<FMT, 5, true> : (const void *)experts_rows_kernel<FMT, 5, false>);
    return {fn, experts_rows_lds<FMT>(groups)};
}

template <int FMT>
static void experts_rows_go(const ExpertRowsArgs &a, unsigned blocks, bool dual, hipStream_t s) {
    typedef void (*Kernel)(const ExpertRowsArgs);
    const KernelRef k = experts_rows_pick<FMT>(a.groups, dual);
    hipLaunchKernelGGL((Kernel)k.fn, dim3(blocks), dim3(ER_THREADS), k.lds, s, a);
}

}  // namespace jitnn
