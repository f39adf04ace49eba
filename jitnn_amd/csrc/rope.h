// Rotary positions: y = m R(pos) x for the first rot values of every head, the rest as they are; and the append of a batch's keys and
// values to a paged cache, which rotates queries and keys on its way.
//
// The angle of pair i at position t is t * f_i.  Held as a fraction of a turn in 64-bit fixed point, the product t * f_i modulo one turn is
// one integer multiplication whose overflow is the whole turns: exact for any 32-bit position, negative ones among them, where a product
// in FP32 has lost the angle (a position of 131072 leaves it 2^-7 rad) and one in FP64 would need its reduction.  The top two bits, rounded,
// are the quadrant; the rest, in [-pi/4, pi/4], goes to FP32 (relative error 2^-24) and into the Taylor series of sine and cosine (the
// first terms left out are below 2e-9).  Sines and cosines are so within 1.5e-7, where FP64 ones rounded once would be within 6e-8: outputs of 4096 tokens are off by 5.3e-8 of their norm
// and not by 4.6e-8.
#pragma once
#include "common.h"
#include "serving.h"

namespace jitnn {

// cos and sin of the angle, times the magnitude
__device__ __forceinline__ float2 rope_turn(unsigned long long turns, int pos, float magnitude) {
    const uint32_t hi = (uint32_t)((turns * (unsigned long long)(long long)pos) >> 32);
    const uint32_t quadrant = (hi + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(hi - (quadrant << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
    const float z = x * x;
    const float s = __builtin_fmaf(x * z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), x);
    const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
    float a = quadrant & 1 ? s : c, b = quadrant & 1 ? c : s;  // |cos|, |sin| of the whole angle up to sign
    a = (quadrant + 1) & 2 ? -a : a;
    b = quadrant & 2 ? -b : b;
    return make_float2(a * magnitude, b * magnitude);
}

// A head in items of eight values: of the rotated part four pairs each (values 8 i .. + 7, or 4 i .. + 3 and those rot / 2 behind them),
// behind it eight neighbours.  The two quads of item i start at values .x and .y.
__device__ __forceinline__ int2 rope_item(int i, int rot, bool interleaved) {
    return 8 * i < rot && !interleaved ? make_int2(4 * i, 4 * i + rot / 2) : make_int2(8 * i, 8 * i + 4);
}
__device__ __forceinline__ void rope_rotate(float4 &a, float4 &b, const unsigned long long *__restrict__ turns, int i, int pos, float magnitude, bool interleaved) {
    float2 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = rope_turn(turns[4 * i + u], pos, magnitude);
    const float4 x = a, y = b;
    if (interleaved) {
        a = make_float4(x.x * w[0].x - x.y * w[0].y, x.x * w[0].y + x.y * w[0].x, x.z * w[1].x - x.w * w[1].y, x.z * w[1].y + x.w * w[1].x);
        b = make_float4(y.x * w[2].x - y.y * w[2].y, y.x * w[2].y + y.y * w[2].x, y.z * w[3].x - y.w * w[3].y, y.z * w[3].y + y.w * w[3].x);
    } else {
        a = make_float4(x.x * w[0].x - y.x * w[0].y, x.y * w[1].x - y.y * w[1].y, x.z * w[2].x - y.z * w[2].y, x.w * w[3].x - y.w * w[3].y);
        b = make_float4(x.x * w[0].y + y.x * w[0].x, x.y * w[1].y + y.y * w[1].x, x.z * w[2].y + y.z * w[2].x, x.w * w[3].y + y.w * w[3].x);
    }
}

constexpr int ROPE_THREADS = 256;

// Bound by memory: 4096 tokens of 32 heads of 128 values are 134 MB read and written, 24.3 us (5.5 TB/s; a copy of 4 GiB runs at 4.7), one token is
// an empty launch.  A thread turns four pairs, two 16-byte loads and two stores, with the sine and cosine of each worked out where they are used: a table per
// token and pair would be read as often as it would be computed.
// x [tokens, heads, D] with rows x_stride apart, y likewise (y == x: in place).  Whole items of eight values whose quads are aligned to
// 16 bytes; rope_pairs_kernel takes the rest.
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeArgs a) {
    const uint32_t items = (uint32_t)a.D / 8, n = (uint32_t)a.heads * items;  // of a token
    const uint64_t all = (uint64_t)a.tokens * n;
    for (uint64_t at = (uint64_t)blockIdx.x * ROPE_THREADS + threadIdx.x; at < all; at += (uint64_t)gridDim.x * ROPE_THREADS) {
        const uint32_t t = (uint32_t)(at / n), r = (uint32_t)(at - (uint64_t)t * n), h = r / items;
        const int i = (int)(r - h * items);
        const int2 e = rope_item(i, a.rot, a.interleaved);
        const float *x = a.x + (size_t)t * a.x_stride + (size_t)h * a.D;
        float *y = a.y + (size_t)t * a.y_stride + (size_t)h * a.D;
        float4 u = *reinterpret_cast<const float4 *>(x + e.x), v = *reinterpret_cast<const float4 *>(x + e.y);
        if (8 * i < a.rot) rope_rotate(u, v, a.turns, i, a.positions[t], a.magnitude, a.interleaved);
        *reinterpret_cast<float4 *>(y + e.x) = u;
        *reinterpret_cast<float4 *>(y + e.y) = v;
    }
}

// The same pair by pair: any even rot and D, any alignment.  4096 tokens of 32 heads of 128 in rows of 4097 floats 28.3 us, of 250 interleaved values 49.9 (5.2 TB/s); in rows of 4096
// floats rope_kernel takes 21.6.
__global__ void __launch_bounds__(ROPE_THREADS) rope_pairs_kernel(const RopeArgs a) {
    const uint32_t pairs = (uint32_t)(a.D + 1) / 2, n = (uint32_t)a.heads * pairs;
    const uint64_t all = (uint64_t)a.tokens * n;
    for (uint64_t at = (uint64_t)blockIdx.x * ROPE_THREADS + threadIdx.x; at < all; at += (uint64_t)gridDim.x * ROPE_THREADS) {
        const uint32_t t = (uint32_t)(at / n), r = (uint32_t)(at - (uint64_t)t * n), h = r / pairs;
        const int i = (int)(r - h * pairs);
        const float *x = a.x + (size_t)t * a.x_stride + (size_t)h * a.D;
        float *y = a.y + (size_t)t * a.y_stride + (size_t)h * a.D;
        if (2 * i < a.rot) {
            const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + a.rot / 2;
            const float2 w = rope_turn(a.turns[i], a.positions[t], a.magnitude);
            const float u = x[i0], v = x[i1];
            y[i0] = u * w.x - v * w.y;
            y[i1] = u * w.y + v * w.x;
        } else {
            y[2 * i] = x[2 * i];
            if (2 * i + 1 < a.D) y[2 * i + 1] = x[2 * i + 1];
        }
    }
}

// ---- append

// The sequence of token t: how many of starts[1 .. sequences] are at or below it; `sequences` for a token behind the last.  One wave.
__device__ __forceinline__ int batch_sequence(const int *__restrict__ starts, int sequences, int t) {
    int s = 0;
    for (int i = threadIdx.x & 63; i < ((sequences + 63) & ~63); i += 64) s += __popcll(__ballot(i < sequences && starts[i + 1] <= t));
    return s;
}

// what the cache holds of an FP32 value.  F16: rounded to nearest, a finite value beyond its range as its largest.
__device__ __forceinline__ _Float16 cache_half(float x) { return (_Float16)(fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x); }
__device__ __forceinline__ void cache_store4(float *p, const float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void cache_store4(_Float16 *p, const float4 v) {
    *reinterpret_cast<f16x4 *>(p) = f16x4{cache_half(v.x), cache_half(v.y), cache_half(v.z), cache_half(v.w)};
}

// Rows of a batch: q rotated to q_out, k rotated and v as it is into the pages of their sequence.  A token behind the last sequence, at a
// position outside its table or on a page that the cache does not have leaves everything as it was, its row of q_out among it.
// Bound by memory: a prompt of 4096 tokens, 32 + 8 + 8 heads of 128 and FP16 pages, 185 MB, 41 us (4.5 TB/s); 64 tokens of 64 sequences 3.9 us, three round trips
// for their places and one for the rows.  A workgroup takes `per_block` tokens: their sequences, positions and pages are found by a wave each (three round trips in a row: starts,
// lens, the page) while nothing else waits for them, and stand in LDS for all heads.
constexpr int APPEND_TOKENS = 32;  // most tokens of a workgroup
template <class T>
__global__ void __launch_bounds__(ROPE_THREADS) paged_append_kernel(const AppendArgs a) {
    __shared__ int at_pos[APPEND_TOKENS];
    __shared__ long long at_row[APPEND_TOKENS];
    const int t0 = blockIdx.x * a.per_block, tokens = min(a.per_block, a.tokens - t0);
    for (int j = threadIdx.x >> 6; j < tokens; j += ROPE_THREADS / 64) {
        const int t = t0 + j, s = batch_sequence(a.starts, a.sequences, t);
        if ((threadIdx.x & 63) == 0) {
            const int pos = s < a.sequences && t >= a.starts[0] ? a.lens[s] - a.starts[s + 1] + t : -1;
            long long row = -1;
            if (pos >= 0 && (pos >> a.page_shift) < a.table_stride) {
                const int page = a.tables[(size_t)s * a.table_stride + (pos >> a.page_shift)];
                if ((unsigned)page < (unsigned)a.pages)
                    row = (((long long)page * a.kv) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
            }
            at_pos[j] = pos;
            at_row[j] = row;
        }
    }
    __syncthreads();
    const uint32_t items = (uint32_t)a.D / 8, hn = (uint32_t)(a.heads + 2 * a.kv), n = hn * items, all = (uint32_t)tokens * n;
    for (uint32_t at = blockIdx.y * ROPE_THREADS + threadIdx.x; at < all; at += gridDim.y * ROPE_THREADS) {
        const uint32_t j = at / n, r = at - j * n;
        const int h = (int)(r / items), i = (int)(r - (uint32_t)h * items), t = t0 + (int)j;
        const long long row = at_row[j];
        if (row < 0) continue;
        const bool value = h >= a.heads + a.kv, key = !value && h >= a.heads;
        const float *x = value ? a.v + (size_t)t * a.v_stride + (size_t)(h - a.heads - a.kv) * a.D
                         : key ? a.k + (size_t)t * a.k_stride + (size_t)(h - a.heads) * a.D : a.q + (size_t)t * a.q_stride + (size_t)h * a.D;
        const bool turned = !value && 8 * i < a.rot;
        const int2 e = rope_item(i, turned ? a.rot : 0, a.interleaved);
        float4 u = *reinterpret_cast<const float4 *>(x + e.x), w = *reinterpret_cast<const float4 *>(x + e.y);
        if (turned) rope_rotate(u, w, a.turns, i, at_pos[j], a.magnitude, a.interleaved);
        if (!value && !key) {
            float *y = a.q_out + (size_t)t * a.q_out_stride + (size_t)h * a.D;
            *reinterpret_cast<float4 *>(y + e.x) = u;
            *reinterpret_cast<float4 *>(y + e.y) = w;
        } else {
            const int g = value ? h - a.heads - a.kv : h - a.heads;
            T *y = (value ? (T *)a.v_pages : (T *)a.k_pages) + (size_t)(row + ((long long)g << a.page_shift)) * a.D;
            cache_store4(y + e.x, u);
            cache_store4(y + e.y, w);
        }
    }
}

// A copy, 16 bytes a thread and step: bound by memory.  Page `from` of every layer to page `to`.
__global__ void __launch_bounds__(256) paged_copy_kernel(uint4 *k, uint4 *v, long long page16, long long layer16, int from, int to) {
    uint4 *p = (blockIdx.z ? v : k) + blockIdx.y * layer16;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < page16; i += (long long)gridDim.x * 256) p[to * page16 + i] = p[from * page16 + i];
}

}  // namespace jitnn
