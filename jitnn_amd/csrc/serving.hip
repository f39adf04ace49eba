// Launches of the operators of a served batch: rotary positions, the paged cache's append, the plan and the merge of its attention (whose kernels
// are in paged_f16.hip and paged_f32.hip), the verification of drafted tokens.
#include "serving.h"

#include <algorithm>
#include <cmath>

#include "paged_attn.h"
#include "rope.h"
#include "verify.h"

namespace jitnn {

static bool aligned16(const void *p, long long stride) { return ((uintptr_t)p & 15) == 0 && stride % 4 == 0; }

void rope_launch(const RopeArgs &a, int cus, hipStream_t s) {
    const bool items = a.rot % 8 == 0 && a.D % 8 == 0 && aligned16(a.x, a.x_stride) && aligned16(a.y, a.y_stride);
    const long long count = (long long)a.tokens * a.heads * (items ? a.D / 8 : (a.D + 1) / 2);
    const unsigned blocks = (unsigned)std::min<long long>((count + ROPE_THREADS - 1) / ROPE_THREADS, (long long)cus * 64);
    if (items) hipLaunchKernelGGL(rope_kernel, dim3(blocks), dim3(ROPE_THREADS), 0, s, a);
    else hipLaunchKernelGGL(rope_pairs_kernel, dim3(blocks), dim3(ROPE_THREADS), 0, s, a);
}

void paged_append_launch(bool half, AppendArgs a, int cus, hipStream_t s) {
    const long long n = (long long)(a.heads + 2 * a.kv) * (a.D / 8);  // items of a token
    a.per_block = (int)std::min<long long>(std::max<long long>(1, ROPE_THREADS / n), APPEND_TOKENS);
    const unsigned blocks = (unsigned)((a.tokens + a.per_block - 1) / a.per_block);
    // few tokens: several workgroups to a token's heads
    const unsigned shares = (unsigned)std::max<long long>(1, std::min<long long>((n * a.per_block + ROPE_THREADS - 1) / ROPE_THREADS, 4ll * cus / blocks));
    if (half) hipLaunchKernelGGL(paged_append_kernel<_Float16>, dim3(blocks, shares), dim3(ROPE_THREADS), 0, s, a);
    else hipLaunchKernelGGL(paged_append_kernel<float>, dim3(blocks, shares), dim3(ROPE_THREADS), 0, s, a);
}

void paged_copy_launch(void *k, void *v, long long page_bytes, long long layer_bytes, int layers, int from, int to, hipStream_t s) {
    const long long page16 = page_bytes / 16;
    hipLaunchKernelGGL(paged_copy_kernel, dim3((unsigned)std::min<long long>((page16 + 255) / 256, 64), layers, 2), dim3(256), 0, s, (uint4 *)k, (uint4 *)v, page16,
                       layer_bytes / 16, from, to);
}

// ---- attention

// How the rows of a part go to workgroups: few rows, all four waves on keys of their own; many, two tiles of rows to a wave (heads of
// up to 128 values: their queries and outputs leave the registers for it) and all waves on the same keys.
static AttnPart rows_shape(long long rows, int D) {
    AttnPart p;
    p.tiles = D <= 128 && rows > 16 ? 2 : 1;
    p.key_waves = rows <= 16 * p.tiles ? 4 : rows <= 32 * p.tiles ? 2 : 1;
    const int per = 16 * p.tiles * (PA_WAVES / p.key_waves);
    p.blocks = (int)std::min<long long>((rows + per - 1) / per, 1 << 24);
    return p;
}

// Spans of a part whose waves share their keys and that is alone: the number for which the workgroups and the merge of what they leave, modelled in
// microseconds, take least; of nearly equal ones the fewest.  A step of a workgroup is its products at 1100 (FP16) or 140 (FP32) TFLOP/s, on top of which it
// waits 0.35 us and 3.5 ns a value of the head, two thirds of that where the CU has another one to work on; before the first it takes 5 (2.5).  The
// merge is a launch, and what is written and read again of each row and span at 4.2 TB/s.  Heads of 128, FP16, 32 of them: 2000 tokens' own positions, one span
// 91 us, two 119; 512 tokens behind 3584 others, one 158, two 99, four 86, eight 101.
static int wide_spans(bool half, int D, long long rows_all, const AttnPart &q, long long units, int keys, double len, double seen, int cus) {
    const int per_cu = D <= 128 ? 2 : 1;
    const double product = (half ? 0.00167 : 0.0067) * D * q.tiles;
    int best = 1;
    double least = 1e30;
    for (int n = 1; n <= 120 && (n - 1) * keys < len; n = std::max(n + 1, n * 5 / 4)) {
        const double longest = std::ceil(len / n / keys), mean = std::max(seen / n / keys, 0.5), rounds = std::ceil((double)units * n / cus);
        const bool two = per_cu == 2 && rounds > 1;
        const double wait = (0.35 + 0.0035 * D) * (two ? 0.65 : 1.);
        const double run = std::max(5 + longest * (product + 0.35 + 0.0035 * D), rounds * ((two ? 2.5 : 5.) + mean * (product + wait)));
        const double time = run + (n > 1 ? 6 + (double)rows_all * std::min(n * seen / len + 0.5, (double)n) * (D + 2) * 8 / 4.2e6 : 0.);
        if (time < 0.95 * least) {
            least = time;
            best = n;
        }
    }
    return best;
}

AttnPlan paged_attn_plan(bool half, int D, int heads, int kv, int sequences, long long tokens, int max_tokens, int max_len, int shared, int cus) {
    const int group = heads / kv, keys = half ? 32 : 16;
    AttnPlan p;
    if (shared > 0) p.ahead = rows_shape(tokens * group, D);
    p.own = rows_shape((long long)max_tokens * group, D);
    // Spans of about equal time: for two workgroups to a CU, as many as run at once, where some share their keys (each leaves its rows' sums in memory, so that
    // more of them cost more than their balance gains: 64 sequences behind 16384 shared positions 70 us with two, 96 with three, 93 with four); for
    // four where all stream (8 sequences of up to 2000 positions 38.1 us, with two 38.7).
    auto step = [](const AttnPart &q) { return q.tiles == 2 ? 1.6 : 1.0; };  // of a wave, in units of one tile's
    const double own_len = std::max(max_len - shared, 1);
    auto work = [&](const AttnPart &q, double n, double len) { return n * q.blocks * kv * len / q.key_waves * step(q); };
    const double all = (shared > 0 ? work(p.ahead, 1, shared) : 0) + work(p.own, sequences, own_len), each = all / ((p.own.key_waves == 1 || (shared > 0 && p.ahead.key_waves == 1) ? 2. : 4.) * cus);
    auto cut = [&](AttnPart &q, double len) {
        const int least = keys * q.key_waves;  // one step of every wave
        const double want = std::max(each * q.key_waves / step(q), len / 120);  // (at most 128 spans of each part: PA_MERGE)
        q.span = (int)std::min<double>(std::ceil(want / least) * least, std::ceil(len / least) * least);
        q.spans = (int)((len + q.span - 1) / q.span);
    };
    // Where a sequence's rows differ much in what they see; where they do not, the fewer units at a time share the more in an XCD's L2 (63 sequences of 40 tokens
    // behind 360 others 54 us, with these 58).  No more units than there are: the order is dense, and so is their spread over the CUs.
    auto side_by_side = [&](AttnPart &q) {
        if (2. * max_tokens < own_len) return;
        const long long units = ((long long)kv * sequences * q.spans + 7) / 8 * 8;
        q.beside = (int)std::min<long long>(units, std::max(8, (D <= 128 ? 2 : 1) * cus / q.blocks / 8 * 8));
    };
    if (shared == 0 && p.own.key_waves == 1) {
        const int n = wide_spans(half, D, tokens * heads, p.own, (long long)p.own.blocks * kv * sequences, keys, own_len, std::max(own_len - 0.5 * max_tokens, 1.), cus);
        p.own.span = (int)std::ceil(own_len / n / keys) * keys;
        p.own.spans = (int)((own_len + p.own.span - 1) / p.own.span);
        side_by_side(p.own);
        return p;
    }
    if (shared > 0) cut(p.ahead, shared);
    cut(p.own, own_len);
    side_by_side(p.own);
    return p;
}

void paged_attn_launch(bool half, int D, int cus, hipStream_t s, AttnArgs a) {
    const unsigned units_ahead = (unsigned)(a.ahead.spans * a.kv), units_own = (unsigned)(a.own.spans * a.kv * a.sequences);
    const unsigned ahead = (units_ahead + a.ahead.beside - 1) / a.ahead.beside * a.ahead.beside * (unsigned)a.ahead.blocks, own = (units_own + a.own.beside - 1) / a.own.beside * a.own.beside * (unsigned)a.own.blocks;
    a.chunk = std::max(8, cus / 8 * 8);  // one to a CU
    a.chunks_ahead = (int)((ahead + a.chunk - 1) / a.chunk);
    a.chunks_own = (int)((own + a.chunk - 1) / a.chunk);
    a.pairs = std::min(a.chunks_ahead, a.chunks_own);
    const unsigned blocks = (unsigned)(a.chunks_ahead + a.chunks_own) * (unsigned)a.chunk;
    if (half) paged_attn_launch_f16(D, blocks, s, a);
    else paged_attn_launch_f32(D, blocks, s, a);
    if (a.ahead.spans + a.own.spans == 1) return;
    auto merge = [&](auto d) {
        constexpr int DD = decltype(d)::value, ROWS = PA_MERGE / (DD / 4);
        // (few spans and rows for every CU: 512 tokens of one sequence behind 4096, 16384 rows of 5 spans, 85 us against 95 with a workgroup to each row; of 8
        // sequences' 256 rows, 8 spans, 38.6 against 37.8)
        if (a.ahead.spans + a.own.spans <= PA_FEW && (long long)a.tokens * a.heads >= (long long)ROWS * cus) hipLaunchKernelGGL(paged_merge_few_kernel<DD>, dim3(a.tokens, (a.heads + ROWS - 1) / ROWS), dim3(PA_MERGE), 0, s, a);
        else hipLaunchKernelGGL(paged_merge_kernel<DD>, dim3((unsigned)((long long)a.tokens * a.heads)), dim3(PA_MERGE), 0, s, a);
    };
    switch (D) {
    case 64: merge(std::integral_constant<int, 64>{}); break;
    case 128: merge(std::integral_constant<int, 128>{}); break;
    case 192: merge(std::integral_constant<int, 192>{}); break;
    default: merge(std::integral_constant<int, 256>{}); break;
    }
}

// ---- verification

static int verify_chunks(int vocab) { return (vocab + VERIFY_CHUNK - 1) / VERIFY_CHUNK; }
size_t verify_workspace(int rows, int sequences, int vocab) {
    return (size_t)verify_chunks(vocab) * ((size_t)rows * sizeof(VerifyStat) + (size_t)sequences * sizeof(double));
}
void verify_launch(VerifyArgs a, hipStream_t s) {
    a.chunks = verify_chunks(a.vocab);
    if (a.rows > 0) hipLaunchKernelGGL(verify_stats_kernel, dim3(a.chunks, a.rows), dim3(VERIFY_THREADS), 0, s, a);
    if (a.draft_probs && a.chunks > VERIFY_FEW) hipLaunchKernelGGL(verify_rest_kernel, dim3(a.chunks, a.sequences), dim3(VERIFY_THREADS), 0, s, a);
    hipLaunchKernelGGL(verify_draw_kernel, dim3(a.sequences), dim3(VERIFY_DRAW_THREADS), 0, s, a);
}

}  // namespace jitnn
