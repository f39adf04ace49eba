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

// What a part takes when it is cut into spans of `steps` steps of a wave, in microseconds: its longest workgroup alone on a CU, and a workgroup's share of a CU that has
// others (as long as that where a CU holds no second one, heads of more than 128 values).  A step is its products at 1100 (FP16) or 140 (FP32) TFLOP/s and what it
// waits for; 40 GB/s and CU come from memory and the L2s.
struct PartTime {
    int span = 0, spans = 0;
    double alone = 0, busy = 0, load = 0, groups = 0;  // load: of a CU that takes its turn of them all
};
// (whole numbers: a call takes as long as its launch, and this is part of it)
static PartTime part_time(const AttnPart &q, bool half, int D, int keys, int len, double mean, long long units, int n, int cus) {
    PartTime t;
    const int least = keys * q.key_waves, all = (len + least - 1) / least, steps = (all + n - 1) / n;
    t.span = steps * least;
    t.spans = (all + steps - 1) / steps;
    const long long groups = units * t.spans * q.blocks;
    t.groups = (double)groups;
    const bool wide = q.key_waves == 1;
    const double product = (half ? 0.00167 : 0.0067) * D * q.tiles, bytes = 2. * least * D * (half ? 2 : 4);
    t.alone = (wide ? 3.7 : 1.9) + steps * (product + (wide ? 0.2 : 0.) + 0.003 * D);
    t.busy = (wide ? 4.4 : 2.7) + mean / (t.spans * least) * std::max(product + 0.04, bytes * (1. / 40e3));
    if (D > 128) t.busy = std::max(t.busy, 0.92 * t.alone);
    t.load = t.busy * (groups < 3ll * cus ? (double)((groups + cus - 1) / cus) : t.groups / cus + 0.7);
    return t;
}

// Spans of the shared positions and of the sequences' own: the numbers for which the modelled time is least.  While there are no more workgroups than CUs, the longest;
// beyond, a CU has one of each kind after the other as often as it takes (they go round the CUs), and those that do not find a place at once, the sequences', end
// later.  The merge is 5 us and what is written and read again of each row and span, at 4.6 TB/s.  A batch's lengths are taken to lie evenly up
// to the longest.  Over 260 batches of all head sizes, types, rows and lengths this took 2 % longer than the best of a sweep on average (spans of equal time for two
// workgroups to a CU: 12 %), and takes 0.1 to 0.8 us of the call.
AttnPlan paged_attn_plan(bool half, int D, int heads, int kv, int sequences, long long tokens, int max_tokens, int max_len, int shared, int cus) {
    const int group = heads / kv, keys = half ? 32 : 16;
    AttnPlan p;
    if (shared > 0) p.ahead = rows_shape(tokens * group, D);
    p.own = rows_shape((long long)max_tokens * group, D);
    const int own_len = std::max(max_len - shared, 1);
    const double own_mean = std::max(0.5 * own_len * (1 + 1. / sequences) - 0.5 * max_tokens, 1.);
    // (the largest two together below PA_MERGE)
    static constexpr int NUMBERS[] = {1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 14, 16, 18, 20, 22, 24, 28, 32, 36, 40, 45, 50, 56, 64, 80, 96, 120};
    constexpr int COUNT = sizeof(NUMBERS) / sizeof(int);
    PartTime ahead[COUNT], own[COUNT];
    int aheads = 0, owns = 0;
    long long before = 0;  // (the first number that leaves every wave one step is the last)
    for (int n : NUMBERS) {
        if (before * keys * p.ahead.key_waves < shared) ahead[aheads++] = part_time(p.ahead, half, D, keys, shared, shared, kv, n, cus);
        if (before * keys * p.own.key_waves < own_len) own[owns++] = part_time(p.own, half, D, keys, own_len, own_mean, (long long)kv * sequences, n, cus);
        before = n;
    }
    if (aheads == 0) aheads = 1;  // (no workgroups, no time)
    const int resident = (D <= 128 ? 2 : 1) * cus;
    const double merge = (double)tokens * heads * (D + 2) * (8 / 4.6e6);
    double least = 1e30;
    const PartTime *best_ahead = ahead, *best_own = own;
    for (int i = 0; i < aheads; ++i)
        for (int j = 0; j < owns; ++j) {
            const PartTime &a = ahead[i], &o = own[j];
            const double load = a.groups + o.groups <= cus ? std::max(a.busy, o.busy) : a.load + o.load;
            const int spans = a.spans + o.spans;
            const double time = std::max(std::max(a.alone, o.alone), load) + (a.groups + o.groups > resident ? 0.43 * o.alone : 0.) + (spans > 1 ? 4.9 + merge * spans : 0.);
            if (time < least) {
                least = time;
                best_ahead = &a;
                best_own = &o;
            }
        }
    p.ahead.span = best_ahead->span;
    p.ahead.spans = best_ahead->spans;
    p.own.span = best_own->span;
    p.own.spans = best_own->spans;
    // How many units are taken together (paged_attn_kernel).  Eight, a unit to an XCD, so that its row blocks share the keys in that XCD's L2 (63 sequences of 40 tokens
    // behind 360 others 54 us, with as many units as run at once 58); these where a sequence's rows differ much in what they see.  Units that are no multiple
    // of eight and all run at once go all together: rounded up they would leave XCDs idle (one prompt of 204 tokens on one key/value head ran on one).
    auto order = [&](AttnPart &q, long long of, bool prompts) {
        const long long units = of * kv * q.spans, whole = units % 8 != 0 && units * q.blocks <= resident ? units : (units + 7) / 8 * 8;
        q.beside = (int)std::min<long long>(whole, prompts ? std::max(8, resident / q.blocks / 8 * 8) : whole % 8 != 0 ? whole : 8);
    };
    if (shared > 0) order(p.ahead, 1, false);
    order(p.own, sequences, 2ll * max_tokens >= own_len);
    return p;
}

void paged_attn_launch(bool half, int D, int cus, hipStream_t s, AttnArgs a) {
    const unsigned units_ahead = (unsigned)(a.ahead.spans * a.kv), units_own = (unsigned)(a.own.spans * a.kv * a.sequences);
    auto groups = [](unsigned units, const AttnPart &q) { return (units + q.beside - 1) / q.beside * q.beside * (unsigned)q.blocks; };
    const unsigned ahead = groups(units_ahead, a.ahead), own = groups(units_own, a.own);
    // one to a CU, and where there are no more than CUs in all, the own behind the shared ones without a gap
    a.chunk = ahead > 0 && ahead + own <= (unsigned)cus ? (int)ahead : std::max(8, cus / 8 * 8);
    a.chunks_ahead = (int)((ahead + a.chunk - 1) / a.chunk);
    a.chunks_own = (int)((own + a.chunk - 1) / a.chunk);
    a.pairs = std::min(a.chunks_ahead, a.chunks_own);
    a.group = a.heads / a.kv;
    a.per_group = 1.f / (float)a.group;
    a.by_group = reciprocal(a.group);
    a.by_kv = reciprocal(a.kv);
    a.by_sequences = reciprocal(a.sequences);
    a.by_chunk = reciprocal(a.chunk);
    a.by_own_beside = reciprocal(a.own.beside);
    a.by_own = reciprocal(a.own.beside * a.own.blocks);
    a.by_own_span = reciprocal(a.own.span);
    if (ahead > 0) {
        a.by_ahead_beside = reciprocal(a.ahead.beside);
        a.by_ahead = reciprocal(a.ahead.beside * a.ahead.blocks);
        a.by_ahead_span = reciprocal(a.ahead.span);
    }
    const unsigned blocks = a.chunk == (int)ahead ? ahead + own : (unsigned)(a.chunks_ahead + a.chunks_own) * (unsigned)a.chunk;
    if (half) paged_attn_launch_f16(D, blocks, s, a);
    else paged_attn_launch_f32(D, blocks, s, a);
    if (a.ahead.spans + a.own.spans == 1) return;
    auto merge = [&](auto d) {
        constexpr int DD = decltype(d)::value, ROWS = PA_MERGE / (DD / 4);
        // (few spans and rows for every CU: 512 tokens of one sequence behind 3584, 16384 rows of 4 spans, 85 us against 95 with a workgroup to each row; 256 rows of 8
        // spans are 0.8 us slower with it)
        if (a.ahead.spans + a.own.spans <= PA_FEW && (long long)a.tokens * a.heads >= (long long)ROWS * cus)
            hipLaunchKernelGGL(paged_merge_few_kernel<DD>, dim3(a.tokens, (a.heads + ROWS - 1) / ROWS), dim3(PA_MERGE), 0, s, a);
        else
            hipLaunchKernelGGL(paged_merge_kernel<DD>, dim3(a.tokens, a.heads), dim3(PA_MERGE), 0, s, a);
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
