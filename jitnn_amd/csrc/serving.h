// Host entry points of serving.hip, paged_f16.hip and paged_f32.hip - rotary positions, the paged cache's append and attention, the verification of
// drafted tokens - and the argument blocks of their kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace jitnn {

// ---- rope.h
struct RopeArgs {
    const float *x;
    float *y;
    const int *positions;
    const unsigned long long *turns;  // [rot / 2] of a pair: 2^64 of its frequency as a fraction of a turn
    long long x_stride, y_stride;
    float magnitude;
    int tokens, heads, D, rot;
    bool interleaved;
};
void rope_launch(const RopeArgs &a, int cus, hipStream_t s);

struct AppendArgs {
    const float *q, *k, *v;
    float *q_out;
    void *k_pages, *v_pages;  // of the layer
    const int *tables, *starts, *lens;
    const unsigned long long *turns;
    long long q_stride, q_out_stride, k_stride, v_stride;
    float magnitude;
    int tokens, sequences, table_stride, pages, page_shift;
    int heads, kv, D, rot;  // heads 0: no queries; rot 0: nothing turns
    int per_block;
    bool interleaved;
};
void paged_append_launch(bool half, AppendArgs a, int cus, hipStream_t s);
void paged_copy_launch(void *k, void *v, long long page_bytes, long long layer_bytes, int layers, int from, int to, hipStream_t s);

// ---- paged_attn.h
// The keys of a part of the work - the shared positions, or one sequence's own - go to workgroups of four waves: 4 / key_waves of them take
// 16 tiles rows each, key_waves of them the same rows on keys of their own, `span` keys to a workgroup.
struct AttnPart {
    int blocks = 0;     // workgroups of one key/value head and one span (of one sequence)
    int key_waves = 4;
    int tiles = 1;      // of 16 rows, per wave
    int span = 0;
    int spans = 0;      // results per row that this part leaves
    int beside = 8;     // units (span, sequence, key/value head) whose row blocks alternate in the order of the workgroups; a multiple of 8
};
// For division by a number that the host knows.  A kernel's own division takes some 150 cycles, and a workgroup has nine before its first load.
inline unsigned reciprocal(unsigned by) { return 0xffffffffu / by; }
struct AttnArgs {
    const void *k, *v;  // of the layer: [pages, kv, page, D]
    const float *q;
    float *y;
    float *part, *stat;  // [rows][spans] x [D] and x [2], rows = tokens x heads; nullptr: one span in all, straight to y
    const int *tables, *starts, *lens;
    long long q_stride, y_stride;
    float scale;         // with log2 e
    int tokens, sequences, heads, kv, group, pages, page_shift, table_stride, max_len;
    int shared;          // positions
    AttnPart ahead, own;
    int chunk, chunks_ahead, chunks_own, pairs;  // the order of the workgroups: see paged_attn_kernel
    float per_group;
    unsigned by_group, by_kv, by_sequences, by_chunk, by_ahead, by_ahead_beside, by_own, by_own_beside, by_ahead_span, by_own_span;  // reciprocals
};
struct AttnPlan {
    AttnPart ahead, own;
    int spans() const { return ahead.spans + own.spans; }
    size_t workspace(long long tokens, int heads, int D) const {
        return spans() == 1 ? 0 : (size_t)tokens * heads * spans() * (D + 2) * sizeof(float);
    }
};
AttnPlan paged_attn_plan(bool half, int D, int heads, int kv, int sequences, long long tokens, int max_tokens, int max_len, int shared, int cus);
void paged_attn_launch_f16(int D, unsigned blocks, hipStream_t s, const AttnArgs &a);
void paged_attn_launch_f32(int D, unsigned blocks, hipStream_t s, const AttnArgs &a);
void paged_attn_launch(bool half, int D, int cus, hipStream_t s, AttnArgs a);  // and the merge of its spans

// ---- verify.h
struct VerifyArgs {
    const float *logits, *draft_probs, *temperatures, *uniforms;
    const int *starts, *tokens;
    int *out, *accepted;
    void *part;  // [rows][chunks] of VerifyStat, then [sequences][chunks] doubles
    long long logits_stride, draft_stride;
    int rows, vocab, sequences, chunks;
};
size_t verify_workspace(int rows, int sequences, int vocab);
void verify_launch(VerifyArgs a, hipStream_t s);

}  // namespace jitnn
