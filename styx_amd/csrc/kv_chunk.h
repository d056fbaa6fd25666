// kv_chunk.h -- arguments of the operators that bring new tokens of a batch
// into its paged KV cache (kv_plan.hip, kv_append.hip, attn_chunk.hip,
// kv_weigh.hip).
#pragma once

#include "attn_batch.h"

namespace styx {

// New tokens of a batch: token i of sequence b is row first[b] + i of q, k, v
// and out, and slot len[b] + i of the sequence.
struct ChunkView {
    int n_rows;
    const int32_t *first, *count, *len;
};
struct ChunkSeq {
    int first, count, len;  // count 0: skipped
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkView &c, const KvView &kv, int b)
{
    if (b >= kv.n_seq) return {0, 0, 0};
    const int f = c.first[b], n = c.count[b], l = c.len[b];
    // (differences of numbers that are not negative: nothing overflows)
    const bool ok = f >= 0 && n > 0 && l >= 0 && n <= c.n_rows && f <= c.n_rows - n && n <= kv.cap && l <= kv.cap - n;
    return {f, ok ? n : 0, l};
}

struct KvPages {
    int32_t *table, *held, *free_pages, *n_free;
};
struct KvPlanArgs {
    KvView kv;  // (pools and table unused)
    KvPages in, out;
    const int32_t *shared, *len, *n_new, *pos;
    int n_rows;
    int32_t *first, *count, *row_seq, *row_pos, *row_at;
};
int64_t kv_plan_grid(const KvPlanArgs &a);
hipError_t launch_kv_plan(hipStream_t st, const KvPlanArgs &a);

struct KvAppendArgs {
    KvView kv;
    int n_rows, nh;
    const int32_t *row_pos, *row_at;
    int in_f16, q_f16;
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv, ldo;
    const float *q_norm, *k_norm;
    float eps;
    const double2 *rope;  // [n_pos][n_rot / 2], or NULL
    int n_pos, n_rot, interleaved;
    void *q_out;
};
int64_t kv_append_grid(const KvAppendArgs &a);
hipError_t launch_kv_append(hipStream_t st, const KvAppendArgs &a);

struct AttnChunkArgs {
    KvView kv;
    ChunkView chunk;
    int nh, gqa, q_f16, window;
    const void *q;
    int64_t ldq, ldo;
    float scale;
    void *out;
    float *lse;
    PageDiv by_gqa;  // (filled by the launch, as is runs)
    int runs;        // a wave's rows of a block lie in one page
};
// Workgroups of the largest launch; bytes of the workspace.
int64_t attn_chunk_grid(int n_seq, int nkv, int gqa, int n_rows);
uint64_t attn_chunk_ws_bytes(int n_seq, int nkv, int hd, int gqa, int n_rows);
hipError_t launch_attn_chunk(hipStream_t st, AttnChunkArgs a, void *ws);

struct KvWeighArgs {
    KvView kv;
    ChunkView chunk;
    const int32_t *pos;
    int nh, gqa, q_f16, window, last;
    const void *q;
    int64_t ldq;
    float scale, decay;
    const float *lse, *acc_in;
    float *acc_out;
    int32_t *slot_pos;
    PageDiv by_gqa;  // (filled by the launch, as is few)
    int few;         // blocks of 32 slots for which a workgroup's waves share a block
};
int64_t kv_weigh_grid(const KvWeighArgs &a);
hipError_t launch_kv_weigh(hipStream_t st, KvWeighArgs a);

}  // namespace styx
