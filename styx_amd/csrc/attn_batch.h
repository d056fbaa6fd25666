// attn_batch.h -- what the operators on a batch's paged KV cache share: the
// cache as the kernels see it, and the arguments of the launches
// (attn_batch.hip, kv_evict.hip).
#pragma once

#include "common.h"

namespace styx {

// Quotients by the page size without a division: t / d = umulhi(2 t, mul) >> sh
// for 0 <= t < 2^31 (sh = ceil(log2 d), mul = ceil(2^(31 + sh) / d) <= 2^32 - 1
// but for d = 1, where mul = 2^31: the error t (mul d - 2^(31+sh)) < 2^31 d
// <= 2^(31+sh) never carries the quotient over).
struct PageDiv {
    uint32_t mul;
    int sh;
    __device__ __forceinline__ int of(int t) const { return (int)(__umulhi(2u * (uint32_t)t, mul) >> sh); }
};
inline PageDiv page_div(uint32_t d)
{
    PageDiv p{0, 0};
    while ((1ull << p.sh) < d) p.sh++;
    p.mul = (uint32_t)(((1ull << (31 + p.sh)) + d - 1) / d);
    return p;
}

struct KvView {
    void *kpool, *vpool;  // [n_pages][page_tokens][nkv][hd] f32 or f16
    const int32_t *table; // [n_seq][table_len]
    int f16, n_seq, nkv, hd, page_tokens, n_pages, table_len;
    int cap;              // slots of a sequence: table_len * page_tokens
    PageDiv div;

    // Page-table entry of slot t, and the row of the pools that it makes: -1
    // where the page is not one of the pool's.
    __device__ __forceinline__ int page_of(int t) const
    {
        return (int)(__umulhi(2u * (uint32_t)t, div.mul) >> div.sh);
    }
    __device__ __forceinline__ int entry(const int32_t *tab, int t) const { return tab[page_of(t)]; }
    __device__ __forceinline__ int row_of(int e, int t) const
    {
        return (uint32_t)e < (uint32_t)n_pages ? e * page_tokens + (t - page_of(t) * page_tokens) : -1;
    }
    __device__ __forceinline__ int row(const int32_t *tab, int t) const { return row_of(entry(tab, t), t); }
};

struct AttnBatchArgs {
    KvView kv;
    const int32_t *len, *pos;
    const float *q, *k, *v, *q_norm, *k_norm;
    const double2 *rope;
    int n_rope, nh, gqa;
    float eps, scale, decay;
    const float *acc_in;
    float *acc_out;
    int32_t *slot_pos;
    float *out;
    // workspace: partials of the pieces, scores of every query head, the split
    float *part_ml, *part_o, *score;
    uint32_t *plan;
    int stride;  // slots of a score row (a multiple of 64)
    int n_merge, tiles;  // the joining launch's workgroups (filled by the launch)
    uint32_t once_units; // units of rows that the Infinity Cache holds (filled by the launch)
};

// Sizes of the workspace's pieces in floats for a cache of this shape.
struct AttnBatchWs {
    int64_t ml, o, plan, score;
    int64_t units, grid, join;  // units of rows at most, workgroups of the two launches
    int stride, tiles, dims;
};
AttnBatchWs attn_batch_ws(int n_seq, int nkv, int hd, int cap, int gqa, bool scored);
hipError_t launch_attn_batch(hipStream_t st, AttnBatchArgs a, float *ws);

// Most slots of a sequence that rows are evicted from: its parts all read each
// other's bins, which takes the square of their number (4096 at most).
constexpr int EVICT_MAX_CAP = 1 << 26;

struct KvEvictArgs {
    KvView kv;
    const int32_t *len, *pos;
    int trigger, keep, recent, sinks;
    const float *acc_in;
    float *acc_out;
    const int32_t *pos_in;
    int32_t *pos_out;
    int32_t *len_out;
    // workspace (filled by the launch)
    unsigned long long *stay; // [n_seq][nkv][stay_words] whether a slot below keep keeps its row
    int2 *left;               // [n_seq] new length, whether rows leave
    int32_t *moves;           // [n_seq][nkv] how many holes and movers
    int32_t *holes, *movers;  // [n_seq][nkv][keep] ascending
    uint32_t *bins;           // long caches: of every part
    int stay_words, parts, move_tiles, copy_tiles;
};
uint64_t kv_evict_ws_bytes(int n_seq, int nkv, int cap, int keep);
// Workgroups of the largest launch, in such of 256 threads.
int64_t kv_evict_grid(KvEvictArgs a);
hipError_t launch_kv_evict(hipStream_t st, KvEvictArgs a, void *ws);

}  // namespace styx
