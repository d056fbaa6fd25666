// kv_plan.hip -- page tables and row maps of a step over a batch's paged KV
// cache.
//
// With P rows to a page, L = len[b], N = n_new[b] (0 where the sequence's rows
// or slots do not fit) and H = held[b]:
//   need  = ceil((L + N) / P), 0 for L < 0
//   stays = min(H, max(need, shared[b])); entries [stays, H) go to the stack
//   asks  = max(0, need - H); given while the sum of asks up to b is at most
//           the stack's height after all entries have come back
// so every number is a running sum over the sequences, and the result does
// not depend on an order of execution.
//
// Two launches: the sequences by one workgroup (1024 at a time; entries that
// come back and pages that go out are dealt to its threads one by one,
// whatever sequence they belong to), then the rows, and where the result goes
// to arrays of its own the entries and pages that stay, by many.
#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int KP_WG = 1024, KP_ROWS = 256;

// Inclusive sums over the workgroup's threads, and their total.
__device__ __forceinline__ int64_t group_upto(int64_t v, int64_t *s_wave, int64_t &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_upto(v);
    __syncthreads();
    if (lane == 63) s_wave[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < KP_WG / 64; w++) {
        before += w < wave ? s_wave[w] : 0;
        total += s_wave[w];
    }
    return before + v;
}

// The first of n ascending sums that exceeds k (it is there).
__device__ __forceinline__ int first_above(const int64_t *upto, int n, int64_t k)
{
    int lo = 0;
    for (int half = n; half > 0;) {
        const int step = half >> 1;
        if (upto[lo + step] <= k) {
            lo += step + 1;
            half -= step + 1;
        } else {
            half = step;
        }
    }
    return lo;
}

struct SeqPlan {
    int n, held, stays, asks;
    int64_t first;
};
__device__ __forceinline__ SeqPlan plan_seq(const KvPlanArgs &a, int b, int64_t first)
{
    const KvView &kv = a.kv;
    const int n = max(a.n_new[b], 0), len = a.len[b];
    SeqPlan s;
    s.first = first;
    s.held = min(max(a.in.held[b], 0), kv.table_len);
    const bool ok = len >= 0 && n <= kv.cap && len <= kv.cap - n && first <= (int64_t)a.n_rows - n;
    s.n = ok ? n : 0;
    int need = 0;
    if (len > kv.cap)
        need = s.held;
    else if (len + s.n > 0)
        need = kv.page_of(len + s.n - 1) + 1;
    s.stays = min(s.held, max(need, a.shared ? a.shared[b] : 0));
    s.asks = s.n > 0 ? max(0, need - s.held) : 0;
    return s;
}

__global__ void __launch_bounds__(KP_WG) k_kv_plan(KvPlanArgs a)
{
    __shared__ int64_t s_wave[KP_WG / 64], s_upto[KP_WG];
    __shared__ int s_from[KP_WG];
    const KvView &kv = a.kv;
    const int tid = threadIdx.x;
    const int had = min(max(a.in.n_free[0], 0), kv.n_pages);
    // entries that come back, in order
    int64_t rows = 0, back = 0;
    for (int c0 = 0; c0 < kv.n_seq; c0 += KP_WG) {
        const int b = c0 + tid;
        const bool is = b < kv.n_seq;
        const int64_t n = is ? max(a.n_new[b], 0) : 0;
        int64_t total, items;
        const int64_t upto = group_upto(n, s_wave, total);
        SeqPlan s{};
        if (is) s = plan_seq(a, b, rows + upto - n);
        rows += total;
        const int64_t mine = group_upto(s.held - s.stays, s_wave, items);
        if (items == 0) continue;
        s_upto[tid] = mine;
        s_from[tid] = s.held;
        __syncthreads();
        for (int64_t k0 = 0; k0 < items; k0 += KP_WG) {
            const int64_t k = k0 + tid;
            int page = -1;
            if (k < items) {
                // counted from the end of the sequence's entries
                const int i = first_above(s_upto, KP_WG, k);
                const int64_t e = (int64_t)(c0 + i) * kv.table_len + s_from[i] - (s_upto[i] - k);
                page = a.in.table[e];
                a.out.table[e] = -1;
            }
            const bool good = (uint32_t)page < (uint32_t)kv.n_pages;
            int64_t found;
            const int64_t at = had + back + group_upto(good, s_wave, found) - 1;
            if (good && at < kv.n_pages) a.out.free_pages[at] = page;
            back += found;
        }
    }
    const int high = (int)min((int64_t)kv.n_pages, had + back);
    // pages that go out
    rows = 0;
    int64_t asked = 0, taken = 0;
    for (int c0 = 0; c0 < kv.n_seq; c0 += KP_WG) {
        const int b = c0 + tid;
        const bool is = b < kv.n_seq;
        const int64_t n = is ? max(a.n_new[b], 0) : 0;
        int64_t total;
        const int64_t upto = group_upto(n, s_wave, total);
        SeqPlan s{};
        if (is) s = plan_seq(a, b, rows + upto - n);
        rows += total;
        const int64_t sum = asked + group_upto(s.asks, s_wave, total);
        asked += total;
        const bool given = s.asks == 0 || sum <= high;
        if (is) {
            a.first[b] = (int)min(s.first, (int64_t)INT32_MAX);
            a.count[b] = given ? s.n : 0;
            a.out.held[b] = s.stays + (given ? s.asks : 0);
        }
        const int64_t mine = group_upto(given ? s.asks : 0, s_wave, total);
        if (total == 0) continue;
        s_upto[tid] = mine;
        s_from[tid] = s.held + s.asks;
        __syncthreads();
        for (int64_t k = tid; k < total; k += KP_WG) {
            const int i = first_above(s_upto, KP_WG, k);
            const int at = high - 1 - (int)(taken + k);
            a.out.table[(int64_t)(c0 + i) * kv.table_len + s_from[i] - (s_upto[i] - k)] =
                at < had ? a.in.free_pages[at] : a.out.free_pages[at];
            a.out.free_pages[at] = -1;
        }
        taken += total;
    }
    if (tid == 0) a.out.n_free[0] = high - (int)taken;
}

// Workgroups below row_groups: rows.  The others, where `out` is not `in`:
// table entries that stay, then stack entries that stay.
__global__ void __launch_bounds__(KP_ROWS) k_kv_plan_rows(KvPlanArgs a, int row_groups)
{
    constexpr int HOLD = 1024;
    __shared__ int s_first[HOLD];
    const KvView &kv = a.kv;
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= row_groups) {
        const int64_t i = (int64_t)(blockIdx.x - row_groups) * KP_ROWS + tid, entries = (int64_t)kv.n_seq * kv.table_len;
        if (i < entries) {
            const int b = (int)(i / kv.table_len), e = (int)(i - (int64_t)b * kv.table_len);
            if (e < min(min(max(a.in.held[b], 0), kv.table_len), a.out.held[b])) a.out.table[i] = a.in.table[i];
        } else if (i - entries < min(min(max(a.in.n_free[0], 0), kv.n_pages), a.out.n_free[0])) {
            a.out.free_pages[i - entries] = a.in.free_pages[i - entries];
        }
        return;
    }
    const bool held = kv.n_seq <= HOLD;
    if (held) {
        for (int b = tid; b < kv.n_seq; b += KP_ROWS) s_first[b] = a.first[b];
        __syncthreads();
    }
    const int r = blockIdx.x * KP_ROWS + tid;
    if (r >= a.n_rows) return;
    // the last sequence that begins at or before the row (those without rows
    // begin where the next one does)
    int lo = 0;
    for (int n = kv.n_seq; n > 1;) {
        const int step = n >> 1, f = held ? s_first[lo + step] : a.first[lo + step];
        if (f <= r) lo += step;
        n = f <= r ? n - step : step;
    }
    const int i = r - a.first[lo];
    const bool mine = i >= 0 && i < a.count[lo];
    int at = -1;
    if (mine && a.row_at) {
        const int t = a.len[lo] + i, e = kv.page_of(t);
        // (the entries that stay are being copied meanwhile)
        const int32_t *table = e < min(max(a.in.held[lo], 0), a.out.held[lo]) ? a.in.table : a.out.table;
        at = kv.row_of(table[(int64_t)lo * kv.table_len + e], t);
    }
    if (a.row_seq) a.row_seq[r] = mine ? lo : -1;
    if (a.row_pos) a.row_pos[r] = mine ? a.pos[lo] + i : -1;
    if (a.row_at) a.row_at[r] = at;
}

static int64_t row_groups(const KvPlanArgs &a)
{
    return a.row_seq || a.row_pos || a.row_at ? ((int64_t)a.n_rows + KP_ROWS - 1) / KP_ROWS : 0;
}

int64_t kv_plan_grid(const KvPlanArgs &a)
{
    const int64_t copied = a.in.table == a.out.table ? 0 : (int64_t)a.kv.n_seq * a.kv.table_len + a.kv.n_pages;
    return row_groups(a) + (copied + KP_ROWS - 1) / KP_ROWS;
}

hipError_t launch_kv_plan(hipStream_t st, const KvPlanArgs &a)
{
    hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(KP_WG), 0, st, a);
    if (const int64_t grid = kv_plan_grid(a))
        hipLaunchKernelGGL(k_kv_plan_rows, dim3((unsigned)grid), dim3(KP_ROWS), 0, st, a, (int)row_groups(a));
    return hipGetLastError();
}

}  // namespace styx
