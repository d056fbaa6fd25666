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
// Two launches: the sequences by one workgroup (1024 at a time), then the
// rows, and where the result goes to arrays of its own the entries and pages
// that stay, by many.  Bound: the latency of the first launch, whose few reads
// wait for each other: lengths, entries, stack.
//
// Entries that come back and pages that go out are cut into runs of 16 within
// a sequence and the runs dealt to the waves in equal shares.  A lane finds
// one run's sequence in the sums, once for up to 1024 entries; four runs at a
// time are then read and written.  With a search for each entry the same 256
// prompts (10437 pages back, 13345 out) took 25.5 us instead of 19, and the
// search, not memory, was what took the time.  Two steps of four runs are in
// flight: more of them make this code longer, whose first fetch costs a small
// call more (2 / 4 / 8 / 16 steps: 64 sequences 8.6 / 9.1 / 10.0 / 11.1 us, 256
// prompts 19.1 / 18.3 / 18.8 / 16.7).
#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int KP_WG = 1024, KP_WAVES = KP_WG / 64, KP_ROWS = 256;
constexpr int KP_RUN = 16, KP_PER = 2;

// Inclusive sums of N numbers over the workgroup's threads, and their totals.
template <typename T, int N> __device__ __forceinline__ void group_upto(T (&v)[N], T (&total)[N], T (*s_wave)[KP_WAVES])
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_upto(v[i]);
    __syncthreads();
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) s_wave[i][wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const T all = wave_upto(lane < KP_WAVES ? s_wave[i][lane] : T(0));
        v[i] += wave ? of_lane(all, wave - 1) : T(0);
        total[i] = of_lane(all, KP_WAVES - 1);
    }
}

// The first of KP_WG ascending sums that exceeds k (it is there).
__device__ __forceinline__ int first_above(const uint32_t *upto, uint32_t k)
{
    int lo = 0;
#pragma unroll
    for (int step = KP_WG / 2; step > 0; step >>= 1)
        if (upto[lo + step - 1] <= k) lo += step;
    return lo;
}

struct SeqPlan {
    int n, held, stays, asks;
    int64_t first;
};
// Of the sequence of this thread, by all threads; rows: those of the sequences
// before the workgroup's, which it adds to.
__device__ __forceinline__ SeqPlan plan_seq(const KvPlanArgs &a, int b, int64_t &rows, int64_t (*s_wave)[KP_WAVES])
{
    const KvView &kv = a.kv;
    const bool is = b < kv.n_seq;
    const int at = is ? b : 0;
    // (all asked for before any is waited for)
    int n = a.n_new[at], len = a.len[at], held = a.in.held[at], shared = a.shared ? a.shared[at] : 0;
    asm volatile("" : "+v"(n), "+v"(len), "+v"(held), "+v"(shared));
    n = is ? max(n, 0) : 0;
    int64_t upto[1] = {n}, total[1];
    group_upto(upto, total, s_wave);
    SeqPlan s{};
    s.first = rows + upto[0] - n;
    rows += total[0];
    if (!is) return s;
    s.held = min(max(held, 0), kv.table_len);
    const bool ok = len >= 0 && n <= kv.cap && len <= kv.cap - n && s.first <= (int64_t)a.n_rows - n;
    s.n = ok ? n : 0;
    int need = 0;
    if (len > kv.cap)
        need = s.held;
    else if (len + s.n > 0)
        need = kv.page_of(len + s.n - 1) + 1;
    s.stays = min(s.held, max(need, shared));
    s.asks = s.n > 0 ? max(0, need - s.held) : 0;
    return s;
}

__device__ __forceinline__ uint32_t run_count(int entries) { return ((uint32_t)entries + KP_RUN - 1) / KP_RUN; }

// A wave's equal share of the runs.
struct Part {
    uint32_t begin, end;
    __device__ __forceinline__ Part(uint32_t runs, int wave)
    {
        constexpr uint32_t ONCE = 64 / KP_RUN;
        const uint32_t each = (runs + KP_WAVES * ONCE - 1) / (KP_WAVES * ONCE) * ONCE;
        begin = min(wave * each, runs);
        end = min(begin + each, runs);
    }
};

// The runs [r0, r0 + 64), one a lane; `upto`: runs up to and with a sequence's
// last, n: its entries, place: of its first in the table.
struct Runs {
    int left, place, nth;
    Runs() = default;
    __device__ __forceinline__ Runs(const uint32_t *upto, const uint32_t *last, const int *n, const int *place_of, uint32_t r0,
                                    uint32_t end)
    {
        const uint32_t r = min(r0 + (threadIdx.x & 63), end - 1);
        const int i = first_above(upto, r), of = n[i];
        const int done = (int)(run_count(of) - (upto[i] - r)) * KP_RUN;  // entries before the run's
        left = r0 + (threadIdx.x & 63) < end ? min(KP_RUN, of - done) : 0;
        place = place_of[i] + done;
        nth = (int)last[i] - of + done;
    }
    // Of the runs [j * 64 / KP_RUN, (j + 1) * 64 / KP_RUN): the lane's entry.
    __device__ __forceinline__ int entry(int j, int &at) const
    {
        const int from = j * (64 / KP_RUN) + (threadIdx.x & 63) / KP_RUN, i = threadIdx.x & (KP_RUN - 1);
        at = __shfl(nth, from) + i;
        const int p = __shfl(place, from) + i;
        return i < __shfl(left, from) ? p : -1;
    }
};

__global__ void __launch_bounds__(KP_WG) k_kv_plan(KvPlanArgs a)
{
    __shared__ int64_t s_rows[1][KP_WAVES];
    __shared__ uint32_t s_wave[3][KP_WAVES], s_runs[KP_WG], s_last[KP_WG];
    __shared__ int s_n[KP_WG], s_place[KP_WG];
    constexpr int ONCE = 64 / KP_RUN;
    const KvView &kv = a.kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int top = a.in.n_free[0];
    const bool one = kv.n_seq <= KP_WG;  // one round: what the first pass finds, the second has
    // entries that come back, in order
    int64_t rows = 0, back = 0;
    SeqPlan s{};
    uint32_t upto[3], total[3];  // runs that come back, runs that go out, entries that go out
    for (int c0 = 0; c0 < kv.n_seq; c0 += KP_WG) {
        s = plan_seq(a, c0 + tid, rows, s_rows);
        upto[0] = run_count(s.held - s.stays);
        upto[1] = run_count(s.asks);
        upto[2] = s.asks;
        group_upto(upto, total, s_wave);
        if (total[0] == 0) continue;
        s_runs[tid] = upto[0];
        s_n[tid] = s.held - s.stays;
        s_place[tid] = (int)((uint32_t)(c0 + tid) * (uint32_t)kv.table_len + (uint32_t)s.stays);
        s_last[tid] = 0;
        __syncthreads();
        const Part part(total[0], wave);
        int e[KP_PER], page[KP_PER];
        const auto read = [&](const Runs &runs, uint32_t r0, int j0) {
#pragma unroll
            for (int j = 0; j < KP_PER; j++) {
                int at;
                e[j] = r0 + (j0 + j) * ONCE < part.end ? runs.entry(j0 + j, at) : -1;
                page[j] = e[j] >= 0 ? a.in.table[e[j]] : -1;
            }
        };
        // pages that are some, of the wave's part and of those before it
        uint32_t found[1] = {0}, all[1];
        for (uint32_t r0 = part.begin; r0 < part.end; r0 += 64) {
            const Runs runs(s_runs, s_last, s_n, s_place, r0, part.end);
#pragma unroll 1
            for (int j0 = 0; j0 < KP_RUN && r0 + j0 * ONCE < part.end; j0 += KP_PER) {
                read(runs, r0, j0);
#pragma unroll
                for (int j = 0; j < KP_PER; j++) found[0] += (uint32_t)__popcll(__ballot((uint32_t)page[j] < (uint32_t)kv.n_pages));
            }
        }
        const uint32_t mine = found[0];
        found[0] = lane == 0 ? mine : 0;
        group_upto(found, all, s_wave);
        const int64_t before = min(max(top, 0), kv.n_pages) + back + of_lane(found[0], 0) - mine;
        uint32_t to = (uint32_t)min(before, (int64_t)kv.n_pages);  // (no more than 2^31 entries come back)
        back += all[0];
        for (uint32_t r0 = part.begin; r0 < part.end; r0 += 64) {
            const bool again = part.end - part.begin > KP_PER * ONCE;
            const Runs runs = again ? Runs(s_runs, s_last, s_n, s_place, r0, part.end) : Runs{};
#pragma unroll 1
            for (int j0 = 0; j0 < KP_RUN && r0 + j0 * ONCE < part.end; j0 += KP_PER) {
                if (again) read(runs, r0, j0);
#pragma unroll
                for (int j = 0; j < KP_PER; j++) {
                    const bool is = (uint32_t)page[j] < (uint32_t)kv.n_pages;
                    const uint64_t those = __ballot(is);
                    const uint32_t at = to + __builtin_amdgcn_mbcnt_hi((uint32_t)(those >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)those, 0));
                    if (e[j] >= 0) a.out.table[e[j]] = -1;
                    if (is && at < (uint32_t)kv.n_pages) a.out.free_pages[at] = page[j];
                    to += (uint32_t)__popcll(those);
                }
            }
        }
    }
    const int had = min(max(top, 0), kv.n_pages), high = (int)min((int64_t)kv.n_pages, had + back);
    // pages that go out
    rows = 0;
    int64_t asked = 0, taken = 0;
    for (int c0 = 0; c0 < kv.n_seq; c0 += KP_WG) {
        const int b = c0 + tid;
        if (!one) {
            s = plan_seq(a, b, rows, s_rows);
            upto[1] = run_count(s.asks);
            upto[2] = s.asks;
            group_upto(upto, total, s_wave);
        }
        const bool given = s.asks == 0 || asked + upto[2] <= high;
        if (b < kv.n_seq) {
            a.first[b] = (int)min(s.first, (int64_t)INT32_MAX);
            a.count[b] = given ? s.n : 0;
            a.out.held[b] = s.stays + (given ? s.asks : 0);
        }
        const int64_t room = high - asked;  // (those who are served come first)
        asked += total[2];
        if (total[2] == 0 || room <= 0) continue;
        __syncthreads();
        s_runs[tid] = upto[1];
        s_last[tid] = upto[2];
        s_n[tid] = s.asks;
        s_place[tid] = (int)((uint32_t)b * (uint32_t)kv.table_len + (uint32_t)s.held);
        __syncthreads();
        uint32_t items = total[2], served = total[1];
        if (items > room) {  // up to the last that is served
            const int i = first_above(s_last, (uint32_t)room);
            items = i ? s_last[i - 1] : 0;
            served = i ? s_runs[i - 1] : 0;
        }
        const Part part(served, wave);
        for (uint32_t r0 = part.begin; r0 < part.end; r0 += 64) {
            const Runs runs(s_runs, s_last, s_n, s_place, r0, part.end);
#pragma unroll 1
            for (int j0 = 0; j0 < KP_RUN && r0 + j0 * ONCE < part.end; j0 += KP_PER) {
                int e[KP_PER], page[KP_PER], at[KP_PER];
#pragma unroll
                for (int j = 0; j < KP_PER; j++) {
                    e[j] = r0 + (j0 + j) * ONCE < part.end ? runs.entry(j0 + j, at[j]) : -1;
                    at[j] = high - 1 - (int)taken - at[j];
                    page[j] = e[j] < 0 ? 0 : at[j] < had ? a.in.free_pages[at[j]] : a.out.free_pages[at[j]];
                }
#pragma unroll
                for (int j = 0; j < KP_PER; j++)
                    if (e[j] >= 0) {
                        a.out.table[e[j]] = page[j];
                        a.out.free_pages[at[j]] = -1;
                    }
            }
        }
        taken += items;
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
