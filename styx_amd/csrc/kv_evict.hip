// kv_evict.hip -- the rows of least accumulated attention weight leave a
// batch's paged KV cache.
//
// Per sequence with n = len > trigger rows and kv head: the `keep` rows of
// the largest weight stay, rows of the `recent` newest positions and of the
// first `sinks` positions before all others, ties to the lower slot.  The
// attention does not ask in which order rows lie, so nothing is compacted:
// a row that leaves a slot below `keep` makes a hole, a row that stays at or
// past `keep` moves into one (both ascending), and no other row is touched.
// Sources and targets of the moves are apart, so they need no order among
// them and the call may be made again on the same lists.
//
// Bound: latency (a selection has to see all weights before its first
// move) and, for long caches, HBM: 8 bytes of weight and position per row
// read, 2 rows of K and V read and written per move.
//
// A selecting launch (four for caches of more than 16K slots) leaves lists of
// holes and movers, and which slots stay; a moving launch does the rest.
//
// Measured: one conversation of 1088 rows cut to 1024, 4 kv heads, 6.9 + 4 us;
// 32 of up to 9001 f16 rows cut to 4096, 14.5 + 25 us, of which the moves
// run at 3.8 TB/s where the call runs alone (behind an attention call that has
// read such a batch's rows, as in use, the moves take 47); two of 65536 f32 rows, 8 kv heads, cut to 16384, 41 us in
// four launches, then 88 us of moves (4.6 TB/s, a large copy's rate).
#include <algorithm>
#include <type_traits>

#include "attn_batch.h"
#include "lanes.h"

namespace styx {

constexpr int EV_WG = 1024, EV_WAVES = EV_WG / 64;
constexpr int EV_KPT = 16;                // most keys of a thread, in registers
constexpr int EV_PART = EV_WG * EV_KPT;   // most slots that a workgroup selects from
constexpr int EV_BINS = 2048, EV_COPIES = 4;
constexpr int EV_LDS = (EV_COPIES + 2) * EV_BINS;
constexpr int EV_HIST = 2 * EV_BINS + EV_BINS / 2;  // bins of a part's three passes
constexpr int MV_WG = 256, MV_DEEP = 4, CP_SLOTS = 1024;
typedef unsigned long long u64;
// for the lambdas that touch a thread's array of keys, which a call would
// put into memory
#define EV_INLINE __attribute__((always_inline))

// A row's key: weights in order, NaN below all; rows that stay anyway above all.
__device__ __forceinline__ uint32_t evict_key(const KvEvictArgs &a, float weight, int32_t pos, int64_t newest)
{
    const float w = weight + 0.0f;  // -0 is 0
    if (pos > newest - a.recent || pos < a.sinks) return 0xFFFFFFFFu;
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Sum of the earlier waves' v (uniform in a wave), *total that of all.  Every
// thread takes part.
__device__ __forceinline__ int waves_before(int v, int wave, int *s, int *total = nullptr)  // s [EV_WAVES]
{
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[wave] = v;
    __syncthreads();
    int sum = 0, all = 0;
#pragma unroll
    for (int w = 0; w < EV_WAVES; w++) {
        sum += w < wave ? s[w] : 0;
        all += s[w];
    }
    if (total) *total = all;
    return sum;
}

// f(I) for I = 0 .. N - 1, each a constant of its own: arrays indexed by it
// stay in registers.
template <int N, int I = 0, typename F> __device__ __forceinline__ void unrolled(F f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        unrolled<N, I + 1>(f);
    }
}

// The radix selection's passes: 11, 11 and 10 bits.
__host__ __device__ constexpr int pass_shift(int p) { return p == 0 ? 21 : p == 1 ? 10 : 0; }
__host__ __device__ constexpr int pass_bins(int p) { return p == 2 ? EV_BINS / 2 : EV_BINS; }
__host__ __device__ constexpr uint32_t pass_mask(int p) { return p == 0 ? 0u : p == 1 ? 0xFFE00000u : 0xFFFFFC00u; }

// The keys of up to EV_WG * KPT slots from t0 on, the waves each a contiguous run
// of rows of 64 slots, a lane one slot of each row.
template <int KPT> struct EvKeys {
    uint32_t key[KPT];
    int per, first, end, lane;  // rows of a wave, its first slot, the slots' end
    __device__ __forceinline__ void load(const KvEvictArgs &a, int64_t base, int t0, int t1, int wave, int64_t newest)
    {
        lane = threadIdx.x & 63;
        per = (t1 - t0 + EV_WG - 1) / EV_WG;
        first = t0 + wave * per * 64;
        end = t1;
        // all loads on every path, rows past the wave's at its last slot: with
        // a branch for each row they were waited for one by one
        float w[KPT];
        int32_t p[KPT];
#pragma unroll
        for (int j = 0; j < KPT; j++) {
            const int t = min(first + 64 * min(j, per - 1) + lane, t1 - 1);
            w[j] = a.acc_in[base + t];
            p[j] = a.pos_in[base + t];
        }
#pragma unroll
        for (int j = 0; j < KPT; j++) key[j] = evict_key(a, w[j], p[j], newest);
    }
    // f(row, key, whether there is one), the wave's lanes together
    template <typename F> __device__ __forceinline__ void each(F f) const
    {
        unrolled<KPT>([&](auto j) EV_INLINE {
            if (j < per) f((int)j, key[j], first + 64 * j + lane < end);
        });
    }
    // Keys that match the prefix counted by their next digit.
    __device__ __forceinline__ void count(int pass, uint32_t prefix, uint32_t *h) const
    {
        const int shift = pass_shift(pass), bins = pass_bins(pass);
        const uint32_t mask = pass_mask(pass);
        each([&](int, uint32_t k, bool there) EV_INLINE {
            if (there && (k & mask) == prefix) atomicAdd(&h[(k >> shift) & (bins - 1)], 1u);
        });
    }
    // Lane j: the mask of row j's slots that stay: keys above the prefix, and
    // of those that equal it the first `need` (`ties` were before these).
    __device__ __forceinline__ u64 masks(uint32_t prefix, bool all_ties, int need, int ties) const
    {
        u64 mine = 0;
        const u64 below = (1ull << lane) - 1;
        each([&](int j, uint32_t k, bool there) EV_INLINE {
            bool stays = there && k >= prefix;
            if (!all_ties) {
                const bool tie = there && k == prefix;
                const u64 m = __ballot(tie);
                stays = stays && (!tie || ties + __popcll(m & below) < need);
                ties += __popcll(m);
            }
            const u64 m = __ballot(stays);
            if (lane == j) mine = m;
        });
        return mine;
    }
    // The slots below `keep` of lane j's row, and those that there are.
    __device__ __forceinline__ u64 low(int keep) const
    {
        const int k = keep - (first + 64 * lane);
        return lane >= per || k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1;
    }
    // f(slot, rank) for the bits of the rows' masks (lane j's: row j's), ranks
    // from `rank` on.
    template <typename F> __device__ __forceinline__ void emit(u64 p, int rank, F f) const
    {
        const int c = (int)__popcll(p), before = wave_upto(c) - c + rank;
        u64 rows = __ballot(c > 0);
        while (rows) {
            const int j = __builtin_ctzll(rows);
            rows &= rows - 1;
            const u64 m = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), j) << 32 |
                          (uint32_t)__builtin_amdgcn_readlane((int)p, j);
            const int r = __builtin_amdgcn_readlane(before, j) + __popcll(m & ((1ull << lane) - 1));
            if ((m >> lane) & 1) f(first + 64 * j + lane, r);
        }
    }
};

// The selection so far: the need-th largest of the `equal` keys that match
// the prefix is looked for.
struct EvPick {
    uint32_t prefix;
    int need, equal;
    // One digit: c0, c1 the numbers in thread i's bins 2 i and 2 i + 1 from
    // the top.  Every thread takes part; s [EV_WAVES], o [3].
    __device__ __forceinline__ int digit(int pass, int c0, int c1, int wave, int *s, int *o)
    {
        const int top = pass_bins(pass) - 1 - 2 * (int)threadIdx.x, incl = wave_upto(c0 + c1);
        const int above = waves_before(of_lane(incl, 63), wave, s) + incl - c0 - c1;
        if (above < need && above + c0 + c1 >= need) {
            const bool second = above + c0 < need;
            o[0] = second ? top - 1 : top;
            o[1] = second ? above + c0 : above;
            o[2] = second ? c1 : c0;
        }
        __syncthreads();
        prefix |= (uint32_t)o[0] << pass_shift(pass);
        need -= o[1];
        equal = o[2];
        return o[0];
    }
};

// Sequence and kv head of a selecting workgroup; keeps for the moving launch
// what it may not read any more, as it overwrites the lengths.
struct EvHead {
    int bk, b, n;
    bool act;
};
__device__ __forceinline__ EvHead evict_head(const KvEvictArgs &a, int bk, bool store)
{
    EvHead h;
    h.bk = bk;
    h.b = bk / a.kv.nkv;
    h.n = a.len[h.b];
    h.act = h.n > a.trigger && h.n <= a.kv.cap;
    if (store && threadIdx.x == 0) {
        if (bk % a.kv.nkv == 0) a.left[h.b] = make_int2(h.act ? a.keep : h.n, h.act);
        if (!h.act) a.moves[bk] = 0;
    }
    return h;
}

// Caches of up to EV_WG * KPT slots: one workgroup per sequence and kv head.  One
// CU does all of a head's work, so what counts are instructions per key and
// barriers.  The first pass counts every key, and weights of one size crowd
// into few bins: four copies of them, by lane, keep the adds of a wave apart.
template <int KPT> __global__ void __launch_bounds__(EV_WG) k_evict_select(KvEvictArgs a)
{
    // bins of the three passes
    __shared__ uint32_t hist[EV_LDS];
    __shared__ int s_cnt[EV_WAVES], s_out[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const EvHead hd = evict_head(a, blockIdx.x, true);
    if (!hd.act) return;
    for (int i = tid; i < EV_LDS; i += EV_WG) hist[i] = 0;
    EvKeys<KPT> k;
    k.load(a, (int64_t)hd.bk * a.kv.cap, 0, hd.n, wave, a.pos[hd.b]);
    EvPick pick{0, a.keep, 0};
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int copies = pass == 0 ? EV_COPIES : 1;
        uint32_t *bin = hist + (pass == 0 ? 0 : (EV_COPIES + pass - 1) * EV_BINS);
        __syncthreads();
        k.count(pass, pick.prefix, bin + (pass == 0 ? lane % EV_COPIES * EV_BINS : 0));
        __syncthreads();
        const int top = pass_bins(pass) - 1 - 2 * tid;
        int c0 = 0, c1 = 0;
        if (top > 0)
            for (int c = 0; c < copies; c++) {
                c0 += bin[c * EV_BINS + top];
                c1 += bin[c * EV_BINS + top - 1];
            }
        pick.digit(pass, c0, c1, wave, s_cnt, s_out);
    }
    const bool all_ties = pick.equal == pick.need;
    int ties = 0;
    if (!all_ties) {
        int eq = 0;
        k.each([&](int, uint32_t v, bool there) EV_INLINE { eq += __popcll(__ballot(there && v == pick.prefix)); });
        ties = waves_before(eq, wave, s_cnt);
    }
    const u64 stay = k.masks(pick.prefix, all_ties, pick.need, ties), low = k.low(a.keep);
    if (low) a.stay[(int64_t)hd.bk * a.stay_words + k.first / 64 + lane] = stay;
    const u64 holes = ~stay & low, movers = stay & ~low;
    // both counts in one sum: each is below 2^15
    int total;
    const int before = waves_before(wave_total((int)(__popcll(holes) | __popcll(movers) << 16)), wave, s_cnt, &total);
    int32_t *to = a.holes + (int64_t)hd.bk * a.keep, *from = a.movers + (int64_t)hd.bk * a.keep;
    k.emit(holes, before & 0xFFFF, [&](int t, int r) EV_INLINE { to[r] = t; });
    k.emit(movers, before >> 16, [&](int t, int r) EV_INLINE { from[r] = t; });
    if (tid == 0) a.moves[hd.bk] = total & 0xFFFF;
}

// Longer caches: a workgroup per part of EV_WG * KPT slots, the slots below keep
// and those from it on each in parts of their own, and a launch per pass of
// the selection (STAGE 0 to 2: the part's bins go to memory), with a last one
// for the lists.  Every workgroup forms the digits found so far from all
// parts' bins; from them also follow the numbers of rows that stay in the
// parts before its own, and with these the ranks of its holes or movers.
template <int STAGE, int KPT> __global__ void __launch_bounds__(EV_WG) k_evict_part(KvEvictArgs a)
{
    constexpr int PART = EV_WG * KPT;
    __shared__ uint32_t hist[STAGE == 0 ? EV_COPIES * EV_BINS : EV_BINS];
    __shared__ int s_cnt[EV_WAVES], s_out[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = blockIdx.x % a.parts, n_low = (a.keep + PART - 1) / PART;
    const EvHead hd = evict_head(a, blockIdx.x / a.parts, STAGE == 3 && part == 0);
    if (!hd.act) return;
    const bool lower = part < n_low;
    const int64_t t0 = lower ? (int64_t)part * PART : a.keep + (int64_t)(part - n_low) * PART;
    if (t0 >= hd.n) return;
    const int t1 = min((int64_t)(lower ? a.keep : hd.n), t0 + PART);
    const int parts = n_low + (hd.n - a.keep + PART - 1) / PART;  // of this head
    EvKeys<KPT> k;
    k.load(a, (int64_t)hd.bk * a.kv.cap, t0, t1, wave, a.pos[hd.b]);
    if constexpr (STAGE < 3)
        for (int i = tid; i < (STAGE == 0 ? EV_COPIES : 1) * EV_BINS; i += EV_WG) hist[i] = 0;
    uint32_t *mine = a.bins + ((int64_t)hd.bk * a.parts + part) * EV_HIST;
    const uint32_t *all = a.bins + (int64_t)hd.bk * a.parts * EV_HIST;
    EvPick pick{0, a.keep, 0};
    // rows above the prefix in the parts of this part's kind before it; ties
    // in all parts before it, and in those before its kind
    int above = 0, ties = 0, ties_low = 0;
    const int kind = lower ? 0 : n_low;
#pragma unroll
    for (int pass = 0; pass < STAGE; pass++) {
        const int top = pass_bins(pass) - 1 - 2 * tid;
        int c[2] = {0, 0}, bef[2] = {0, 0}, lo[2] = {0, 0};
        if (top > 0)
            for (int q0 = 0; q0 < parts; q0 += 8) {
                uint2 v[8];
#pragma unroll
                for (int j = 0; j < 8; j++)
                    v[j] = *(const uint2 *)(all + (int64_t)min(q0 + j, parts - 1) * EV_HIST + pass * EV_BINS + top - 1);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int q = q0 + j, w[2] = {q < parts ? (int)v[j].y : 0, q < parts ? (int)v[j].x : 0};
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        c[i] += w[i];
                        bef[i] += q < part ? w[i] : 0;
                        lo[i] += q < kind ? w[i] : 0;
                    }
                }
            }
        const int d = pick.digit(pass, c[0], c[1], wave, s_cnt, s_out);
        if (STAGE == 3) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                above += top - i > d ? bef[i] - lo[i] : 0;
                if (pass == 2 && top - i == d) {
                    ties += bef[i];
                    ties_low += lo[i];
                }
            }
        }
        __syncthreads();
    }
    if constexpr (STAGE < 3) {
        __syncthreads();
        k.count(STAGE, pick.prefix, hist + (STAGE == 0 ? lane % EV_COPIES * EV_BINS : 0));
        __syncthreads();
        for (int i = tid; i < pass_bins(STAGE); i += EV_WG) {
            uint32_t v = hist[i];
            if (STAGE == 0)
                for (int c = 1; c < EV_COPIES; c++) v += hist[c * EV_BINS + i];
            mine[STAGE * EV_BINS + i] = v;
        }
    } else {
        int all_above, all_ties_before, all_ties_low;
        waves_before(wave_total(above), wave, s_cnt, &all_above);
        waves_before(wave_total(ties), wave, s_cnt, &all_ties_before);
        waves_before(wave_total(ties_low), wave, s_cnt, &all_ties_low);
        const bool all_ties = pick.equal == pick.need;
        int eq = 0;
        if (!all_ties)
            k.each([&](int, uint32_t v, bool there) EV_INLINE { eq += __popcll(__ballot(there && v == pick.prefix)); });
        const int eq_before = waves_before(eq, wave, s_cnt);
        const u64 stay = k.masks(pick.prefix, all_ties, pick.need, all_ties_before + eq_before), low = k.low(a.keep);
        if (low) a.stay[(int64_t)hd.bk * a.stay_words + k.first / 64 + lane] = stay;
        // rows that stay in this kind's parts before this one
        const int stays = all_above + min(pick.need, all_ties_before) - min(pick.need, all_ties_low);
        const u64 out = lower ? ~stay & low : stay;
        int total;
        const int before = waves_before(wave_total((int)__popcll(out)), wave, s_cnt, &total);
        const int rank = lower ? (int)t0 - stays : stays;
        int32_t *list = (lower ? a.holes : a.movers) + (int64_t)hd.bk * a.keep;
        k.emit(out, rank + before, [&](int t, int r) EV_INLINE { list[r] = t; });
        if (part == parts - 1 && tid == 0) a.moves[hd.bk] = rank + total;
    }
}

// The moves of a list: weight and position by one lane, the rows of K and V
// by ROW16 lanes, MV_DEEP moves in flight for each; workgroups past
// move_tiles per head: weights and positions of the rows that lie still,
// where these go to other buffers.  (Rows stored with non-temporal stores: 22
// us instead of 25 where the call runs alone, but 57 behind an attention call
// that has read the rows, as in use, where plain stores took 49 and, since
// there are 32 workgroups per CU, take 47.)
template <int ROW16>  // 16-byte pieces of a row
__global__ void __launch_bounds__(MV_WG) k_evict_move(KvEvictArgs a)
{
    constexpr int GROUPS = MV_WG / ROW16, STEP = GROUPS * MV_DEEP;
    const KvView &kv = a.kv;
    const int tiles = a.move_tiles + a.copy_tiles, bk = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const int b = bk / kv.nkv, kvh = bk % kv.nkv, tid = threadIdx.x;
    const int64_t base = (int64_t)bk * kv.cap;
    if (tile >= a.move_tiles) {
        const int2 left = a.left[b];  // the new length, whether rows leave
        const int n = left.x > kv.cap ? 0 : left.x;
        const u64 *stay = a.stay + (int64_t)bk * a.stay_words;
        const int s0 = (tile - a.move_tiles) * CP_SLOTS + tid;
#pragma unroll
        for (int j = 0; j < CP_SLOTS / MV_WG; j++) {
            const int s = s0 + j * MV_WG;
            if (s < n && (!left.y || (stay[s / 64] >> (s & 63)) & 1)) {
                a.acc_out[base + s] = a.acc_in[base + s];
                a.pos_out[base + s] = a.pos_in[base + s];
            }
        }
        return;
    }
    if (tile == 0 && kvh == 0 && tid == 0) a.len_out[b] = a.left[b].x;
    const int moves = a.moves[bk];
    const int32_t *tab = kv.table + (int64_t)b * kv.table_len;
    const int32_t *to = a.holes + (int64_t)bk * a.keep, *from = a.movers + (int64_t)bk * a.keep;
    const int64_t stride = (int64_t)kv.nkv * ROW16;
    const int group = tid / ROW16, piece = kvh * ROW16 + tid % ROW16;
    const styx_u4 *kp = (const styx_u4 *)kv.kpool + piece, *vp = (const styx_u4 *)kv.vpool + piece;
    styx_u4 *kd = (styx_u4 *)kv.kpool + piece, *vd = (styx_u4 *)kv.vpool + piece;
    for (int i0 = tile * STEP; i0 < moves; i0 += a.move_tiles * STEP) {
        if (tid < STEP && i0 + tid < moves) {
            const int f = from[i0 + tid], t = to[i0 + tid];
            a.acc_out[base + t] = a.acc_in[base + f];
            a.pos_out[base + t] = a.pos_in[base + f];
        }
        int f[MV_DEEP], t[MV_DEEP];
        styx_u4 k[MV_DEEP], v[MV_DEEP];
#pragma unroll
        for (int j = 0; j < MV_DEEP; j++) {
            const int i = min(i0 + group + j * GROUPS, moves - 1);
            f[j] = from[i];
            t[j] = to[i];
        }
#pragma unroll
        for (int j = 0; j < MV_DEEP; j++) {
            f[j] = kv.row(tab, f[j]);
            t[j] = i0 + group + j * GROUPS < moves ? kv.row(tab, t[j]) : -1;
        }
#pragma unroll
        for (int j = 0; j < MV_DEEP; j++) {
            k[j] = kp[max(f[j], 0) * stride];
            v[j] = vp[max(f[j], 0) * stride];
        }
#pragma unroll
        for (int j = 0; j < MV_DEEP; j++)
            if (f[j] >= 0 && t[j] >= 0) {
                kd[t[j] * stride] = k[j];
                vd[t[j] * stride] = v[j];
            }
    }
}

// Keys of a selecting thread, and parts of a head.  Parts of 4K slots where
// 16K would not give every CU one: 16 heads of 64K rows, 61 us with 16K in
// the four launches, 41 with 4K.
static int parts_in(int cap, int keep, int part) { return (keep - 1) / part + (cap - keep + part - 1) / part + 1; }
static int keys_of(int64_t heads, int cap, int keep)
{
    if (cap <= EV_PART) return cap <= 4 * EV_WG ? 4 : 16;
    return heads * parts_in(cap, keep, EV_PART) < 256 ? 4 : 16;
}
static int parts_of(int64_t heads, int cap, int keep)
{
    return cap <= EV_PART ? 1 : parts_in(cap, keep, keys_of(heads, cap, keep) * EV_WG);
}

// In 4-byte words: the lists, the masks of what stays, lengths, moves, bins.
uint64_t kv_evict_ws_bytes(int n_seq, int nkv, int cap, int keep)
{
    const uint64_t heads = (uint64_t)n_seq * nkv, parts = parts_of(heads, cap, keep);
    return 4 * (2 * heads * ((keep + 63) / 64) + 2 * (uint64_t)n_seq + (heads + 1) / 2 * 2 + 2 * heads * keep +
                (parts > 1 ? heads * parts * EV_HIST : 0));
}

static void evict_tiles(KvEvictArgs &a)
{
    const KvView &kv = a.kv;
    const int heads = kv.n_seq * kv.nkv, most = std::min(a.keep, kv.cap - a.keep);
    const int step = MV_WG / (kv.hd * (kv.f16 ? 2 : 4) / 16) * MV_DEEP;
    // 32 workgroups per CU, of which 8 run at once, or one for every step of
    // the longest list: 39.2 us in all for 32 conversations, where 16 take
    // 39.9; two of 64K rows take the same with either, and more gain nothing
    a.move_tiles = std::max(1, std::min((most + step - 1) / step, 8192 / heads));
    // rows that lie still are copied only into other buffers
    const bool apart = a.acc_out != a.acc_in || a.pos_out != a.pos_in;
    a.copy_tiles = apart ? (std::min(a.trigger, kv.cap) + CP_SLOTS - 1) / CP_SLOTS : 0;
    a.parts = parts_of(heads, kv.cap, a.keep);
}
int64_t kv_evict_grid(KvEvictArgs a)
{
    evict_tiles(a);
    const int64_t heads = (int64_t)a.kv.n_seq * a.kv.nkv;
    // (a part's workgroup is four of the others' size)
    return heads * std::max<int64_t>(a.move_tiles + a.copy_tiles, 4 * (int64_t)a.parts);
}

template <int KPT> static void launch_parts(hipStream_t st, const KvEvictArgs &a, int64_t heads)
{
    const dim3 grid((unsigned)(heads * a.parts));
    hipLaunchKernelGGL((k_evict_part<0, KPT>), grid, dim3(EV_WG), 0, st, a);
    hipLaunchKernelGGL((k_evict_part<1, KPT>), grid, dim3(EV_WG), 0, st, a);
    hipLaunchKernelGGL((k_evict_part<2, KPT>), grid, dim3(EV_WG), 0, st, a);
    hipLaunchKernelGGL((k_evict_part<3, KPT>), grid, dim3(EV_WG), 0, st, a);
}

hipError_t launch_kv_evict(hipStream_t st, KvEvictArgs a, void *ws)
{
    const KvView &kv = a.kv;
    const int64_t heads = (int64_t)kv.n_seq * kv.nkv;
    evict_tiles(a);
    a.stay_words = (a.keep + 63) / 64;
    a.stay = (u64 *)ws;
    a.left = (int2 *)(a.stay + heads * a.stay_words);
    a.moves = (int32_t *)(a.left + kv.n_seq);
    a.holes = a.moves + (heads + 1) / 2 * 2;
    a.movers = a.holes + heads * a.keep;
    a.bins = (uint32_t *)(a.movers + heads * a.keep);
    const int keys = keys_of(heads, kv.cap, a.keep);
    if (a.parts == 1) {
        if (keys == 4)
            hipLaunchKernelGGL(k_evict_select<4>, dim3((unsigned)heads), dim3(EV_WG), 0, st, a);
        else
            hipLaunchKernelGGL(k_evict_select<16>, dim3((unsigned)heads), dim3(EV_WG), 0, st, a);
    } else if (keys == 4) {
        launch_parts<4>(st, a, heads);
    } else {
        launch_parts<16>(st, a, heads);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)(heads * (a.move_tiles + a.copy_tiles)));
    switch (kv.hd * (kv.f16 ? 2 : 4) / 16) {
    case 8: hipLaunchKernelGGL(k_evict_move<8>, grid, dim3(MV_WG), 0, st, a); break;
    case 16: hipLaunchKernelGGL(k_evict_move<16>, grid, dim3(MV_WG), 0, st, a); break;
    case 32: hipLaunchKernelGGL(k_evict_move<32>, grid, dim3(MV_WG), 0, st, a); break;
    default: hipLaunchKernelGGL(k_evict_move<64>, grid, dim3(MV_WG), 0, st, a); break;
    }
    return hipGetLastError();
}

}  // namespace styx
