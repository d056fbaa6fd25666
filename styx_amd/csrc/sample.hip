// sample.hip -- the next token of each row of logits by temperature, top-k,
// top-p and min-p and a given random number.
//
// A word's weight is e^((x - max) / T) in whole units of 2^-44, so that sums
// are exact in whatever order they are formed and a result never depends on
// one (words below half a unit have weight 0 and are never chosen).  Words
// are ordered by logit, larger first, then by index.  top-k keeps the first
// k, top-p of those the shortest run from the first that holds `top_p` of
// their weight, min-p of those the words of at least `min_p` times the
// largest weight; the first word always stays.  With S the weight that is
// left and t = floor(u S), the token is the first word, in the order of the
// indices, at which the running sum exceeds t.
//
// Nothing is sorted.  Four launches over blocks of 2048 words:
//   1 the rows' largest logits
//   2 weight and number of the words in bins of about 1/64 of (max - x) / T
//   3 from these, the bins in which the k-th word and the end of the top-p
//     run lie: the words of those bins are listed, the weight that surely
//     stays is summed per block
//   4 one workgroup per row: the border words in their order, which of them
//     stay, and the token in its block
// Bound: latency, for a few rows (each launch waits for all of the one before)
// and in each workgroup of many.
//
// Measured: one row of 151936 words with top-k and top-p 2.6 + 5.2 + 6.2 + 8.7
// us, of 4096 with a temperature alone 13 us in all; 64 rows of 151936 with
// settings of their own 8 + 19 + 23 + 16 us (logits read three times, 1.8
// TB/s); 17 flat rows of 50257, a nucleus of most words, 30 us.  Of the 64
// rows, those that are greedy or that nothing cuts take no part in launch 2,
// and those with a top-p but no small top-k are weighed in both 2 and 3.
// Neither launch is bound by its VALU work: it takes 35 and 43% of the cycles
// (4 and 6 million instructions), and half of the waves' time is waiting.
// Launch 2's bins (48.5 KB of LDS) let three workgroups run on a CU where
// sample_ws plans about four, so they come in uneven rounds, 6.6 waves per CU
// on average (launch 3: 8.5), and every workgroup forms its row's settings
// from the blocks' first words, in launch 3 also the border from the bins,
// before it asks for its words.  (A wave per block of 512 words without
// barriers, the border found by a launch of its own, and words weighed four
// side by side were tried: each no faster over these.)
#include "../../include/styx_hip.h"
#include "lanes.h"
#include "sample.h"

#include <algorithm>

namespace styx {

constexpr int SA_WG = 256, FI_WG = 1024, FI_WAVES = FI_WG / 64;
constexpr int SA_BLOCK = 2048, SA_PER = SA_BLOCK / SA_WG;  // words of a block, of a thread
constexpr int FI_BLOCKS = (SAMPLE_MAX_N + SA_BLOCK - 1) / SA_BLOCK;
constexpr int FI_LIST = 2048;       // border words that are kept in LDS
constexpr int FI_PAIRS = FI_WG / 8;  // words that are ranked each against all, by 8 threads each
constexpr double SA_ONE = 17592186044416.0;  // 2^44
typedef unsigned long long u64;

// Order of the words: larger logit first, then lower index; 0: no candidate
// (NaN, -inf).
__device__ __forceinline__ u64 word_key(float x, uint32_t i)
{
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 is 0
    return (u64)(u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(u64 k)
{
    const uint32_t h = (uint32_t)(k >> 32);
    return __uint_as_float(h & 0x80000000u ? h ^ 0x80000000u : ~h);
}
__device__ __forceinline__ uint32_t key_index(u64 k) { return ~(uint32_t)k; }

struct RowAt {
    const float *x;
    u64 kmax;       // the first word
    float mx;
    float x_min;    // no word below it is one of the first k
    double inv_t, p, min_w;
    bool greedy, top_p, min_p;
    int k;          // 0: all
};

// The row's settings and, from the blocks' first words, its own; every wave
// by itself.  (The k-th largest of the blocks' first words has k words at or
// above it: none below it is one of the row's first k.  Looked for in its
// upper 16 bits, so a little lower.)
__device__ __forceinline__ RowAt row_at(const SampleArgs &a, int r)
{
    RowAt w;
    const styx_sample_params p = a.params[a.one_params ? 0 : r];
    const int lane = threadIdx.x & 63;
    u64 top[FI_BLOCKS / 64], k = 0;
#pragma unroll
    for (int j = 0; j < FI_BLOCKS / 64; j++) {
        const int c = lane + 64 * j;
        top[j] = c < a.blocks ? a.top[(int64_t)r * a.blocks + c] : 0;
        k = top[j] > k ? top[j] : k;
    }
    w.x = a.logits + r * a.ld;
    w.kmax = wave_most(k);
    w.mx = key_value(w.kmax);
    w.greedy = !(p.temperature > 0.0f);
    w.inv_t = 1.0 / (double)p.temperature;
    w.top_p = p.top_p < 1.0f;
    w.p = p.top_p;
    w.min_p = p.min_p > 0.0f;
    w.min_w = (double)p.min_p * SA_ONE;
    w.k = p.top_k > 0 && p.top_k < a.n ? p.top_k : 0;
    w.x_min = -INFINITY;
    if (w.k && w.k <= a.blocks) {
        uint32_t least = 0;
        for (uint32_t bit = 0x8000; bit; bit >>= 1) {
            int n = 0;
#pragma unroll
            for (int j = 0; j < FI_BLOCKS / 64; j++) n += __popcll(__ballot((uint32_t)(top[j] >> 48) >= (least | bit)));
            if (n >= w.k) least |= bit;
        }
        // (below every candidate's key, or a NaN's: fewer than k blocks have one)
        if (least > 0x007Fu) w.x_min = key_value((u64)least << 48);
    }
    return w;
}

// Weight of a candidate, and its bin: with k = rint(64 d / ln 2) the weight is
// 2^(44 - k/64) e^(k ln2/64 - d), the power from a table of 64 in LDS, the
// rest, of at most ln2/128, by its series to the fifth power (3e-17).  The
// product k ln2/64 is off by 2^-60 k, which reaches a thousandth of a unit
// nowhere.  14 operations in f64, where a library exponential takes three
// times as many.  Every launch must come to the same weights and bins:
// contraction is off.
__device__ __forceinline__ void fill_powers(double *pow)  // 64, by the first wave
{
    if (threadIdx.x < 64) pow[threadIdx.x] = exp2((double)threadIdx.x * (-1.0 / 64.0));
}
__device__ __forceinline__ u64 word_weight(const RowAt &w, const double *pow, float x, int *bin)
{
#pragma clang fp contract(off)
    constexpr double ROUND = 6755399441055744.0;  // 1.5 2^52: a sum with it is a whole number
    *bin = 0;
    if (x == w.mx) return (u64)SA_ONE;
    const double d = ((double)w.mx - (double)x) * w.inv_t;
    if (!(x > -INFINITY) || !(d < 31.5)) return 0;
    const double t = d * 92.33248261893498 + ROUND;  // 64 / ln 2
    const int k = (int)(uint32_t)__builtin_bit_cast(u64, t);
    const double s = __builtin_fma(t - ROUND, 0.010830424696249145, -d);  // ln 2 / 64
    double p = __builtin_fma(s, 1.0 / 120.0, 1.0 / 24.0);
    p = __builtin_fma(s, p, 1.0 / 6.0);
    p = __builtin_fma(s, p, 0.5);
    p = __builtin_fma(s, p, 1.0);
    p = __builtin_fma(s, p, 1.0);
    const u64 v = __builtin_bit_cast(u64, pow[k & 63] * p) + ((u64)(44 - (k >> 6)) << 52);
    *bin = k * 11 >> 4;  // k is at most 2909
    // rounded to a whole number by a sum with 2^52
    return __builtin_bit_cast(u64, __builtin_bit_cast(double, v) + 4503599627370496.0) - 0x4330000000000000ull;
}
__device__ __forceinline__ bool min_p_stays(const RowAt &w, u64 weight, float x, uint32_t i)
{
    return !w.min_p || (double)weight >= w.min_w || word_key(x, i) == w.kmax;
}

// f(block) for the blocks of this workgroup.
template <typename F> __device__ __forceinline__ void my_blocks(const SampleArgs &a, F f)
{
    const int b1 = min(a.blocks, (int)(blockIdx.x + 1) * a.per);
    for (int b = blockIdx.x * a.per; b < b1; b++) f(b);
}
// A thread's words of a block, all in flight at once: word SA_WG j + thread;
// words past the row are NaN.
__device__ __forceinline__ void load_block(const SampleArgs &a, const float *x, int b, float (&v)[SA_PER])
{
    const int i0 = b * SA_BLOCK + threadIdx.x;
#pragma unroll
    for (int j = 0; j < SA_PER; j++) v[j] = x[min(i0 + j * SA_WG, a.n - 1)];
#pragma unroll
    for (int j = 0; j < SA_PER; j++)
        if (i0 + j * SA_WG >= a.n) v[j] = __int_as_float(0x7FC00000);
}

// ------------------------------------------------------------- 1: largest --
__global__ void __launch_bounds__(SA_WG) k_sample_max(SampleArgs a)
{
    __shared__ u64 s[2][SA_WG / 64];
    const int r = blockIdx.y;
    // the row's bins, emptied by its workgroups together
    for (int i = blockIdx.x * SA_WG + threadIdx.x; i < SAMPLE_BINS; i += a.G * SA_WG) {
        a.hw[(int64_t)r * SAMPLE_BINS + i] = 0;
        a.hc[(int64_t)r * SAMPLE_BINS + i] = 0;
    }
    my_blocks(a, [&](int b) {
        float v[SA_PER];
        load_block(a, a.logits + r * a.ld, b, v);
        // a thread's first of its largest words (NaN and -inf are above
        // nothing); a third of the instructions of comparing keys
        float best = -INFINITY;
        int at = 0;
#pragma unroll
        for (int j = 0; j < SA_PER; j++) {
            const bool more = v[j] > best;
            best = more ? v[j] : best;
            at = more ? j * SA_WG : at;
        }
        u64 k = wave_most(word_key(best, b * SA_BLOCK + at + threadIdx.x));
        u64 *t = s[b & 1];  // (a block later than one whose reader may be behind)
        if ((threadIdx.x & 63) == 0) t[threadIdx.x >> 6] = k;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < SA_WG / 64; w++) k = t[w] > k ? t[w] : k;
            a.top[(int64_t)r * a.blocks + b] = k;
        }
    });
}

// ---------------------------------------------------------------- 2: bins --
__global__ void __launch_bounds__(SA_WG) k_sample_bins(SampleArgs a)
{
    // two copies by lane: logits in steps crowd into few bins
    __shared__ u64 hw[2 * SAMPLE_BINS];
    __shared__ uint32_t hc[2 * SAMPLE_BINS];
    __shared__ double pow[64];
    const int r = blockIdx.y;
    const RowAt w = row_at(a, r);
    if (w.kmax == 0 || w.greedy || !(w.top_p || w.k)) return;
    for (int i = threadIdx.x; i < 2 * SAMPLE_BINS; i += SA_WG) hw[i] = hc[i] = 0;
    fill_powers(pow);
    __syncthreads();
    my_blocks(a, [&](int b) {
        float v[SA_PER];
        load_block(a, w.x, b, v);
#pragma unroll
        for (int j = 0; j < SA_PER; j++) {
            if (!(v[j] >= w.x_min)) continue;
            int bin;
            const u64 m = word_weight(w, pow, v[j], &bin);
            if (m == 0) continue;
            bin += (threadIdx.x & 1) * SAMPLE_BINS;
            if (w.top_p) atomicAdd(&hw[bin], m);
            if (w.k) atomicAdd(&hc[bin], 1u);
        }
    });
    __syncthreads();
    for (int i = threadIdx.x; i < SAMPLE_BINS; i += SA_WG) {
        const u64 m = hw[i] + hw[SAMPLE_BINS + i];
        const uint32_t c = hc[i] + hc[SAMPLE_BINS + i];
        if (m) atomicAdd(&a.hw[(int64_t)r * SAMPLE_BINS + i], m);
        if (c) atomicAdd(&a.hc[(int64_t)r * SAMPLE_BINS + i], c);
    }
}

// -------------------------------------------------------------- 3: border --
// The bins that hold the border: words of bins below `sure` stay as far as
// top-k and top-p go; those of [sure, p_end] (top-p) and of k_bin (top-k)
// are looked at one by one; all others leave.
struct Border {
    int sure, p_end, k_bin;
    uint32_t k_count;
    u64 k_weight;   // weight and number (k_count) of the bins before k_bin
    u64 p_weight;   // weight of the bins before `sure`
    u64 total;      // of all bins
};

// All threads of the workgroup (NT of them) take part.
template <int NT> __device__ Border find_border(const SampleArgs &a, const RowAt &w, int r)
{
    constexpr int PER = SAMPLE_BINS / NT, NW = NT / 64;
    __shared__ u64 s_w[NW];
    __shared__ uint32_t s_c[NW];
    __shared__ Border s_b;
    __shared__ u64 s_lo, s_hi;
    if (!(w.top_p || w.k)) return {SAMPLE_BINS, -1, -1, 0, 0, 0, 0};
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u64 vw[PER], aw = 0;
    uint32_t vc[PER], ac = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        vw[j] = a.hw[(int64_t)r * SAMPLE_BINS + tid * PER + j];
        vc[j] = a.hc[(int64_t)r * SAMPLE_BINS + tid * PER + j];
        aw += vw[j];
        ac += vc[j];
    }
    u64 iw = wave_upto(aw);
    uint32_t ic = wave_upto(ac);
    if (lane == 63) {
        s_w[wave] = iw;
        s_c[wave] = ic;
    }
    __syncthreads();
    u64 total = 0;
    for (int q = 0; q < NW; q++) {
        if (q < wave) {
            iw += s_w[q];
            ic += s_c[q];
        }
        total += s_w[q];
    }
    // running sums before this thread's first bin
    const u64 w0 = iw - aw;
    const uint32_t k0 = ic - ac;
    if (tid == 0) {
        s_b = {SAMPLE_BINS, -1, -1, 0, 0, 0, total};
        s_lo = s_hi = total;
    }
    __syncthreads();
    if (w.k) {
        u64 rw = w0;
        uint32_t rc = k0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            // the k-th word lies here; where there are fewer, all stay
            if (rc < (uint32_t)w.k && rc + vc[j] >= (uint32_t)w.k) {
                s_b.k_bin = tid * PER + j;
                s_b.k_weight = rw;
                s_b.k_count = rc;
                s_b.sure = tid * PER + j;
                s_b.p_weight = rw;
                s_lo = rw;
                s_hi = rw + vw[j];
            }
            rw += vw[j];
            rc += vc[j];
        }
        __syncthreads();
    }
    if (w.top_p) {
        // the run ends at the first word before which at least top_p S lies;
        // S is between s_lo and s_hi
        const double lo = w.p * (double)s_lo, hi = w.p * (double)s_hi;
        u64 rw = w0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int bin = tid * PER + j;
            const bool first = bin == 0;
            const double before = (double)rw, upto = (double)(rw + vw[j]);
            if ((first || before < lo) && upto >= lo) {
                s_b.sure = bin;
                s_b.p_weight = rw;
            }
            if ((first || before < hi) && upto >= hi) s_b.p_end = bin;
            rw += vw[j];
        }
        __syncthreads();
    }
    return s_b;
}

__global__ void __launch_bounds__(SA_WG) k_sample_border(SampleArgs a)
{
    __shared__ u64 s_sum[SA_WG / 64];
    __shared__ uint32_t s_cnt[SA_WG / 64], s_n;
    __shared__ double pow[64];
    const int r = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const RowAt w = row_at(a, r);
    if (w.kmax == 0 || w.greedy) return;
    fill_powers(pow);
    const Border bd = find_border<SA_WG>(a, w, r);
    // words below x_lim lie past the last bin that matters: k rounds to one
    // of that bin's only up to (bin + 1) 16/11 + 1/2
    const int past = max(max(bd.p_end, bd.k_bin), bd.sure - 1) + 1;
    float x_lim = (float)((double)w.mx - (past * (16.0 / 11.0) + 2.0) / 92.33248261893498 / w.inv_t);
    x_lim = past >= SAMPLE_BINS || !(x_lim > -INFINITY) || w.mx == INFINITY ? -INFINITY : x_lim - fabsf(x_lim) * 1e-6f;
    x_lim = fmaxf(x_lim, w.x_min);
    my_blocks(a, [&](int b) {
        float v[SA_PER];
        load_block(a, w.x, b, v);
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        u64 sum = 0;
        uint32_t cnt = 0;
#pragma unroll
        for (int j = 0; j < SA_PER; j++) {
            const uint32_t at = j * SA_WG + threadIdx.x;
            if (!__any(v[j] >= x_lim)) continue;
            int bin;
            const u64 m = v[j] >= x_lim ? word_weight(w, pow, v[j], &bin) : 0;
            const bool border = m && bin >= bd.sure && (bin <= bd.p_end || bin == bd.k_bin);
            if (m && bin < bd.sure && min_p_stays(w, m, v[j], b * SA_BLOCK + at)) {
                sum += m;
                cnt++;
            }
            if (const u64 listed = __ballot(border)) {
                uint32_t base = 0;
                if (lane == __builtin_ctzll(listed)) base = atomicAdd(&s_n, (uint32_t)__popcll(listed));
                base = of_lane(base, __builtin_ctzll(listed));
                if (border)
                    a.list[((int64_t)r * a.blocks + b) * SA_BLOCK + base + __popcll(listed & ((1ull << lane) - 1))] = at;
            }
        }
        sum = wave_total(sum);
        cnt = wave_total(cnt);
        if (lane == 0) {
            s_sum[wave] = sum;
            s_cnt[wave] = cnt;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int q = 1; q < SA_WG / 64; q++) {
                sum += s_sum[q];
                cnt += s_cnt[q];
            }
            const int64_t o = (int64_t)r * a.blocks + b;
            a.sum[o] = sum;
            a.cnt[o] = cnt;
            a.lcnt[o] = s_n;
        }
        __syncthreads();
    });
}

// -------------------------------------------------------------- 4: finish --
// The border words of a row: key, and weight with the bin above 48 bits, in
// LDS where there are at most FI_LIST, else formed from the
// lists whenever they are looked at.
struct Words {
    const SampleArgs &a;
    const RowAt &w;
    int r, m;
    const uint32_t *s_cnt;  // [blocks]
    const double *pow;
    u64 *s_key, *s_val;     // [FI_LIST]
    __device__ __forceinline__ void word(int b, uint32_t at, u64 &k, u64 &v) const
    {
        const uint32_t i = b * SA_BLOCK + at;
        const float x = w.x[i];
        int bin;
        v = word_weight(w, pow, x, &bin) | (u64)bin << 48;
        k = word_key(x, i);
    }
    // f(key, weight and bin) for all words, over the workgroup's threads
    template <typename F> __device__ __forceinline__ void each(bool from_lists, F f) const
    {
        if (!from_lists) {
            for (int j = threadIdx.x; j < m; j += FI_WG) f(s_key[j], s_val[j]);
            return;
        }
        for (int b = threadIdx.x >> 6; b < a.blocks; b += FI_WAVES) {
            const uint16_t *list = a.list + ((int64_t)r * a.blocks + b) * SA_BLOCK;
            for (uint32_t j = threadIdx.x & 63; j < s_cnt[b]; j += 64) {
                u64 k, v;
                word(b, list[j], k, v);
                f(k, v);
            }
        }
    }
};
constexpr u64 WEIGHT = (1ull << 48) - 1;

// The last key that stays of the words in bins [b0, b1], of which those below
// `floor` do not count: the first `need_n` of them (BY_WEIGHT: the shortest
// run, the first word of the row at least, before whose end less than need_w
// lies; `base` lies before them all); *weight: all weight up to it.  A radix
// selection of 8 bits a pass, from the highest bit in which the words that
// are left differ, until at most FI_PAIRS are; these are ranked each against
// all.
struct Chosen {
    u64 key, weight;
};
// Sum over eight lanes.
template <typename T> __device__ __forceinline__ T eight_total(T v)
{
    v += by_words(v, [](uint32_t x) { return dpp_u<0xB1>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x4E>(x); });
    v += by_words(v, [](uint32_t x) { return dpp_u<0x141>(x); });
    return v;
}
template <bool BY_WEIGHT>
__device__ Chosen choose(const Words &ws, int b0, int b1, u64 floor, uint32_t need_n, u64 base, double need_w)
{
    __shared__ u64 bw[256], p_key[FI_PAIRS], p_val[FI_PAIRS], s_lo, s_hi, s_w, s_key, s_weight;
    __shared__ uint32_t bc[256], s_n, s_left, s_digit;
    const int tid = threadIdx.x, lane = tid & 63;
    u64 prefix = 0, mask = 0, before_w = base;
    uint32_t before_n = 0;
    const bool lists = ws.m > FI_LIST;
    auto in = [&](u64 k, u64 v) {
        const int bin = (int)(v >> 48);
        return bin >= b0 && bin <= b1 && k >= floor && (k & mask) == prefix;
    };
    // few words altogether: ranked where they lie
    const bool few = ws.m <= FI_PAIRS;
    while (!few) {
        if (tid == 0) {
            s_left = s_n = 0;
            s_lo = ~0ull;
            s_hi = 0;
        }
        if (tid < 256) bw[tid] = bc[tid] = 0;
        __syncthreads();
        u64 lo = ~0ull, hi = 0;
        uint32_t mine = 0;
        ws.each(lists, [&](u64 k, u64 v) {
            if (!in(k, v)) return;
            mine++;
            lo = k < lo ? k : lo;
            hi = k > hi ? k : hi;
        });
        mine = wave_total(mine);
        lo = ~wave_most(~lo);
        hi = wave_most(hi);
        if (lane == 0 && mine) {
            atomicAdd(&s_left, mine);
            atomicMin(&s_lo, lo);
            atomicMax(&s_hi, hi);
        }
        __syncthreads();
        if (s_left <= FI_PAIRS) break;
        const int top = 63 - __builtin_clzll(s_lo ^ s_hi), shift = top > 7 ? top - 7 : 0;
        ws.each(lists, [&](u64 k, u64 v) {
            if (!in(k, v)) return;
            atomicAdd(&bw[(k >> shift) & 255], v & WEIGHT);
            atomicAdd(&bc[(k >> shift) & 255], 1u);
        });
        __syncthreads();
        if (tid < 64) {
            // lane i: digits 255 - 4 i downwards
            u64 w4[4], sw = 0;
            uint32_t c4[4], sc = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                w4[j] = bw[255 - 4 * lane - j];
                c4[j] = bc[255 - 4 * lane - j];
                sw += w4[j];
                sc += c4[j];
            }
            u64 aw = before_w + wave_upto(sw) - sw;
            uint32_t an = before_n + wave_upto(sc) - sc;
            // the first digit whose words reach what is needed; should
            // rounding leave none, the last that has words
            int at = -1, any = -1;
            u64 at_w = 0, any_w = 0;
            uint32_t at_n = 0, any_n = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const bool reach = c4[j] && (BY_WEIGHT ? (double)(aw + w4[j]) >= need_w : an + c4[j] >= need_n);
                if (reach && at < 0) at = 255 - 4 * lane - j, at_w = aw, at_n = an;
                if (c4[j]) any = 255 - 4 * lane - j, any_w = aw, any_n = an;
                aw += w4[j];
                an += c4[j];
            }
            const u64 hit = __ballot(at >= 0), has = __ballot(any >= 0);
            const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(has);
            if (lane == l) {
                s_digit = hit ? at : any;
                s_w = hit ? at_w : any_w;
                s_n = hit ? at_n : any_n;
            }
        }
        __syncthreads();
        // all bits from the digit's lowest up are settled
        mask = ~0ull << shift;
        prefix = (s_hi & ~(255ull << shift) & mask) | (u64)s_digit << shift;
        before_w = s_w;
        before_n = s_n;
        __syncthreads();
    }
    if (!few)
        ws.each(lists, [&](u64 k, u64 v) {
            if (!in(k, v)) return;
            const uint32_t p = atomicAdd(&s_n, 1u);
            p_key[p] = k;
            p_val[p] = v;
        });
    const u64 *key = few ? ws.s_key : p_key, *val = few ? ws.s_val : p_val;
    if (tid == 0) {
        s_key = ~0ull;
        s_weight = before_w;
    }
    __syncthreads();
    const int left = few ? ws.m : (int)s_left, item = tid / 8;
    if (item < left) {
        const u64 k = key[item], mine = val[item];
        uint32_t rank = 0;
        u64 sum = 0;
        for (int j = tid % 8; j < left; j += 8) {
            const u64 v = val[j];
            const bool first = key[j] > k && in(key[j], v);
            rank += first;
            sum += first ? v & WEIGHT : 0;
        }
        rank = before_n + eight_total(rank);
        sum = before_w + eight_total(sum);
        if (tid % 8 == 0 && in(k, mine) && (BY_WEIGHT ? (double)sum < need_w || k == ws.w.kmax : rank < need_n)) {
            // the last that stays has the smallest key and the largest sum
            atomicMin(&s_key, k);
            atomicMax(&s_weight, sum + (mine & WEIGHT));
        }
    }
    __syncthreads();
    return {s_key, s_weight};
}

__global__ void __launch_bounds__(FI_WG) k_sample_finish(SampleArgs a)
{
    __shared__ u64 s_key[FI_LIST], s_val[FI_LIST], s_sum[FI_BLOCKS], s_wave[FI_WAVES], s_total, s_target;
    __shared__ uint32_t s_lcnt[FI_BLOCKS], s_cnt, s_block;
    __shared__ int s_begin[FI_BLOCKS], s_m;
    __shared__ double pow[64];
    static_assert(FI_BLOCKS == 256, "four blocks a lane");
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t o = (int64_t)r * a.blocks;
    const RowAt w = row_at(a, r);
    if (w.kmax == 0 || w.greedy) {
        if (tid == 0) {
            a.token[r] = w.kmax == 0 ? SKIP : key_index(w.kmax);
            if (a.logprob) a.logprob[r] = w.kmax == 0 ? -INFINITY : 0.0f;
            if (a.n_kept) a.n_kept[r] = w.kmax == 0 ? 0 : 1;
        }
        return;
    }
    fill_powers(pow);
    uint32_t cnt = 0;
    if (tid < FI_BLOCKS) {
        const bool there = tid < a.blocks;
        s_sum[tid] = there ? a.sum[o + tid] : 0;
        s_lcnt[tid] = there ? a.lcnt[o + tid] : 0;
        cnt = there ? a.cnt[o + tid] : 0;
    }
    if (tid == 0) s_cnt = 0;
    u64 stay = 0;  // keys at or above it are left of the border
    if (w.top_p || w.k) {
        const Border bd = find_border<FI_WG>(a, w, r);
        // the border words into LDS, if they fit
        Words ws{a, w, r, 0, s_lcnt, pow, s_key, s_val};
        if (wave == 0) {
            int c[4], all = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                c[j] = s_lcnt[4 * lane + j];
                all += c[j];
            }
            int at = wave_upto(all) - all;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s_begin[4 * lane + j] = at;
                at += c[j];
            }
            if (lane == 63) s_m = at;
        }
        __syncthreads();
        ws.m = s_m;
        if (ws.m <= FI_LIST)
            for (int j = tid; j < ws.m; j += FI_WG) {
                // the last block that begins at or before j
                int b = 0;
#pragma unroll
                for (int d = FI_BLOCKS / 2; d; d /= 2)
                    if (s_begin[b + d] <= j) b += d;
                ws.word(b, a.list[(o + b) * SA_BLOCK + j - s_begin[b]], s_key[j], s_val[j]);
            }
        __syncthreads();
        if (bd.k_bin >= 0) {
            const Chosen ck = choose<false>(ws, bd.k_bin, bd.k_bin, 1, w.k - bd.k_count, bd.k_weight, 0.0);
            stay = ck.key;
            if (w.top_p)
                stay = choose<true>(ws, bd.sure, bd.p_end, stay, 0, bd.p_weight, w.p * (double)ck.weight).key;
        } else if (w.top_p) {
            // (no word is cut off by top-k: S is the weight of all bins)
            stay = choose<true>(ws, bd.sure, bd.p_end, 1, 0, bd.p_weight, w.p * (double)bd.total).key;
        }
        // block sums: what surely stays, and the border words that do
        ws.each(ws.m > FI_LIST, [&](u64 k, u64 v) {
            const uint32_t i = key_index(k);
            if (k < stay || (w.min_p && !((double)(v & WEIGHT) >= w.min_w || k == w.kmax))) return;
            atomicAdd(&s_sum[i / SA_BLOCK], v & WEIGHT);
            cnt++;
        });
    }
    __syncthreads();
    cnt = wave_total(cnt);
    if (lane == 0 && cnt) atomicAdd(&s_cnt, cnt);
    if (wave == 0) {
        u64 v[4], run = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = s_sum[4 * lane + j];
            run += v[j];
        }
        const u64 incl = wave_upto(run), total = of_lane(incl, 63);
        // (the largest total is 2^63 - 2^44: what is below it can be converted)
        const double f = (double)a.u[r] * (double)total;
        u64 t = f > 0.0 ? f < (double)total ? (u64)f : total - 1 : 0;
        if (t >= total) t = total - 1;
        u64 at = incl - run;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (at <= t && t < at + v[j]) {
                s_block = 4 * lane + j;
                s_target = t - at;
            }
            at += v[j];
        }
        if (lane == 0) s_total = total;
    }
    __syncthreads();
    // the token in its block: 128 words of each wave, in two rows of 64
    constexpr int ROWS = SA_BLOCK / FI_WG;
    const int i0 = s_block * SA_BLOCK + wave * ROWS * 64 + lane;
    u64 v[ROWS], upto[ROWS], part = 0;
#pragma unroll
    for (int j = 0; j < ROWS; j++) {
        const int i = i0 + 64 * j;
        int bin;
        const float x = i < a.n ? w.x[i] : -INFINITY;
        v[j] = word_weight(w, pow, x, &bin);
        if (word_key(x, i) < stay || !min_p_stays(w, v[j], x, i)) v[j] = 0;
        upto[j] = part + wave_upto(v[j]);
        part = of_lane(upto[j], 63);
    }
    if (lane == 0) s_wave[wave] = part;
    __syncthreads();
    u64 at = 0;
    for (int q = 0; q < wave; q++) at += s_wave[q];
    const u64 t = s_target;
#pragma unroll
    for (int j = 0; j < ROWS; j++)
        if (v[j] && t < at + upto[j] && t >= at + upto[j] - v[j]) {
            a.token[r] = i0 + 64 * j;
            if (a.logprob) a.logprob[r] = (float)log((double)v[j] / (double)s_total);
            if (a.n_kept) a.n_kept[r] = s_cnt;
        }
}

SampleWs sample_ws(int rows, int n)
{
    SampleWs s{};
    s.blocks = (n + SA_BLOCK - 1) / SA_BLOCK;
    // about four workgroups per CU over all rows
    s.per = (int)std::max<int64_t>(1, (int64_t)s.blocks * rows / 1024);
    s.G = (s.blocks + s.per - 1) / s.per;
    const int64_t per_row = (int64_t)s.blocks * (24 + 2 * SA_BLOCK) + SAMPLE_BINS * 12;
    s.bytes = rows * per_row;
    return s;
}

hipError_t launch_sample(hipStream_t st, SampleArgs a, void *ws)
{
    const SampleWs s = sample_ws(a.rows, a.n);
    a.blocks = s.blocks;
    a.per = s.per;
    a.G = s.G;
    const int64_t rows = a.rows;
    a.top = (u64 *)ws;
    a.sum = a.top + rows * a.blocks;
    a.hw = a.sum + rows * a.blocks;
    a.hc = (uint32_t *)(a.hw + rows * SAMPLE_BINS);
    a.cnt = a.hc + rows * SAMPLE_BINS;
    a.lcnt = a.cnt + rows * a.blocks;
    a.list = (uint16_t *)(a.lcnt + rows * a.blocks);
    const dim3 grid(a.G, a.rows);
    hipLaunchKernelGGL(k_sample_max, grid, dim3(SA_WG), 0, st, a);
    hipLaunchKernelGGL(k_sample_bins, grid, dim3(SA_WG), 0, st, a);
    hipLaunchKernelGGL(k_sample_border, grid, dim3(SA_WG), 0, st, a);
    hipLaunchKernelGGL(k_sample_finish, dim3(a.rows), dim3(FI_WG), 0, st, a);
    return hipGetLastError();
}

}  // namespace styx
