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
// Nothing is sorted.  Four launches over chunks of the rows:
//   1 the rows' largest logits
//   2 weight and number of the words in bins of 1/64 of (max - x) / T
//   3 from these, the bins in which the k-th word and the end of the top-p
//     run lie: the words of those bins go to a list, the weight that surely
//     stays is summed per chunk
//   4 one workgroup per row: the border words in their order, which of them
//     stay, and the token in its chunk
// Bound: latency for a few rows (each launch waits for all of the one
// before), reads of the logits from HBM once and from the Infinity Cache
// twice more for many.
#include "../../include/styx_hip.h"
#include "sample.h"

#include <algorithm>

namespace styx {

constexpr int SA_WG = 256, FI_WG = 1024, FI_WAVES = FI_WG / 64;
constexpr int SA_MIN = 2048;        // fewest words of a chunk
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
    styx_sample_params p;
    u64 kmax;       // the first word
    float mx;
    double inv_t;
    bool greedy, top_p, min_p;
    int k;          // 0: all
};

__device__ __forceinline__ u64 wave_max64(u64 v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ u64 wave_add64(u64 v)
{
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ u64 wave_scan64(u64 v)  // inclusive
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// The row's settings and, from the chunks, its first word; every wave by itself.
__device__ __forceinline__ RowAt row_at(const SampleArgs &a, int r)
{
    RowAt w;
    w.x = a.logits + r * a.ld;
    w.p = a.params[a.one_params ? 0 : r];
    u64 k = 0;
    for (int c = threadIdx.x & 63; c < a.G; c += 64) {
        const u64 o = a.cmax[(int64_t)r * a.G + c];
        k = o > k ? o : k;
    }
    w.kmax = wave_max64(k);
    w.mx = key_value(w.kmax);
    w.greedy = !(w.p.temperature > 0.0f);
    w.inv_t = 1.0 / (double)w.p.temperature;
    w.top_p = w.p.top_p < 1.0f;
    w.min_p = w.p.min_p > 0.0f;
    w.k = w.p.top_k > 0 && w.p.top_k < a.n ? w.p.top_k : 0;
    return w;
}

__device__ __forceinline__ double word_dist(const RowAt &w, float x) { return ((double)w.mx - (double)x) * w.inv_t; }
// Weight of a candidate, and its bin.
__device__ __forceinline__ u64 word_weight(const RowAt &w, float x, int *bin)
{
    *bin = 0;
    if (x == w.mx) return (u64)SA_ONE;
    if (!(x > -INFINITY) || w.mx == INFINITY) return 0;
    const double d = word_dist(w, x);
    if (!(d < 31.5)) return 0;
    *bin = (int)(d * 64.0);
    return (u64)rint(exp(-d) * SA_ONE);
}
__device__ __forceinline__ bool min_p_stays(const RowAt &w, u64 weight, u64 key)
{
    return !w.min_p || (double)weight >= (double)w.p.min_p * SA_ONE || key == w.kmax;
}

// ------------------------------------------------------------- 1: largest --
__global__ void __launch_bounds__(SA_WG) k_sample_max(SampleArgs a)
{
    __shared__ u64 s[SA_WG / 64];
    const int c = blockIdx.x, r = blockIdx.y, c0 = c * a.ch, c1 = min(a.n, c0 + a.ch);
    const float *x = a.logits + r * a.ld;
    u64 k = 0;
    for (int i = c0 + threadIdx.x; i < c1; i += SA_WG) {
        const u64 o = word_key(x[i], i);
        k = o > k ? o : k;
    }
    k = wave_max64(k);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = k;
    // the bins and the list of the row, emptied by its chunks together
    for (int i = c * SA_WG + threadIdx.x; i < SAMPLE_BINS; i += a.G * SA_WG) {
        a.hw[(int64_t)r * SAMPLE_BINS + i] = 0;
        a.hc[(int64_t)r * SAMPLE_BINS + i] = 0;
    }
    if (c == 0 && threadIdx.x == 0) a.nlist[r] = 0;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < SA_WG / 64; w++) k = s[w] > k ? s[w] : k;
        a.cmax[(int64_t)r * a.G + c] = k;
    }
}

// ---------------------------------------------------------------- 2: bins --
__global__ void __launch_bounds__(SA_WG) k_sample_bins(SampleArgs a)
{
    __shared__ u64 hw[SAMPLE_BINS];
    __shared__ uint32_t hc[SAMPLE_BINS];
    const int c = blockIdx.x, r = blockIdx.y, c0 = c * a.ch, c1 = min(a.n, c0 + a.ch);
    const RowAt w = row_at(a, r);
    if (w.kmax == 0 || w.greedy || !(w.top_p || w.k)) return;
    for (int i = threadIdx.x; i < SAMPLE_BINS; i += SA_WG) hw[i] = hc[i] = 0;
    __syncthreads();
    for (int i = c0 + threadIdx.x; i < c1; i += SA_WG) {
        int bin;
        const u64 v = word_weight(w, w.x[i], &bin);
        if (v == 0) continue;
        atomicAdd(&hw[bin], v);
        if (w.k) atomicAdd(&hc[bin], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SAMPLE_BINS; i += SA_WG)
        if (hw[i]) {
            atomicAdd(&a.hw[(int64_t)r * SAMPLE_BINS + i], hw[i]);
            if (w.k) atomicAdd(&a.hc[(int64_t)r * SAMPLE_BINS + i], hc[i]);
        }
}

// -------------------------------------------------------------- 3: border --
// The bins that hold the border: words of bins below `sure` stay as far as
// top-k and top-p go; those of [sure, p_end] (top-p) and of k_bin (top-k)
// are looked at one by one; all others leave.
struct Border {
    int sure, p_end, k_bin;
    u64 k_weight;   // weight and number of the bins before k_bin
    uint32_t k_count;
    u64 p_weight;   // weight of the bins before `sure`
};

// All threads of the workgroup (NT of them) take part.
template <int NT> __device__ Border find_border(const SampleArgs &a, const RowAt &w, int r)
{
    constexpr int PER = SAMPLE_BINS / NT, NW = NT / 64;
    __shared__ u64 s_w[NW];
    __shared__ uint32_t s_c[NW];
    __shared__ Border s_b;
    __shared__ u64 s_lo, s_hi;
    if (!(w.top_p || w.k)) return {SAMPLE_BINS, -1, -1, 0, 0, 0};
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
    u64 iw = wave_scan64(aw);
    uint32_t ic = (uint32_t)wave_scan64(ac);
    if (lane == 63) {
        s_w[wave] = iw;
        s_c[wave] = ic;
    }
    if (tid == 0) s_b = {SAMPLE_BINS, -1, -1, 0, 0, 0};
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
    if (tid == 0) s_lo = s_hi = total;
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
    }
    __syncthreads();
    if (w.top_p) {
        // the run ends at the first word before which at least top_p S lies;
        // S is between s_lo and s_hi
        const double lo = (double)w.p.top_p * (double)s_lo, hi = (double)w.p.top_p * (double)s_hi;
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
    }
    __syncthreads();
    return s_b;
}

__global__ void __launch_bounds__(SA_WG) k_sample_border(SampleArgs a)
{
    __shared__ u64 s_sum[SA_WG / 64];
    __shared__ uint32_t s_cnt[SA_WG / 64];
    const int c = blockIdx.x, r = blockIdx.y, c0 = c * a.ch, c1 = min(a.n, c0 + a.ch);
    const RowAt w = row_at(a, r);
    if (w.kmax == 0 || w.greedy) return;
    const Border bd = find_border<SA_WG>(a, w, r);
    u64 sum = 0;
    uint32_t cnt = 0;
    for (int i = c0 + threadIdx.x; i < c1; i += SA_WG) {
        int bin;
        const float x = w.x[i];
        const u64 v = word_weight(w, x, &bin);
        if (v == 0) continue;
        if (bin < bd.sure) {
            if (min_p_stays(w, v, word_key(x, i))) {
                sum += v;
                cnt++;
            }
        } else if (bin <= bd.p_end || bin == bd.k_bin) {
            a.list[(int64_t)r * a.n + atomicAdd(&a.nlist[r], 1u)] = i;
        }
    }
    sum = wave_add64(sum);
    cnt = (uint32_t)wave_add64(cnt);
    if ((threadIdx.x & 63) == 0) {
        s_sum[threadIdx.x >> 6] = sum;
        s_cnt[threadIdx.x >> 6] = cnt;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int q = 1; q < SA_WG / 64; q++) {
            sum += s_sum[q];
            cnt += s_cnt[q];
        }
        a.csum[(int64_t)r * a.G + c] = sum;
        a.ccnt[(int64_t)r * a.G + c] = cnt;
    }
}

// -------------------------------------------------------------- 4: finish --
// The last key that stays of the list's words in bins [b0, b1], of which
// those below `floor` do not count: the first `need` of them (BY_WEIGHT: the
// shortest run, the first word at least, before whose end less than `need`
// lies); *weight their weight.  Words are told apart by a radix selection of
// 8 bits a pass until at most FI_WG are left, which are then ranked each
// against all.
struct Chosen {
    u64 key, weight;
};
template <bool BY_WEIGHT>
__device__ Chosen choose(const SampleArgs &a, const RowAt &w, const uint32_t *list, uint32_t m, int b0, int b1,
                         u64 floor, uint32_t need_n, u64 base, double need_w, u64 *s_key, u64 *s_val)
{
    __shared__ u64 bw[256];
    __shared__ uint32_t bc[256], s_left, s_digit, s_n;
    __shared__ u64 s_w, s_out_key, s_out_w;
    const int tid = threadIdx.x;
    u64 prefix = 0, mask = 0, before_w = base;
    uint32_t before_n = 0;
    auto word = [&](uint32_t j, u64 *v) -> u64 {
        int bin;
        const uint32_t i = list[j];
        const float x = w.x[i];
        *v = word_weight(w, x, &bin);
        const u64 k = word_key(x, i);
        return bin >= b0 && bin <= b1 && k >= floor && (k & mask) == prefix ? k : 0;
    };
    int shift = 56;
    for (;; shift -= 8) {
        if (tid < 256) bw[tid] = bc[tid] = 0;
        if (tid == 0) s_left = 0;
        __syncthreads();
        uint32_t mine = 0;
        for (uint32_t j = tid; j < m; j += FI_WG) {
            u64 v;
            const u64 k = word(j, &v);
            if (!k) continue;
            mine++;
            if (shift >= 0) {
                atomicAdd(&bw[(k >> shift) & 255], v);
                atomicAdd(&bc[(k >> shift) & 255], 1u);
            }
        }
        mine = (uint32_t)wave_add64(mine);
        if ((tid & 63) == 0 && mine) atomicAdd(&s_left, mine);
        __syncthreads();
        if (s_left <= FI_WG || shift < 0) break;
        if (tid == 0) {
            uint32_t n = before_n;
            u64 s = before_w;
            for (int d = 255; d >= 0; d--) {
                if (!bc[d]) continue;
                s_digit = d;
                s_n = n;
                s_w = s;
                n += bc[d];
                s += bw[d];
                if (BY_WEIGHT ? (double)s >= need_w : n >= need_n) break;
            }
        }
        __syncthreads();
        prefix |= (u64)s_digit << shift;
        mask |= 255ull << shift;
        before_n = s_n;
        before_w = s_w;
        __syncthreads();
    }
    // at most FI_WG words: each against all
    const uint32_t left = s_left;
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (uint32_t j = tid; j < m; j += FI_WG) {
        u64 v;
        const u64 k = word(j, &v);
        if (!k) continue;
        const uint32_t p = atomicAdd(&s_n, 1u);
        s_key[p] = k;
        s_val[p] = v;
    }
    if (tid == 0) {
        s_out_key = ~0ull;
        s_out_w = before_w;
    }
    __syncthreads();
    if (tid < (int)left) {
        const u64 k = s_key[tid];
        uint32_t rank = before_n;
        u64 sum = before_w;
        for (uint32_t j = 0; j < left; j++)
            if (s_key[j] > k) {
                rank++;
                sum += s_val[j];
            }
        const bool in = BY_WEIGHT ? (double)sum < need_w || k == w.kmax : rank < need_n;
        if (in) {
            // the last that stays has the smallest key and the largest sum
            atomicMin(&s_out_key, k);
            atomicMax(&s_out_w, sum + s_val[tid]);
        }
    }
    __syncthreads();
    return {s_out_key, s_out_w};
}

__global__ void __launch_bounds__(FI_WG) k_sample_finish(SampleArgs a)
{
    __shared__ u64 s_key[FI_WG], s_val[FI_WG], s_sum[256], s_wave[FI_WAVES], s_total, s_target;
    __shared__ uint32_t s_cnt, s_chunk;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const RowAt w = row_at(a, r);
    if (w.kmax == 0 || w.greedy) {
        if (tid == 0) {
            a.token[r] = w.kmax == 0 ? SKIP : key_index(w.kmax);
            if (a.logprob) a.logprob[r] = w.kmax == 0 ? -INFINITY : 0.0f;
            if (a.n_kept) a.n_kept[r] = w.kmax == 0 ? 0 : 1;
        }
        return;
    }
    const Border bd = find_border<FI_WG>(a, w, r);
    const uint32_t *list = a.list + (int64_t)r * a.n;
    const uint32_t m = w.top_p || w.k ? a.nlist[r] : 0;
    // keys at or above `stay` are left of the border
    u64 stay = 0;
    if (bd.k_bin >= 0) {
        const Chosen ck = choose<false>(a, w, list, m, bd.k_bin, bd.k_bin, 1, w.k - bd.k_count, bd.k_weight, 0.0,
                                        s_key, s_val);
        stay = ck.key;
        if (w.top_p) {
            __syncthreads();
            stay = choose<true>(a, w, list, m, bd.sure, bd.p_end, stay, 0, bd.p_weight,
                                (double)w.p.top_p * (double)ck.weight, s_key, s_val)
                       .key;
        }
    } else if (w.top_p) {
        // (no word is cut off by top-k: S is the weight of all bins)
        u64 total = 0;
        for (int i = lane; i < SAMPLE_BINS; i += 64) total += a.hw[(int64_t)r * SAMPLE_BINS + i];
        total = wave_add64(total);
        stay = choose<true>(a, w, list, m, bd.sure, bd.p_end, 1, 0, bd.p_weight,
                            (double)w.p.top_p * (double)total, s_key, s_val)
                   .key;
    }
    __syncthreads();
    // chunk sums: what surely stays, and the border words that do
    if (tid < 256) s_sum[tid] = tid < a.G ? a.csum[(int64_t)r * a.G + tid] : 0;
    if (tid == 0) s_cnt = 0;
    __syncthreads();
    uint32_t cnt = tid < a.G ? a.ccnt[(int64_t)r * a.G + tid] : 0;
    for (uint32_t j = tid; j < m; j += FI_WG) {
        int bin;
        const uint32_t i = list[j];
        const float x = w.x[i];
        const u64 k = word_key(x, i), v = word_weight(w, x, &bin);
        if (k < stay || !min_p_stays(w, v, k)) continue;
        atomicAdd(&s_sum[i / a.ch], v);
        cnt++;
    }
    cnt = (uint32_t)wave_add64(cnt);
    if (lane == 0 && cnt) atomicAdd(&s_cnt, cnt);
    __syncthreads();
    if (wave == 0) {
        u64 v[4], run = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = s_sum[4 * lane + j];
            run += v[j];
        }
        const u64 incl = wave_scan64(run);
        const u64 total = __shfl(incl, 63);
        const double f = (double)a.u[r] * (double)total;
        u64 t = f > 0.0 ? (u64)fmin(f, 9.2e18) : 0;
        if (t >= total) t = total - 1;
        u64 at = incl - run;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (at <= t && t < at + v[j]) {
                s_chunk = 4 * lane + j;
                s_target = t - at;
            }
            at += v[j];
        }
        if (lane == 0) s_total = total;
    }
    __syncthreads();
    // the token in its chunk: a contiguous part per wave, then 64 at a time
    const int c0 = s_chunk * a.ch, c1 = min(a.n, c0 + a.ch), per = (c1 - c0 + FI_WAVES - 1) / FI_WAVES;
    auto kept = [&](int i) -> u64 {
        int bin;
        const float x = w.x[i];
        const u64 v = word_weight(w, x, &bin), k = word_key(x, i);
        if (v == 0 || !min_p_stays(w, v, k)) return 0;
        return k >= stay ? v : 0;
    };
    const int i0 = c0 + wave * per, i1 = min(c1, i0 + per);
    u64 part = 0;
    for (int i = i0 + lane; i < i1; i += 64) part += kept(i);
    part = wave_add64(part);
    if (lane == 0) s_wave[wave] = part;
    __syncthreads();
    u64 at = 0;
    for (int q = 0; q < wave; q++) at += s_wave[q];
    const u64 t = s_target;
    if (at <= t && t < at + part) {
        for (int i = i0; i < i1; i += 64) {
            const u64 v = i + lane < i1 ? kept(i + lane) : 0, incl = at + wave_scan64(v);
            const unsigned long long hit = __ballot(v && incl > t);
            if (hit) {
                if (lane == __builtin_ctzll(hit)) {
                    a.token[r] = i + lane;
                    if (a.logprob) a.logprob[r] = (float)log((double)v / (double)s_total);
                    if (a.n_kept) a.n_kept[r] = s_cnt;
                }
                break;
            }
            at = __shfl(incl, 63);
        }
    }
}

SampleWs sample_ws(int rows, int n)
{
    SampleWs s{};
    // about four workgroups per CU over all rows; at most 256 chunks
    const int most = std::min(256, (n + SA_MIN - 1) / SA_MIN);
    s.G = std::max(1, std::min(most, 1024 / rows));
    s.ch = ((n + s.G - 1) / s.G + SA_WG - 1) / SA_WG * SA_WG;
    s.G = (n + s.ch - 1) / s.ch;
    const int64_t per = (int64_t)s.G * 20 + SAMPLE_BINS * 12 + 8 + 4 * (int64_t)n + 8;
    s.bytes = rows * per;
    return s;
}

hipError_t launch_sample(hipStream_t st, SampleArgs a, void *ws)
{
    const SampleWs s = sample_ws(a.rows, a.n);
    a.G = s.G;
    a.ch = s.ch;
    const int64_t rows = a.rows;
    a.cmax = (u64 *)ws;
    a.csum = a.cmax + rows * a.G;
    a.hw = a.csum + rows * a.G;
    a.hc = (uint32_t *)(a.hw + rows * SAMPLE_BINS);
    a.ccnt = a.hc + rows * SAMPLE_BINS;
    a.nlist = a.ccnt + rows * a.G;
    a.list = a.nlist + rows;
    const dim3 grid(a.G, a.rows);
    hipLaunchKernelGGL(k_sample_max, grid, dim3(SA_WG), 0, st, a);
    hipLaunchKernelGGL(k_sample_bins, grid, dim3(SA_WG), 0, st, a);
    hipLaunchKernelGGL(k_sample_border, grid, dim3(SA_WG), 0, st, a);
    hipLaunchKernelGGL(k_sample_finish, dim3(a.rows), dim3(FI_WG), 0, st, a);
    return hipGetLastError();
}

}  // namespace styx
