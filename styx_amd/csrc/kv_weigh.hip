// kv_weigh.hip -- the attention weights of the last tokens of each sequence's
// chunk, added to the accumulator by which rows are evicted.
//
//   acc_out[j][t] = decay acc_in[j][t] (0 for the new rows)
//                 + sum over the last tokens i that see t and the heads h of j
//                   of e^(scale q_ih . K[t] - lse_ih),  t < len + count
//
// A wave holds 32 slots of a kv head in registers and goes over the query rows
// (tokens times heads) in tiles of 32 that its workgroup keeps in LDS, the next
// tile on its way meanwhile: K is read once, and no sum crosses waves.  Scores
// are formed queries x slots, so a lane has its own slot's of 16 rows of a tile
// (its other half, lane ^ 32, the other 16): weights are summed lane by lane.
//
// Bound: products and exponentials, a score costing 256 FLOP and one exponential
// at head_dim 128.  64 tokens of 32 f16 heads over 32768 slots, 17 GFLOP: 33 us,
// 15 for the products; f32 queries on them 51, 30 for two pieces.  16
// conversations, 16 tokens of 64 f32 heads each, 4.3 GFLOP: 63 us, 28 for the
// products.  What is lost is waits: as built, each operand of a tile is read from
// LDS right before the product that takes it (four products for f32), which waits
// for it, in one chain of sums, and a tile's factors follow its products in the
// same wave.  For the f32 batch 540 workgroups of equal length for 256 CUs, so
// that some take three and most two, make 28 into 40.  Smaller workgroups even
// that out, but each fetches all query rows (kw_waves).  One token for each of 24
// sequences over 8192 f16 slots, 208 MB: 61 us, 45 at a copy's rate.
#include <algorithm>
#include <type_traits>

#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int KW_ROWS = 32;
// Where blocks of 32 slots are few, the waves of a workgroup take one of them
// together, each other tiles of query rows, read as they lie, and add their sums
// up in order: half of KW_FEW blocks at most, all of it where there are 8 tiles
// and more and no pieces to form of each (launch_kv_weigh).  One conversation of
// 4000 slots over 4 kv heads, 64 tokens: 500 blocks, f16 15 us, 22 without,
// f32 32 and 49, heads of 256 47 and 92; f32 queries on f16 rows 38 and 33; 16
// tokens over 2000 f32 slots 8.7 and 15.9.  With 1024 blocks and 4 tiles 17.8 and 9.4.
constexpr int KW_FEW = 512;
// Waves of a workgroup, all of which read its tiles: f16 products are so fast
// that fetching the tiles counts (64 tokens over 32768 slots: 8 waves 31 us, 4
// waves 35, 2 waves 36), f32 ones are not, and smaller workgroups fill the chip
// more evenly (16 conversations: 4 waves 63 us, 2 waves 69, 1 wave 77).
// (Heads of 64 have no 16 bytes of a tile for more than 4 waves' threads.)
__host__ __device__ constexpr int kw_waves(bool f16, int hd) { return f16 && hd > 64 ? 8 : 4; }
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

// A tile of query rows in LDS, of type T: 16-byte pieces permuted within 256
// bytes, so that 16 rows' reads of a piece lie in banks of their own.
template <typename T, int HD> struct RowLay {
    static constexpr int ROW = HD * (int)sizeof(T);
    static __device__ __forceinline__ int at(int r, int byte)
    {
        const int p = ROW == 128 ? (r >> 1) & 7 : r & 15;
        return r * ROW + (byte ^ (p << 4));
    }
};

// f32 queries on f16 rows are two f16 pieces, brought to [2^9, 2^10) by a power
// of two per row (m: its largest value), as in the attention.
__device__ __forceinline__ float up_of(float m)
{
    const int e = m > 0.0f && m < INFINITY ? (int)((__float_as_uint(m) >> 23) & 255) - 127 : 9;
    return e < -100 ? ldexpf(1.0f, 109) : ldexpf(1.0f, 9 - e);
}
__device__ __forceinline__ void pieces(const float *v, float up, h8 &hi, h8 &lo)
{
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y = v[e] * up;
        hi[e] = (_Float16)y;
        lo[e] = (_Float16)(y - (float)hi[e]);
    }
}

// Waves of a SIMD: two workgroups of f16 rows a CU, but for heads of 256.
template <typename TQ, typename TC, int HD> constexpr int KW_SIMD = HD == 256 && sizeof(TQ) == 4 ? 2 : sizeof(TC) == 2 && HD <= 128 ? 4 : 3;
template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(64 * kw_waves(sizeof(TC) == 2, HD), (KW_SIMD<TQ, TC, HD>)) k_kv_weigh(KvWeighArgs a)
{
    constexpr int NP = sizeof(TQ) == 4 && sizeof(TC) == 2 ? 2 : 1;
    using La = RowLay<TC, HD>;
    constexpr int KW_NW = kw_waves(sizeof(TC) == 2, HD), KW_WG = 64 * KW_NW;
    constexpr int NK = sizeof(TC) == 2 ? HD / 16 : HD / 8;  // operands of a row
    constexpr int PER = KW_ROWS * HD / KW_WG;               // values of a thread in a tile
    constexpr int TPR = HD / PER;                           // threads of a row
    static_assert(PER % 8 == 0 || (sizeof(TQ) == 4 && NP == 1 && PER % 4 == 0), "whole pieces");
    typedef typename std::conditional<sizeof(TC) == 2, h8, styx_f4>::type Op;
    __shared__ __align__(16) char s_q[2][NP][KW_ROWS * La::ROW];
    __shared__ __align__(16) float s_lse[2][KW_ROWS], s_mul[2][KW_ROWS];
    __shared__ __align__(16) int s_at[2][KW_ROWS];
    // of each wave's own tile; sums by wave
    __shared__ __align__(16) float s_own[KW_NW][2][KW_ROWS];
    __shared__ __align__(16) int s_own_at[KW_NW][KW_ROWS];
    __shared__ float s_sum[KW_NW][KW_ROWS];
    const KvView &kv = a.kv;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t stride = (int64_t)kv.nkv * HD;
    bool few = a.few != 0;
    if (few) {
        int blocks = 0;  // up to one more than KW_FEW
        for (int b0 = 0; b0 < kv.n_seq; b0 += 64) {
            const ChunkSeq mine = chunk_seq(a.chunk, kv, b0 + lane);
            blocks = min(blocks + (mine.count ? min((mine.len + mine.count + 31) / 32, KW_FEW + 1) : 0), KW_FEW + 1);
        }
        few = (int64_t)of_lane(wave_total((uint32_t)blocks), 0) * kv.nkv <= a.few;
    }
    const int keys = few ? 32 : 32 * KW_NW;
    for (int64_t item = blockIdx.x;; item += gridDim.x) {
        // (numbers that the compiler takes for new ones in every trip: what is
        // computed from them would else be kept in registers over the trips)
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int n = tid & 31, h = tid >> 5 & 1;
        // the sequence and its slots
        const int kvh = (int)(item % kv.nkv);
        int64_t nth = item / kv.nkv;
        int b = -1;
        ChunkSeq s{};
        for (int b0 = 0; b0 < kv.n_seq && b < 0; b0 += 64) {
            const ChunkSeq mine = chunk_seq(a.chunk, kv, b0 + lane);
            const int64_t tiles = mine.count ? ((int64_t)mine.len + mine.count + keys - 1) / keys : 0, upto = wave_upto(tiles);
            if (const unsigned long long hit = __ballot(upto > nth)) {
                const int l = __builtin_ctzll(hit);
                b = b0 + l;
                s = {(int)__builtin_amdgcn_readlane(mine.first, l), (int)__builtin_amdgcn_readlane(mine.count, l),
                     (int)__builtin_amdgcn_readlane(mine.len, l)};
                nth -= of_lane(upto, l) - of_lane(tiles, l);
            } else {
                nth -= of_lane(upto, 63);
            }
        }
        if (b < 0) return;
        const int k0 = (int)nth * keys, slots = s.len + s.count;
        const int w0 = k0 + (few ? 0 : 32 * wave), t = w0 + n;  // this lane's slot
        const int row = t < slots ? kv.row(kv.table + (int64_t)b * kv.table_len, t) : -1;
        Op k[NK];
        const TC *kp = (const TC *)kv.kpool + max(row, 0) * stride + kvh * HD + (sizeof(TC) == 2 ? 8 : 4) * h;
#pragma unroll
        for (int i = 0; i < NK; i++) k[i] = *(const Op *)(kp + (sizeof(TC) == 2 ? 16 : 8) * i);
        // tokens that count and see any of these slots, and their rows
        const int i0 = max(max(s.count - min(a.last, s.count), k0 - s.len), 0);
        const int i1 = a.window ? (int)max((int64_t)i0, min((int64_t)s.count, (int64_t)k0 + keys - 1 + a.window - s.len)) : s.count;
        const int r0 = i0 * a.gqa, r1 = max(i0, i1) * a.gqa;
        // a thread's part of a row of the next tile
        __align__(16) TQ in[PER];
        float in_lse = 0.0f;
        const int mr = tid / TPR, md = tid % TPR * PER;
        auto ask = [&](int base) {
            const int r = min(base + mr, r1 - 1), tok = a.by_gqa.of(r), head = kvh * a.gqa + (r - tok * a.gqa);
            const TQ *p = (const TQ *)a.q + (int64_t)(s.first + tok) * a.ldq + (int64_t)head * HD + md;
            constexpr int M = 16 / sizeof(TQ);
            typedef typename std::conditional<sizeof(TQ) == 2, h8, styx_f4>::type V;
#pragma unroll
            for (int i = 0; i < PER; i += M) *(V *)(in + i) = *(const V *)(p + i);
            in_lse = a.lse[(int64_t)(s.first + tok) * a.nh + head];
        };
        auto put = [&](int buf, int base) {
            float mul = a.scale;
            if constexpr (NP == 2) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < PER; i++) m = fmaxf(m, fabsf((float)in[i]));
#pragma unroll
                for (int d = 1; d < TPR; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
                const float up = up_of(m);
                mul /= up;
#pragma unroll
                for (int i = 0; i < PER; i += 8) {
                    h8 hi, lo;
                    pieces((const float *)in + i, up, hi, lo);
                    *(h8 *)(s_q[buf][0] + La::at(mr, 2 * (md + i))) = hi;
                    *(h8 *)(s_q[buf][NP - 1] + La::at(mr, 2 * (md + i))) = lo;
                }
            } else {
                constexpr int M = 16 / sizeof(TC);
#pragma unroll
                for (int i = 0; i < PER; i += M) *(Op *)(s_q[buf][0] + La::at(mr, (int)sizeof(TC) * (md + i))) = *(const Op *)(in + i);
            }
            if (tid % TPR == 0) {
                const int r = base + mr;
                // a token that sees nothing has no weights: none that are NaN, either
                const bool counts = r < r1 && in_lse != -INFINITY;
                s_lse[buf][mr] = counts ? in_lse * 1.44269504f : INFINITY;
                s_mul[buf][mr] = mul;
                s_at[buf][mr] = counts ? s.len + a.by_gqa.of(r) : -1;
            }
        };
        float sum[2] = {};
        auto add = [&](const f16v &x, int base, bool all, const float *s_l, const float *s_m, const int *s_a) {
            // whether every row of the tile counts and sees all of the wave's slots
            const bool whole = all && w0 + 31 <= s.len + a.by_gqa.of(base) &&
                               (!a.window || w0 > s.len + a.by_gqa.of(base + KW_ROWS - 1) - a.window);
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int r = 2 * i + 4 * h;
                const styx_f4 lse = *(const styx_f4 *)&s_l[r], mul = *(const styx_f4 *)&s_m[r];
#pragma unroll
                for (int e = 0; e < 4; e++) w[i + e] = __builtin_amdgcn_exp2f(fmaf(x[i + e], mul[e], -lse[e]));
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int at = s_a[8 * (i >> 2) + 4 * h + (i & 3)];
                    const bool see = (t <= at) & ((a.window == 0) | (t > at - a.window));
                    w[i] = see ? w[i] : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                sum[0] += w[i];
                sum[1] += w[i + 1];
            }
        };
        __syncthreads();  // (the last item's tiles are read no more)
        if (r0 < r1 && !few) {
            ask(r0);
            put(0, r0);
            // (waited for here.  The loop as built counts these loads down once more
            // before its products, as the branch past this one reaches it, too; what
            // it then waits for with them, the next tile's rows, it stages next)
#pragma unroll
            for (int i = 0; i < NK; i++) asm volatile("" : "+v"(k[i]));
            if (r0 + KW_ROWS < r1) ask(r0 + KW_ROWS);
        }
        for (int base = few ? r1 : r0, buf = 0; base < r1; base += KW_ROWS, buf ^= 1) {
            __syncthreads();
            const int last = s_at[buf][n];
            f16v x = {};
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const int at = La::at(n, 32 * i + 16 * h);
                if constexpr (sizeof(TC) == 2) {
#pragma unroll
                    for (int y = 0; y < NP; y++) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const h8 *)(s_q[buf][y] + at), k[i], x, 0, 0, 0);
                } else {
                    const styx_f4 q = *(const styx_f4 *)(s_q[buf][0] + at);
#pragma unroll
                    for (int e = 0; e < 4; e++) x = __builtin_amdgcn_mfma_f32_32x32x2f32(q[e], k[i][e], x, 0, 0, 0);
                }
            }
            if (base + KW_ROWS < r1) {
                put(buf ^ 1, base + KW_ROWS);
                if (base + 2 * KW_ROWS < r1) ask(base + 2 * KW_ROWS);
            }
            add(x, base, __ballot(last < 0) == 0, s_lse[buf], s_mul[buf], s_at[buf]);
        }
        for (int base = few ? r0 + KW_ROWS * wave : r1; base < r1; base += KW_ROWS * KW_NW) {
            // row n of a tile of the wave's own, as it lies
            const int r = min(base + n, r1 - 1), tok = a.by_gqa.of(r), head = kvh * a.gqa + (r - tok * a.gqa);
            const TQ *p = (const TQ *)a.q + (int64_t)(s.first + tok) * a.ldq + (int64_t)head * HD + (sizeof(TC) == 2 ? 8 : 4) * h;
            const float lse = a.lse[(int64_t)(s.first + tok) * a.nh + head];
            constexpr int AHEAD = sizeof(TQ) == 2 ? (NK < 8 ? NK : 8) : NP == 2 || HD == 256 ? 2 : 4;
            struct Raw {
                Op v[sizeof(TQ) == 4 && NP == 2 ? 2 : 1];
            };
            auto read = [&](int i) { return *(const Raw *)(p + (sizeof(TC) == 2 ? 16 : 8) * i); };
            float mul = a.scale, up = 1.0f;
            if constexpr (NP == 2) {
                float m = 0.0f;
#pragma unroll 2
                for (int i = 0; i < NK; i++) {
                    const Raw y = read(i);
                    const float *f = (const float *)&y;
#pragma unroll
                    for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(f[e]));
                    __builtin_amdgcn_sched_barrier(0);
                }
                m = fmaxf(m, __shfl_xor(m, 32));
                up = up_of(m);
                mul /= up;
            }
            if (h == 0) {
                const bool counts = base + n < r1 && lse != -INFINITY;
                s_own[wave][0][n] = counts ? lse * 1.44269504f : INFINITY;
                s_own[wave][1][n] = mul;
                s_own_at[wave][n] = counts ? s.len + tok : -1;
            }
            Raw y[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) y[i] = read(i);
            f16v x = {};
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const Raw q = y[i % AHEAD];
                if (i + AHEAD < NK) y[i % AHEAD] = read(i + AHEAD);
                if constexpr (NP == 2) {
                    h8 hi, lo;
                    pieces((const float *)&q, up, hi, lo);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, k[i], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo, k[i], x, 0, 0, 0);
                } else if constexpr (sizeof(TC) == 2) {
                    x = __builtin_amdgcn_mfma_f32_32x32x16_f16(q.v[0], k[i], x, 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) x = __builtin_amdgcn_mfma_f32_32x32x2f32(q.v[0][e], k[i][e], x, 0, 0, 0);
                }
                // (loads stay AHEAD: all at once they cost registers, and the
                // long calls the second workgroup of a CU)
                __builtin_amdgcn_sched_barrier(0);
            }
            // (a wave's LDS operations are carried out in order)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            add(x, base, __ballot(s_own_at[wave][n] < 0) == 0, s_own[wave][0], s_own[wave][1], s_own_at[wave]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        float all = sum[0] + sum[1];
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(all), __float_as_uint(all), false, false);
        all = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        if (few) {
            if (h == 0) s_sum[wave][n] = all;
            __syncthreads();
            if (wave) continue;
            all = s_sum[0][n];
#pragma unroll
            for (int w = 1; w < KW_NW; w++) all += s_sum[w][n];
        }
        if (h == 0 && t < slots) {
            const int64_t at = ((int64_t)b * kv.nkv + kvh) * kv.cap + t;
            a.acc_out[at] = (a.acc_in && t < s.len ? a.decay * a.acc_in[at] : 0.0f) + (row >= 0 ? all : 0.0f);
            if (a.slot_pos && t >= s.len) a.slot_pos[at] = a.pos[b] + (t - s.len);
        }
    }
}

int64_t kv_weigh_grid(const KvWeighArgs &a)
{
    const int64_t heads = (int64_t)a.kv.n_seq * a.kv.nkv, blocks = ((int64_t)a.kv.cap + 31) / 32 * heads;
    return std::min<int64_t>(blocks, std::max<int64_t>(KW_FEW, std::min<int64_t>(4096, blocks / kw_waves(a.kv.f16, a.kv.hd) + heads)));
}

template <typename TQ, typename TC> static void launch_hd(hipStream_t st, const KvWeighArgs &a)
{
    const dim3 g((unsigned)kv_weigh_grid(a)), wg(64 * kw_waves(a.kv.f16, a.kv.hd));
    switch (a.kv.hd) {
    case 64: hipLaunchKernelGGL((k_kv_weigh<TQ, TC, 64>), g, wg, 0, st, a); break;
    case 128: hipLaunchKernelGGL((k_kv_weigh<TQ, TC, 128>), g, wg, 0, st, a); break;
    default: hipLaunchKernelGGL((k_kv_weigh<TQ, TC, 256>), g, wg, 0, st, a); break;
    }
}
hipError_t launch_kv_weigh(hipStream_t st, KvWeighArgs a)
{
    a.scale = (float)((double)a.scale * 1.4426950408889634);  // log2 e
    a.by_gqa = page_div((uint32_t)a.gqa);
    const int64_t rows = (int64_t)std::min(a.last, a.chunk.n_rows) * a.gqa;
    a.few = rows <= KW_ROWS ? 0 : (!a.kv.f16 || a.q_f16) && rows >= 8 * KW_ROWS ? KW_FEW : KW_FEW / 2;
    if (!a.kv.f16)
        launch_hd<float, float>(st, a);
    else if (a.q_f16)
        launch_hd<_Float16, _Float16>(st, a);
    else
        launch_hd<float, _Float16>(st, a);
    return hipGetLastError();
}

}  // namespace styx
