// attn_chunk.hip -- causal attention of the new tokens of a batch over their
// sequences' slots of a paged KV cache.
//
// Token i of sequence b with n = len[b] rows, query head h of kv head j:
//   s_t = scale q . K[t], t <= n + i (and t > n + i - window), pages in the pool
//   M = max s_t, L = sum e^(s_t - M), out = sum e^(s_t - M) V[t] / L, lse = M + ln L
//
// A workgroup takes a tile of query rows -- a row is a token and one of a kv
// head's gqa heads, token by token -- and goes once over the slots that they see,
// in blocks that lie in LDS for its waves, the next block under way meanwhile.
// Scores are formed transposed, slots x queries: lane (n = lane & 31, h = lane >>
// 5) then has its own query's scores of slots 8 (i / 4) + 4 h + i % 4 of each 32,
// the softmax factors are lane-local, and they are the operand of the value
// product as they stand.
//
// Bound: the matrix cores, and for narrow heads the exponentials beside them.
// 32 query heads over 4 kv heads of 128, f16, a prompt of 8192 tokens (550
// GFLOP): 600 us, 915 of the 1146 TFLOP/s that a product of 8192^3 reaches.  Half
// of a CU's cycles have a product under way, and the clock is at 1.77 to 1.85 GHz
// under them: with q, K and V all 0 the same launch takes as many cycles, at up to
// 2.4 GHz, and 450 us.  f32 queries on f16 rows, 406 GFLOP in two pieces: 473 us,
// 860 TFLOP/s.  f32, three documents, heads of 256, 211 GFLOP: 1.75 ms, 121 of 152
// TFLOP/s.  f16 heads of 64 under a window of 1024, 21 GFLOP: 50 us; a score costs
// 256 FLOP there and its exponential, maximum, sum and rounding more time than
// they, which explains about half of the distance to the products' 18.
//
// Why 32 rows a wave: their queries, sums and scores stay in 256 registers; 64
// rows moved sums between register files in every block (1494 us).  Why four
// waves a block, two workgroups a CU: while one waits at a barrier the other
// multiplies; with eight waves (256 rows) the prompt took as long, one of 2048
// tokens 77 us against 65, a mixed step 472 against 458.
#include <algorithm>
#include <type_traits>

#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// The other lane of the same query.
__device__ __forceinline__ float other_half(float v)
{
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? x[0] : x[1]);
}
// A value that all lanes have, for the scalar unit.
template <typename T> __device__ __forceinline__ T uniform(T v)
{
    return by_words(v, [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); });
}

// 16 bytes a lane from memory to LDS at off + 16 lane (off uniform), in the
// background: the caller waits (landed) before it reads them.  Not the builtin:
// behind that the compiler waits for all of them before any read of LDS.
__device__ __forceinline__ void to_lds(const void *from, uint32_t off)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(off), "v"(from) : "memory");
}
__device__ __forceinline__ void to_lds(const void *base, uint32_t at, uint32_t off)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(off), "v"(at), "s"(base) : "memory");
}
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_at(const char *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p; }

// Factors are 2^(x - m + AC_OFF), with a reference m that follows the largest
// score x (in units of ln 2) only when that is more than AC_LAG above it: the
// sums are then multiplied rarely.  Factors stay below 2^(AC_OFF + AC_LAG),
// within f16, and are normal f16 numbers down to 2^-21 of the largest.
constexpr float AC_OFF = 7.0f, AC_LAG = 8.0f;

// How a head of HD values of type TC lies in a block in LDS: rows one after
// another, 16-byte pieces permuted within 256 bytes so that the 16 rows of a
// score operand, and the 4 rows by 64 bytes of a value operand, lie in banks
// of their own.
template <typename TC, int HD> struct Lay {
    static constexpr int ROW = HD * (int)sizeof(TC), LPR = ROW / 16, RPI = 64 / LPR;
    static __device__ __forceinline__ int perm(int t)
    {
        return ROW == 128 ? (((t >> 1) & 1) << 2) | ((t >> 2) & 3) : ((t & 3) << 2) | ((t >> 2) & 3);
    }
    // byte of dim d of row t
    static __device__ __forceinline__ int at(int t, int d)
    {
        const int b = d * (int)sizeof(TC);
        return t * ROW + (((b >> 4) ^ perm(t)) << 4) + (b & 15);
    }
};

// The bits of a word whose values are not finite.
template <typename TC> __device__ __forceinline__ uint32_t not_finite(uint32_t v)
{
    if constexpr (sizeof(TC) == 4) return (v & 0x7F800000u) == 0x7F800000u ? ~0u : 0u;
    return (((v & 0x7FFF7FFFu) + 0x04000400u) >> 15 & 0x00010001u) * 0xFFFFu;
}

// Nothing is moved across: the products below are written in the order in which
// they are to be issued, operand reads some matrix instructions ahead of their
// use, the factors' arithmetic between matrix instructions.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// RG: groups of 32 rows in a tile.
template <typename TQ, typename TC, int HD, int RG = 4> struct Wave;

// f16 caches: v_mfma_f32_32x32x16_f16.  f32 queries and their factors are two
// f16 pieces each, hi + lo with |x - hi - lo| <= 2^-22 |x|, queries brought to
// [2^9, 2^10) by a power of two per row so that the low pieces of all that
// counts are normal numbers.  f16 queries take factors rounded to f16: an
// error of at most 2^-11 of each, as large as the output's own rounding.
template <typename TQ, int HD> struct Wave<TQ, _Float16, HD, 4> {
    using TC = _Float16;
    using La = Lay<TC, HD>;
    static constexpr int NP = sizeof(TQ) == 4 ? 2 : 1;  // pieces
    // waves that share a query's dims, dims of a wave (f16 queries with heads of
    // 256: with one, registers spill; with two, both form all factors.  Neither
    // wins everywhere.  16 heads, a prompt of 2048 tokens 95 us with two, 122 with
    // one, single tokens of 16 sequences over 4000 slots 40 and 56; but a prompt of
    // 4096 270 and 265, eight of 512 74 and 65, four chunks of 256 tokens behind
    // 8000 slots 233 and 220)
    static constexpr int DS = HD == 256 ? 2 : 1, HW = HD / DS, NK = HW / 16, ND = HW / 32;
    static constexpr int KT = HD == 256 ? 32 : 64;
    static constexpr int NW = 4 * DS, PER_CU = 8 / NW, BM = 128;
    static constexpr int IDLE = 5, BUSY = 16, ALONE = 0;  // line_of
    static constexpr float PART = HD / 3000.0f;  // (half to twice of it: within 10%)
    h8 q[NP][NK], p[KT / 32][NP][2];
    f16v s[KT / 32], o[ND];
    float mul, ref, sum[2];  // score to factor: 2^(s mul + ref); the factors' sum
    int lane;

    // row: this wave's dims of the query, the first of which is d0
    __device__ __forceinline__ void init(const TQ *row, int d0, float scale)
    {
        const int h = lane >> 5;
        // (a scale of 0 goes into q: -infinity times it would be NaN)
        const float a = scale == 0.0f ? 1.0f : fabsf(scale), sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
        if constexpr (NP == 1) {
            mul = a;
#pragma unroll
            for (int i = 0; i < NK; i++) q[0][i] = *(const h8 *)(row + 16 * i + 8 * h) * (_Float16)sign;
        } else {
            styx_f4 v[NK][2];
            float m = 0.0f;
            if constexpr (DS == 2) {  // the dims of the other wave
#pragma unroll
                for (int i = 0; i < NK; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const styx_f4 y = *(const styx_f4 *)(row + (HW - 2 * d0) + 16 * i + 8 * h + 4 * j);
#pragma unroll
                        for (int e = 0; e < 4; e++) m = fmaxf(m, fabsf(y[e]));
                    }
            }
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    v[i][j] = *(const styx_f4 *)(row + 16 * i + 8 * h + 4 * j);
#pragma unroll
                    for (int e = 0; e < 4; e++) m = fmaxf(m, fabsf(v[i][j][e]));
                }
            m = fmaxf(m, other_half(m));
            const int e = m > 0.0f && m < INFINITY ? (int)((__float_as_uint(m) >> 23) & 255) - 127 : 9;
            // 2^(9 - e), in range for every exponent: 9 - e within [-118, 136]
            const float up = e < -100 ? ldexpf(1.0f, 109) : ldexpf(1.0f, 9 - e);
            mul = a / up;
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const float y = v[i][x >> 2][x & 3] * (up * sign);
                    const _Float16 hi = (_Float16)y;
                    q[0][i][x] = hi;
                    q[NP - 1][i][x] = (_Float16)(y - (float)hi);
                }
        }
    }
    // The scores of 32 slots, with fill(j, N) done behind the j-th of N operands.
    template <typename F> __device__ __forceinline__ void scores(int kt, const char *kb, int d0, F fill)
    {
        static_assert(DS == 1 || 2 * HW % 256 == 0, "whole permuted pieces");
        kb += 2 * d0;
        constexpr int AHEAD = 4;
        const int m = lane & 31, h = lane >> 5;
        const f16v zero = {};
        const int at = m * La::ROW + ((h ^ La::perm(m)) << 4);
        // (piece 2 i + h: its bits above 256 bytes are not permuted)
        auto read = [&](int i) { return *(const h8 *)(kb + (at ^ ((32 * i) & 255)) + ((32 * i) & ~255) + kt * 32 * La::ROW); };
        h8 k[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) k[i] = read(i);
        in_order();
#pragma unroll
        for (int i = 0; i < NK; i++) {
#pragma unroll
            for (int x = 0; x < NP; x++)
                s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i % AHEAD], q[x][i], i + x == 0 ? zero : s[kt], 0, 0, 0);
            if (i + AHEAD < NK) k[i % AHEAD] = read(i + AHEAD);
            fill(i, NK);
            in_order();
        }
    }
    // The factor of score i of 32 slots.
    __device__ __forceinline__ void factor(int kt, int i)
    {
        const float f = exp2_(fmaf(s[kt][i], mul, ref));
        sum[i & 1] += f;
        asm volatile("" : "+v"(sum[i & 1]));  // (here, not behind the products)
        const _Float16 hi = (_Float16)f;
        p[kt][0][i >> 3][i & 7] = hi;
        if constexpr (NP == 2) p[kt][1][i >> 3][i & 7] = (_Float16)(f - (float)hi);
    }
    // o += factors of 32 slots times V, with fill(j, N) done behind the j-th of N
    // operands; the factors of a step of 16 slots are needed at its first.
    template <typename F> __device__ __forceinline__ void values(int kt, const char *vb, int d0, F fill)
    {
        vb += 2 * d0;
        constexpr int N = 2 * ND, AHEAD = 4;
        const int h = lane >> 5, u = (lane >> 4) & 1, kk = (lane & 15) >> 2;
        // piece of dims 16 u + 4 (lane & 3) .. of the first 32, row kk + 4 (h + 2 r)
        auto at = [&](int r) {
            const int t = kk + 4 * h + 8 * r;
            return t * La::ROW + (((2 * u + ((lane & 3) >> 1)) ^ La::perm(t)) << 4) + 8 * (lane & 1);
        };
        const int at0 = at(0), at1 = at(1);
        typedef __attribute__((address_space(3))) s4 *lds4;
        union Part {
            s4 part[2];
            h8 v;
        };
        auto read = [&](int j) {
            const int d = j % ND, k = 2 * kt + j / ND;
            const int flip = (64 * d) & (La::ROW < 256 ? La::ROW - 1 : 255), far = ((64 * d) & ~255) + k * 16 * La::ROW;
            Part x;
            x.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vb + (at0 ^ flip) + far));
            x.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vb + (at1 ^ flip) + far));
            return x.v;
        };
        h8 v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) v[j] = read(j);
        in_order();
#pragma unroll
        for (int j = 0; j < N; j++) {
#pragma unroll
            for (int y = 0; y < NP; y++)
                o[j % ND] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[j % AHEAD], p[kt][y][j / ND], o[j % ND], 0, 0, 0);
            if (j + AHEAD < N) v[j % AHEAD] = read(j + AHEAD);
            fill(j, N);
            in_order();
        }
    }
    // All but the scores times c, a power of two; `pending`: factors of the first
    // 32 slots that have not met V.  Those in f32, as c need not be an f16 number:
    // below 2^-24 it would be 0, where a factor of up to 2^15 times it is one.
    __device__ __forceinline__ void rescale(float c, bool pending)
    {
        sum[0] *= c;
        sum[1] *= c;
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] *= c;
        if (pending)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float f = (float)p[0][0][i >> 3][i & 7];
                if constexpr (NP == 2) f += (float)p[0][1][i >> 3][i & 7];
                f *= c;
                const _Float16 hi = (_Float16)f;
                p[0][0][i >> 3][i & 7] = hi;
                if constexpr (NP == 2) p[0][1][i >> 3][i & 7] = (_Float16)(f - (float)hi);
            }
    }
};

// f32 caches: v_mfma_f32_32x32x2_f32, dims in fours on both sides of the score
// product for 16-byte reads.  Sequences of at most 64 or 32 query rows would leave
// two or three of four waves without any: two or four waves take the same rows,
// each a part of the dims (one token over 2000 slots: 22.3 us with two, 18.3 with
// four; over 32000 58 and 45; more: with_kernel).
template <int HD, int RG> struct Wave<float, float, HD, RG> {
    using TC = float;
    using La = Lay<TC, HD>;
    static constexpr int DS = HD == 256 && RG == 4 ? 2 : 4 / RG, HW = HD / DS, NK = HW / 8, ND = HW / 32;
    static constexpr int KT = 32;
    static constexpr int NW = RG * DS, PER_CU = HD == 256 ? 1 : 2, BM = 32 * RG;
    static constexpr int IDLE = HD == 64 ? 2 : 1, BUSY = 8, ALONE = PER_CU == 2 ? 12 : 0;
    static constexpr float PART = 0.025f * RG / 4;
    styx_f4 q[NK];
    f16v s[1], o[ND];
    float mul, ref, sum[2], p[2];
    int lane;

    __device__ __forceinline__ void init(const float *row, int, float scale)
    {
        const int h = lane >> 5;
        mul = scale == 0.0f ? 1.0f : fabsf(scale);
        const float sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < NK; i++) q[i] = *(const styx_f4 *)(row + 8 * i + 4 * h) * sign;
    }
    template <typename F> __device__ __forceinline__ void scores(int, const char *kb, int d0, F)
    {
        const int m = lane & 31, h = lane >> 5;
        const f16v zero = {};
        const int at = (m * La::ROW + ((h ^ La::perm(m)) << 4)) ^ ((4 * d0) & 255);
        kb += (4 * d0) & ~255;
        f16v c[2];  // two chains: a product follows the one before on its sum at once otherwise
        constexpr int AHEAD = 2;
        auto read = [&](int i) { return *(const styx_f4 *)(kb + (at ^ ((32 * i) & 255)) + ((32 * i) & ~255)); };
        styx_f4 k[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) k[i] = read(i);
        in_order();
#pragma unroll
        for (int i = 0; i < NK; i++) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                c[e & 1] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[i % AHEAD][e], q[i][e], i == 0 && e < 2 ? zero : c[e & 1], 0, 0, 0);
            if (i + AHEAD < NK) k[i % AHEAD] = read(i + AHEAD);
            in_order();
        }
        s[0] = c[0] + c[1];
    }
    __device__ __forceinline__ void factor(int, int i)
    {
        p[i & 1] = exp2_(fmaf(s[0][i], mul, ref));
        sum[i & 1] += p[i & 1];
    }
    template <typename F> __device__ __forceinline__ void values(int, const char *vb, int d0, F fill)
    {
        constexpr int N = 16 * ND, AHEAD = 8;
        const int m = lane & 31, h = lane >> 5;
        vb += (4 * d0) & ~255;
        auto read = [&](int j) {
            const int d = j % ND, i = j / ND, t = 8 * (i >> 2) + 4 * h + (i & 3);
            const int at = (t * La::ROW + (((m >> 2) ^ La::perm(t)) << 4) + 4 * (m & 3)) ^ ((4 * d0) & 255);
            return *(const float *)(vb + (at ^ ((128 * d) & 255)) + ((128 * d) & ~255));
        };
        float v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) v[j] = read(j);
        in_order();
#pragma unroll
        for (int j = 0; j < N; j++) {
            o[j % ND] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[j % AHEAD], p[j / ND & 1], o[j % ND], 0, 0, 0);
            if (j + AHEAD < N) v[j % AHEAD] = read(j + AHEAD);
            fill(j, N);
            in_order();
        }
    }
    __device__ __forceinline__ void rescale(float c, bool)
    {
        sum[0] *= c;
        sum[1] *= c;
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] *= c;
    }
};

// ------------------------------------------------------------- the split ---
// The work of a kv head is a line: sequences one after another, of each its
// tiles of query rows, of each tile its blocks.  Either a workgroup takes a
// tile, the longest of a sequence first, or every workgroup takes an equal
// share of the line, as many as run at once: a share ends inside a tile, whose
// pieces are joined afterwards.  Both are known from the lengths alone, to every
// workgroup by itself.
constexpr int AC_CUS = 256;
constexpr int AC_TILE = 4;    // what a tile's start costs, in blocks (its rows of q, its first blocks)

// A sequence's part of the line: tile t is first + t step long, in slots times
// rows of a token.  (With a tile's start: of a prompt's many short first tiles a
// share would else hold a dozen.  4096 tokens, head_dim 256, with a wave to every
// 32 rows: 351 us, 257 with.)
struct SeqLine {
    int tiles, blocks;  // of the longest tile
    int64_t first, step;
    __device__ __forceinline__ int64_t upto(int64_t t) const { return t * first + step * (t * (t - 1) / 2); }
};
template <int BM, int KT> __device__ __forceinline__ SeqLine seq_line(const AttnChunkArgs &a, const ChunkSeq &s)
{
    if (s.count == 0) return {0, 0, 0, 0};
    const int tiles = (s.count * a.gqa + BM - 1) / BM;
    const int64_t most = (int64_t)a.window * a.gqa + BM;
    const int64_t start = (int64_t)AC_TILE * KT * a.gqa;
    const int end = (s.len + s.count + KT - 1) / KT;
    if (a.window && most < ((int64_t)s.len + s.count) * a.gqa)
        return {tiles, min(end, (int)((a.window + (int64_t)BM / a.gqa + KT - 1) / KT) + 1), most + start, 0};
    return {tiles, end, (int64_t)s.len * a.gqa + BM + start, BM};
}
struct Line {
    int64_t share, total;  // share 0: by tiles
};
template <typename W> __device__ __forceinline__ Line line_of(const AttnChunkArgs &a)
{
    constexpr int BM = W::BM, KT = W::KT, slots = AC_CUS * W::PER_CU;
    const int lane = threadIdx.x & 63;
    int64_t tiles = 0, total = 0;
    int longest = 0;
    for (int b0 = 0; b0 < a.kv.n_seq; b0 += 64) {
        const SeqLine w = seq_line<BM, KT>(a, chunk_seq(a.chunk, a.kv, b0 + lane));
        tiles += w.tiles;
        total += w.upto(w.tiles);
        longest = max(longest, w.blocks);
    }
    tiles = uniform(wave_total(tiles));
    total = uniform(wave_total(total));
    longest = uniform(wave_most(longest));
    if (tiles == 0) return {0, 0};
    // What either costs: tiles that all run at once take as long as the longest,
    // more of them leave half a tile's time unused at the end; shares cost their
    // partial results and the joining, little on a chip that is mostly idle
    // (IDLE blocks, f16: one token over 400 slots 11.5 us cut, 15.1 by tiles, 20
    // tokens over 300 slots 19.4 and 14.8) and more where all write at once
    // (BUSY: a prompt of 2048 tokens 74 us cut, 63 by tiles).
    const int64_t unit = (int64_t)KT * a.gqa, even = total * a.kv.nkv / slots;
    const int64_t by_tiles = tiles * a.kv.nkv <= slots ? (longest + AC_TILE) * unit : even + total / tiles / 2;
    const int start = 8 * tiles * a.kv.nkv <= slots ? W::IDLE : W::BUSY;
    if (by_tiles <= even + even / 10 + (start + AC_TILE) * unit) return {0, tiles};
    // Shares of fewer blocks only add partial results.  n blocks in shares of l
    // take the time of l blocks and of n / l partial results, each PART of a
    // block's for a whole tile: least for l = sqrt(n PART).  (64 f16 tokens over
    // 2000 slots: 27 us with 4 blocks at least, 39 with one; one token 15.3 and 13.)
    const float blocks = (float)(total * a.kv.nkv) / (float)unit;
    const float full = fminf(1.0f, (float)a.chunk.n_rows * a.gqa / ((float)tiles * BM));
    const int64_t least = max((int)__builtin_amdgcn_sqrtf(blocks * full * W::PART), 1) * unit;
    // Of two workgroups of f32 products on a CU each takes twice the time: one
    // where it has fewer than ALONE blocks (8 tokens over 2000 slots 20 us, 22 with
    // two; single tokens of 24 sequences over 2000 slots, 23 blocks, 65 and 52).
    const int64_t shares = max((blocks < W::ALONE * AC_CUS ? AC_CUS : slots) / a.kv.nkv, 1);
    return {uniform(max((total + shares - 1) / shares, least)), total};
}

// A tile and what of its length lies before `at`.  TILES: `at` counts tiles, the
// last of each sequence first.  b < 0: past the end.
struct Place {
    int b, tile;
    int64_t in, length, before;  // at - before = in, of length
    ChunkSeq s;
};
template <int BM, int KT, bool TILES> __device__ __forceinline__ Place find_place(const AttnChunkArgs &a, int64_t at)
{
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.kv.n_seq; b0 += 64) {
        const ChunkSeq s = chunk_seq(a.chunk, a.kv, b0 + lane);
        const SeqLine w = seq_line<BM, KT>(a, s);
        const int64_t mine = TILES ? w.tiles : w.upto(w.tiles), upto = base + wave_upto(mine);
        if (const unsigned long long hit = __ballot(upto > at)) {
            const int l = __builtin_ctzll(hit);
            const SeqLine o{(int)__builtin_amdgcn_readlane(w.tiles, l), 0, of_lane(w.first, l), of_lane(w.step, l)};
            const int64_t start = of_lane(upto, l) - of_lane(mine, l), in = at - start;
            int tile = 0;
            if (TILES)
                tile = o.tiles - 1 - (int)in;
            else
                for (int n = o.tiles; n > 1;) {  // the last tile that begins at or before it
                    const int half = n >> 1;
                    const bool on = o.upto(tile + half) <= in;
                    tile += on ? half : 0;
                    n = on ? n - half : half;
                }
            const int64_t before = o.upto(tile);
            return {b0 + l, tile, TILES ? 0 : in - before, o.upto(tile + 1) - before, start + before,
                    {(int)__builtin_amdgcn_readlane(s.first, l), (int)__builtin_amdgcn_readlane(s.count, l),
                     (int)__builtin_amdgcn_readlane(s.len, l)}};
        }
        base = of_lane(upto, 63);
    }
    return {-1, 0, 0, 0, 0, {0, 0, 0}};
}

// ------------------------------------------------------------- the tiles ---
// A tile that begins in a share and goes on in the next: its pieces, one in
// each of as many shares, the first at `part0`.  pieces 0: there is none.
struct alignas(16) Across {
    int pieces, row0, part0;
    ChunkSeq s;
};
// Partial results, of a share's first piece and of its last (sums o, and m and
// l), and the tiles that they are of, by share and kv head.
struct Parts {
    float *o;
    float2 *ml;
    Across *across;
    int rows, shares;  // of a piece; at most
};

template <typename TQ, typename TC, int HD, int RG>
__global__ void __launch_bounds__((64 * Wave<TQ, TC, HD, RG>::NW), (Wave<TQ, TC, HD, RG>::PER_CU * Wave<TQ, TC, HD, RG>::NW / 4))
    k_attn_chunk(AttnChunkArgs a, Parts parts)
{
    using W = Wave<TQ, TC, HD, RG>;
    using La = Lay<TC, HD>;
    constexpr int KT = W::KT, DS = W::DS, HW = W::HW, BM = W::BM, ND = W::ND;
    constexpr int NW = W::NW, WG = 64 * NW, BLOCK = KT * La::ROW, PER_WAVE = KT / NW, NI = PER_WAVE / La::RPI;
    static_assert(PER_WAVE % La::RPI == 0, "whole loads");
    __shared__ __align__(1024) char s_k[2][BLOCK];
    __shared__ __align__(1024) char s_v[2][BLOCK];
    // scores of half the dims; in the block of K where there is no other place
    constexpr int PIECES = 4;
    constexpr bool APART = 4 * BLOCK + NW * PIECES * 1024 <= 163840 / W::PER_CU;
    __shared__ styx_f4 s_half[DS > 1 && APART ? NW * PIECES : 1][64];
    const KvView &kv = a.kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int dw = wave % DS * HW;  // the wave's first dim
    const Line line = line_of<W>(a);
    const int kvh = blockIdx.x % kv.nkv, nth = blockIdx.x / kv.nkv;
    int64_t u = nth * line.share;
    const int64_t end = min(u + line.share, line.total);
    const int64_t stride = (int64_t)kv.nkv * La::ROW;
    const char *kp = (const char *)kv.kpool + kvh * La::ROW, *vp = (const char *)kv.vpool + kvh * La::ROW;
    const uint32_t lk = lds_at(&s_k[0][0]), lv = lds_at(&s_v[0][0]);
    if (threadIdx.x == 0 && nth < parts.shares) parts.across[nth * kv.nkv + kvh].pieces = 0;
    for (bool more = true; more;) {
    // (a lane number that the compiler takes for a new one in every trip: what
    // is computed from it would else be kept in registers over the trips)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int n = lane & 31, h = lane >> 5;
    const Place it = line.share ? find_place<BM, KT, false>(a, u) : find_place<BM, KT, true>(a, nth);
    if (it.b < 0 || (line.share && u >= end)) return;
    const ChunkSeq &s = it.s;
    const int rows = s.count * a.gqa, row0 = it.tile * BM;
    // tokens of the tile, the slots that any of them sees, the piece's blocks
    const int tok0 = a.by_gqa.of(row0), tok1 = a.by_gqa.of(min(row0 + BM, rows) - 1);
    const int t1 = s.len + tok1 + 1, t0 = a.window && s.len + tok0 >= a.window ? s.len + tok0 - a.window + 1 : 0;
    int b0 = t0 / KT, b1 = (t1 + KT - 1) / KT;
    bool whole = true;
    // a piece that is not whole is its share's first, or its last, which goes on
    // in the next share's first
    const int64_t part = (2 * (int64_t)nth + (it.in == 0 && u > nth * line.share)) * kv.nkv + kvh;
    more = false;
    if (line.share) {
        const int64_t to = min(it.in + (end - u), it.length);
        whole = it.in == 0 && to == it.length;
        if (!whole) {
            const int64_t nb = b1 - b0;
            b1 = b0 + (int)((uint64_t)(to * nb) / (uint64_t)it.length);
            b0 += (int)((uint64_t)(it.in * nb) / (uint64_t)it.length);
        }
        u += to - it.in;
        more = u < end;
        if (threadIdx.x == 0 && it.in == 0 && !whole) {
            const int pieces = (int)((it.before + it.length - 1) / line.share) - nth + 1;
            parts.across[nth * kv.nkv + kvh] = Across{pieces, row0, (int)(part / kv.nkv), s};
        }
    }
    b0 = uniform(b0);
    b1 = uniform(b1);
    const int32_t *tab = kv.table + (int64_t)it.b * kv.table_len;

    // this lane's query
    W x;
    x.lane = lane;
    const int wrow0 = row0 + 32 * (wave / DS);
    const bool works = wrow0 < rows;
    const int r = min(wrow0 + n, rows - 1), tok = a.by_gqa.of(r), head = kvh * a.gqa + (r - tok * a.gqa);
    const int at = wrow0 + n < rows ? s.len + tok : -1;  // last slot seen, -1: no such row
    const int64_t orow = s.first + tok;                  // row of q and out
    // the reference: a whole number, or the first block's largest score, whose
    // factor then has no rounding to f16 (a token that sees one slot gets its V)
    constexpr bool ONE = sizeof(TQ) == 2;
    float m = -INFINITY;
    x.ref = AC_OFF;
    x.sum[0] = x.sum[1] = 0.0f;
    constexpr int NANS = (HW + 63) / 64;
    uint32_t nan_at[NANS];  // dims that are NaN whatever the sums are
#pragma unroll
    for (int w = 0; w < NANS; w++) nan_at[w] = 0;
    x.init((const TQ *)a.q + orow * a.ldq + (int64_t)head * HD + dw, dw, a.scale);
#pragma unroll
    for (int d = 0; d < ND; d++) x.o[d] = f16v{};
    // slots that all of the wave's queries see, and those that none sees
    const int wtok0 = a.by_gqa.of(min(wrow0, rows - 1)), wtok1 = a.by_gqa.of(min(wrow0 + 32, rows) - 1);
    const int all_hi = s.len + wtok0, any_hi = s.len + wtok1;
    const int all_lo = a.window ? s.len + wtok1 - a.window + 1 : 0, any_lo = a.window ? s.len + wtok0 - a.window + 1 : 0;

    // rows of the pools: a lane's slot of a block (KT = 32: both halves alike)
    const int my = lane & (KT - 1);
    auto entry_of = [&](int blk) { return kv.entry(tab, min(blk * KT + my, t1 - 1)); };
    auto row_of = [&](int e, int blk) { return blk * KT + my < t1 ? kv.row_of(e, min(blk * KT + my, t1 - 1)) : -1; };
    // where a lane's 16 bytes of a load come from, of the first of the wave's rows
    uint32_t from[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int t = i * La::RPI + lane / La::LPR;
        from[i] = t * (uint32_t)stride + 16 * ((lane & (La::LPR - 1)) ^ La::perm(wave * PER_WAVE + t));
    }
    auto fetch = [&](int buf, int row) {
        const uint32_t to = buf * BLOCK + wave * PER_WAVE * La::ROW;
        if (a.runs) {  // a wave's rows lie one after another
            const int64_t off = (int64_t)max((int)__builtin_amdgcn_readlane(row, wave * PER_WAVE), 0) * stride;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                to_lds(kp + off, from[i], lk + to + i * 1024);
                to_lds(vp + off, from[i], lv + to + i * 1024);
            }
        } else {
            int64_t off[NI];
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int t = wave * PER_WAVE + i * La::RPI + lane / La::LPR;
                off[i] = max(__shfl(row, t), 0) * stride + 16 * ((lane & (La::LPR - 1)) ^ La::perm(t));
            }
#pragma unroll
            for (int i = 0; i < NI; i++) {
                to_lds(kp + off[i], lk + to + i * 1024);
                to_lds(vp + off[i], lv + to + i * 1024);
            }
        }
    };
    unsigned long long there = 0;  // slots of the block under way whose page is there
    int entry = 0;
    if (b0 < b1) {
        const int row = row_of(entry_of(b0), b0);
        there = __ballot(row >= 0);
        fetch(0, row);
        entry = entry_of(min(b0 + 1, b1 - 1));
    }
    constexpr unsigned long long full = ~0ull;
    for (int blk = b0; blk < b1; blk++) {
        const int buf = (blk - b0) & 1;
        landed();
        __syncthreads();
        const unsigned long long seen = there;
        if (blk + 1 < b1) {
            const int row = row_of(entry, blk + 1);
            there = __ballot(row >= 0);
            fetch(buf ^ 1, row);
            entry = entry_of(min(blk + 2, b1 - 1));
        }
        const int tb = blk * KT;
        const char *kb = s_k[buf], *vb = s_v[buf];
        // the slots of the block that this lane's query sees
        uint32_t vis[KT / 32];
        // (uniform over the workgroup: whether every query of the tile sees the block)
        if (seen != full || tb + KT - 1 > s.len + tok0 || (a.window && tb <= s.len + tok1 - a.window)) {
#pragma unroll
            for (int kt = 0; kt < KT / 32; kt++) {
                const int last = at - (tb + 32 * kt), before = a.window ? last - a.window : -1;
                uint32_t v = (uint32_t)(seen >> (32 * kt));
                v &= last < 0 ? 0u : last > 30 ? ~0u : (2u << last) - 1u;
                v &= before < 0 ? ~0u : before > 30 ? 0u : ~0u << (before + 1);
                vis[kt] = v;
            }
            // A value that is not finite must not reach those that do not see
            // it, whose factor is 0: where there is one, the dims of those that
            // do see it are noted to be NaN, and the value becomes 0.
            char *mine = s_v[buf] + (64 * wave + lane) * (BLOCK / WG);
            bool odd = false;
#pragma unroll
            for (int i = 0; i < BLOCK / WG; i += 16) {
                const styx_u4 v = *(const styx_u4 *)(mine + i);
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= not_finite<TC>(v[e]) != 0;
            }
            bool any;
            if constexpr (DS > 1 && APART) {
                // (in the place of the scores: those of the last block have been
                // read, and there may be no more LDS)
                int *const odds = (int *)s_half;
                const bool mine_odd = __ballot(odd) != 0;
                if (lane == 0) odds[wave] = mine_odd;
                __syncthreads();
                any = __ballot(lane < NW && odds[lane & (NW - 1)]) != 0;
                __syncthreads();
            } else {
                any = __syncthreads_or(odd) != 0;
            }
            if (any) {
#pragma unroll 1
                for (int t = 0; t < KT; t++) {
                    const uint32_t see = 0u - (vis[KT == 64 ? t >> 5 : 0] >> (t & 31) & 1);
                    // bits 4 j + e: dims 8 j + 4 h + e
#pragma unroll 1
                    for (int j = 0; j < HW / 8; j++) {
                        const TC *v = (const TC *)(vb + La::at(t, dw + 8 * j + 4 * h));
                        uint32_t bad = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) bad |= (uint32_t) !(fabsf((float)v[e]) < INFINITY) << e;
                        if (bad)
#pragma unroll
                            for (int w = 0; w < NANS; w++) nan_at[w] |= w == j >> 3 ? (bad & see) << (4 * (j & 7)) : 0;
                    }
                }
                __syncthreads();
                for (int i = 0; i < BLOCK / WG; i += 4) {
                    uint32_t *v = (uint32_t *)(mine + i);
                    *v &= ~not_finite<TC>(*v);
                }
                __syncthreads();
            }
        }
        const bool idle = !works || tb > any_hi || tb + KT <= any_lo;
        const bool masked = seen != full || tb + KT - 1 > all_hi || tb < all_lo;
        auto mask = [&](int kt) {
            const uint32_t mine = vis[kt] >> (4 * h);
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (!(mine >> (8 * (i >> 2) + (i & 3)) & 1)) x.s[kt][i] = -INFINITY;
        };
        auto follow = [&](int kt) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i += 2) mx = fmaxf(fmaxf(mx, x.s[kt][i]), x.s[kt][i + 1]);
            mx = fmaxf(mx, other_half(mx)) * x.mul;
            if (__ballot(mx > m + AC_LAG)) {
                // (by whole numbers, so that sums are multiplied by powers of two)
                const float mn = !ONE ? fmaxf(m, ceilf(mx)) : m == -INFINITY ? mx : m + fmaxf(ceilf(mx - m), 0.0f);
                if (mn != -INFINITY) {
                    x.rescale(exp2_(m - mn), kt > 0);
                    x.ref = AC_OFF - mn;
                }
                m = mn;
            }
        };
        auto nothing = [](int, int) {};
        if constexpr (KT == 64) {
            // the products of one half of the block while the other's factors are formed
            if (idle) continue;
            auto factors = [&](int kt, int j, int steps) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (i / (16 / steps) == j) x.factor(kt, i);
            };
            x.scores(0, kb, 0, nothing);
            if (masked) mask(0);
            follow(0);
            x.scores(1, kb, 0, [&](int j, int steps) { factors(0, j, steps); });
            if (masked) mask(1);
            follow(1);
            x.values(0, vb, 0, [&](int j, int steps) { factors(1, j, steps); });
            x.values(1, vb, 0, nothing);
        } else {
            if constexpr (DS == 1) {
                if (idle) continue;
                x.scores(0, kb, 0, nothing);
            } else {
                // each of DS waves has a part of the dims: all add the parts up
                styx_f4 (*half)[64] = APART ? s_half : (styx_f4(*)[64])s_k[buf];
                if (!idle) x.scores(0, kb, dw, nothing);
                if constexpr (!APART) {
                    static_assert(NW * PIECES * 1024 <= BLOCK, "scores in the place of K");
                    __syncthreads();
                }
                if (!idle)
#pragma unroll
                    for (int i = 0; i < PIECES; i++)
                        half[wave * PIECES + i][lane] = styx_f4{x.s[0][4 * i], x.s[0][4 * i + 1], x.s[0][4 * i + 2], x.s[0][4 * i + 3]};
                __syncthreads();
                if (idle) continue;
#pragma unroll
                for (int i = 0; i < PIECES; i++) {
                    styx_f4 y = half[(DS == 2 ? wave ^ 1 : wave & -DS) * PIECES + i][lane];
                    if constexpr (DS == 2) {
#pragma unroll
                        for (int e = 0; e < 4; e++) x.s[0][4 * i + e] += y[e];
                    } else {  // in one order, so that they all have the same sums
#pragma unroll
                        for (int w = 1; w < DS; w++) y += half[((wave & -DS) + w) * PIECES + i][lane];
#pragma unroll
                        for (int e = 0; e < 4; e++) x.s[0][4 * i + e] = y[e];
                    }
                }
            }
            if (masked) mask(0);
            follow(0);
            // factors a step ahead of their product: 8 of f16 caches, one of f32
            constexpr int LEAD = sizeof(TC) == 2 ? 8 : 1;
#pragma unroll
            for (int i = 0; i < LEAD; i++) x.factor(0, i);
            x.values(0, vb, dw, [&](int j, int steps) {
                if constexpr (sizeof(TC) == 4) {
                    if (j % (steps / 16) == 0 && j < steps - steps / 16) x.factor(0, j / (steps / 16) + 1);
                } else {
#pragma unroll
                    for (int i = LEAD; i < 16; i++)
                        if ((i - LEAD) * steps / 16 == j) x.factor(0, i);
                }
            });
        }
    }
    if (more) __syncthreads();  // (the next piece's blocks take the place of this one's)
    if (at < 0) continue;
    float l = x.sum[0] + x.sum[1];
    l += other_half(l);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (nan_at[d / 2] >> (16 * (d & 1) + i) & 1) x.o[d][i] = NAN;
    if (!whole) {
        const int64_t p = part * parts.rows + (wrow0 - row0) + n;
        if (h == 0 && dw == 0) parts.ml[p] = float2{m, l};
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(styx_f4 *)(parts.o + p * HD + dw + 32 * d + 2 * i + 4 * h) =
                    styx_f4{x.o[d][i], x.o[d][i + 1], x.o[d][i + 2], x.o[d][i + 3]};
        continue;
    }
    // no slot with a weight (m = -inf): 0, or NaN
    const bool none = m == -INFINITY;
    const float f = none ? 1.0f : 1.0f / l, add = none ? l : 0.0f;
    TQ *out = (TQ *)a.out + orow * a.ldo + (int64_t)head * HD + dw;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            TQ *dst = out + 32 * d + 2 * i + 4 * h;
            if constexpr (sizeof(TQ) == 2) {
                h4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = (_Float16)(x.o[d][i + e] * f + add);
                *(h4 *)dst = v;
            } else {
                styx_f4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = x.o[d][i + e] * f + add;
                *(styx_f4 *)dst = v;
            }
        }
    if (a.lse && h == 0 && dw == 0)
        a.lse[orow * a.nh + head] = none ? (l == 0.0f ? -INFINITY : l) : (m - AC_OFF + __builtin_amdgcn_logf(l)) * 0.69314718056f;
    }
}

// The pieces of a tile that lies across ends of shares joined: ROWS rows a
// workgroup, four dims a thread, threads beyond the rows taking every other
// piece.  Bound: the latency of its loads, AHEAD pieces in flight a thread; 16 us
// for three documents cut 128 times a kv head, 2 to 3 where there is nothing to
// join.  512 threads: one token over 32K rows 31 us a call with 256, 27 with 512,
// no less with 1024.
constexpr int AC_JOIN = 512;
template <typename TQ, typename TC, int HD, int ROWS>
__global__ void __launch_bounds__(AC_JOIN) k_attn_chunk_join(AttnChunkArgs a, Parts parts)
{
    constexpr int PER_ROW = HD / 4, GROUPS = AC_JOIN / PER_ROW / ROWS, AHEAD = 4;
    static_assert(GROUPS >= 1, "threads for the rows");
    __shared__ styx_f4 s_o[AC_JOIN];
    __shared__ float2 s_ml[AC_JOIN];
    const KvView &kv = a.kv;
    const int w0 = blockIdx.z, kvh = blockIdx.y;
    const Across it = parts.across[w0 * kv.nkv + kvh];
    const int pieces = it.pieces, rows = min(it.s.count * a.gqa - it.row0, parts.rows);
    const int tid = threadIdx.x, d = tid % PER_ROW * 4, in = blockIdx.x * ROWS + tid / PER_ROW % ROWS, group = tid / PER_ROW / ROWS;
    if (pieces == 0 || (int)blockIdx.x * ROWS >= rows) return;
    const int r = it.row0 + in;
    const bool is = in < rows;
    float m = -INFINITY, l = 0.0f;
    styx_f4 o = {};
    for (int c0 = group; c0 < pieces; c0 += GROUPS * AHEAD) {
        float2 ml[AHEAD];
        styx_f4 po[AHEAD];
        float mn = m;
#pragma unroll
        for (int c = 0; c < AHEAD; c++) {
            const int cc = min(c0 + c * GROUPS, pieces - 1);
            const int64_t p = ((int64_t)(cc ? 2 * (w0 + cc) : it.part0) * kv.nkv + kvh) * parts.rows + (is ? in : 0);
            ml[c] = parts.ml[p];
            po[c] = *(const styx_f4 *)(parts.o + p * HD + d);
        }
#pragma unroll
        for (int c = 0; c < AHEAD; c++) {
            if (c0 + c * GROUPS >= pieces) {
                ml[c] = float2{-INFINITY, 0.0f};
                po[c] = styx_f4{};
            }
            mn = fmaxf(mn, ml[c].x);
        }
        const float f = m == -INFINITY ? 1.0f : exp2_(m - mn);
        l *= f;
        o *= f;
#pragma unroll
        for (int c = 0; c < AHEAD; c++) {
            // a piece without a slot that counts has sums of 0, or of NaN
            const float g = ml[c].x == -INFINITY ? 1.0f : exp2_(ml[c].x - mn);
            l += ml[c].y * g;
            o += po[c] * g;
        }
        m = mn;
    }
    if constexpr (GROUPS > 1) {
        s_o[tid] = o;
        s_ml[tid] = float2{m, l};
        __syncthreads();
        if (group) return;
        float mn = m;
#pragma unroll
        for (int c = 1; c < GROUPS; c++) mn = fmaxf(mn, s_ml[tid + c * ROWS * PER_ROW].x);
        const float f = m == -INFINITY ? 1.0f : exp2_(m - mn);
        l *= f;
        o *= f;
#pragma unroll
        for (int c = 1; c < GROUPS; c++) {
            const float2 y = s_ml[tid + c * ROWS * PER_ROW];
            const float g = y.x == -INFINITY ? 1.0f : exp2_(y.x - mn);
            l += y.y * g;
            o += s_o[tid + c * ROWS * PER_ROW] * g;
        }
        m = mn;
    }
    if (!is) return;
    const int tok = a.by_gqa.of(r), head = kvh * a.gqa + (r - tok * a.gqa);
    const int64_t row = it.s.first + tok;
    const bool none = m == -INFINITY;
    const float f = none ? 1.0f : 1.0f / l, add = none ? l : 0.0f;
    TQ *dst = (TQ *)a.out + row * a.ldo + (int64_t)head * HD + d;
    if constexpr (sizeof(TQ) == 2) {
        h4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (_Float16)(o[e] * f + add);
        *(h4 *)dst = v;
    } else {
        *(styx_f4 *)dst = o * f + add;
    }
    if (a.lse && d == 0) a.lse[row * a.nh + head] = none ? (l == 0.0f ? -INFINITY : l) : (m - AC_OFF + __builtin_amdgcn_logf(l)) * 0.69314718056f;
}

// ----------------------------------------------------------------- launch ---
struct ChunkShape {
    int64_t tiles;  // at most
    int shares;     // of a kv head, at most
    int rows;       // of a piece's partial results
    int64_t parts(int nkv) const { return 2 * (int64_t)shares * nkv * rows; }
    int64_t floats(int nkv, int hd) const { return parts(nkv) * (hd + 2) + (int64_t)shares * nkv * (int)(sizeof(Across) / 4); }
};
static ChunkShape shape_of(int bm, int per_cu, int n_seq, int nkv, int gqa, int n_rows)
{
    ChunkShape s{};
    // (a sequence has at least a row, and its last tile may be partly filled)
    s.tiles = (((int64_t)n_rows * gqa + bm - 1) / bm + std::min(n_seq, n_rows)) * nkv;
    s.shares = std::max(AC_CUS * per_cu / nkv, 1);
    s.rows = (int)std::min<int64_t>(bm, (int64_t)n_rows * gqa);
    return s;
}
// f(query type, row type, head_dim, groups of rows) for the kernel of a call with
// so many rows.  The fewer groups a tile has the more tiles there are, and the
// more often a slot is read.  What a sequence has is known to the device alone:
// the sequences' average counts, and a total that one sequence may have alone.
// (Places of the batch that hold no sequence, or one that asks for nothing, count
// among the sequences: in a large batch a single chunk of some hundred rows gets
// smaller tiles than it would alone.)
// One token for each of 24 over 2000 slots, heads of 128, 1 / 2 / 4 groups: 53 /
// 72 / 82 us; 16 tokens of one over 500 17 / 20 / 22, 64 of one over 2000 44 / 43 /
// 48, 128 of one 71 / 66 / 65; a prompt of 512 50 / 55 / 50, of 1024 124 / 119 /
// 111.  Heads of 64: 16 tokens of one over 2000 - / 19 / 22, 128 of one - / 45 / 43.
// Heads of 256: 64 of one 74 / 67 / 77, 128 of one 134 / 114 / 105, 32 for each of 16
// over 500 138 / 107 / 160.
template <typename F> static auto with_kernel(bool f16, bool q16, int hd, int n_seq, int64_t rows, F f)
{
    const auto four = std::integral_constant<int, 4>{};
    auto by_rows = [&](auto hd) {
        const int64_t each = rows <= 4096 ? n_seq : 0;
        if constexpr (hd() > 64)
            if (rows <= 128 || rows <= 32 * each) return f(float{}, float{}, hd, std::integral_constant<int, 1>{});
        if (rows <= 512 || rows <= (hd() == 256 ? 256 : 64) * each)
            return f(float{}, float{}, hd, std::integral_constant<int, 2>{});
        return f(float{}, float{}, hd, four);
    };
    auto by_type = [&](auto hd) {
        if (!f16) return by_rows(hd);
        return q16 ? f(_Float16{}, _Float16{}, hd, four) : f(float{}, _Float16{}, hd, four);
    };
    switch (hd) {
    case 64: return by_type(std::integral_constant<int, 64>{});
    case 128: return by_type(std::integral_constant<int, 128>{});
    default: return by_type(std::integral_constant<int, 256>{});
    }
}
// (times 8, so that rows times gqa stay below 2^28)
int64_t attn_chunk_grid(int n_seq, int nkv, int gqa, int n_rows)
{
    const ChunkShape s = shape_of(128, 2, n_seq, nkv, gqa, n_rows);
    return std::max<int64_t>(s.tiles, (int64_t)s.shares * nkv) * 8;
}
uint64_t attn_chunk_ws_bytes(int n_seq, int nkv, int hd, int gqa, int n_rows)
{
    // the types that the call may bring
    int64_t floats = 4;
    for (int t = 0; t < 3; t++)
        with_kernel(t > 0, t > 1, hd, n_seq, (int64_t)n_rows * gqa, [&](auto tq, auto tc, auto n, auto rg) {
            using W = Wave<decltype(tq), decltype(tc), n(), rg()>;
            static_assert((W::BM >= 128 || rg() < 4) && W::PER_CU <= 2, "attn_chunk_grid");
            floats = std::max(floats, shape_of(W::BM, W::PER_CU, n_seq, nkv, gqa, n_rows).floats(nkv, hd));
            return 0;
        });
    return 4ull * floats;
}

template <typename TQ, typename TC, int HD, int RG> static void launch_chunk(hipStream_t st, AttnChunkArgs a, void *ws)
{
    using W = Wave<TQ, TC, HD, RG>;
    const ChunkShape s = shape_of(W::BM, W::PER_CU, a.kv.n_seq, a.kv.nkv, a.gqa, a.chunk.n_rows);
    // (the tiles first: they want 16 bytes' alignment, and sums of few rows have it behind them)
    Across *across = (Across *)ws;
    float *o = (float *)(across + (int64_t)s.shares * a.kv.nkv);
    const Parts parts{o, (float2 *)(o + s.parts(a.kv.nkv) * HD), across, s.rows, s.shares};
    // rows of a wave in pages one after another, within 32 bits
    constexpr int PER_WAVE = W::KT / W::NW;
    a.runs = a.kv.page_tokens % PER_WAVE == 0 && (int64_t)a.kv.nkv * HD * (int)sizeof(TC) < (1 << 26);
    const int64_t grid = std::max<int64_t>(s.tiles, (int64_t)s.shares * a.kv.nkv);
    hipLaunchKernelGGL((k_attn_chunk<TQ, TC, HD, RG>), dim3((unsigned)grid), dim3(64 * W::NW), 0, st, a, parts);
    // (tiles of at most IDLE blocks are never cut: line_of)
    if (s.shares == 1 || a.kv.cap <= W::IDLE * W::KT) return;
    constexpr int MANY = AC_JOIN / (HD / 4), SOME = MANY > 4 ? 4 : MANY;
    if (s.rows > 64)
        hipLaunchKernelGGL((k_attn_chunk_join<TQ, TC, HD, MANY>), dim3((s.rows + MANY - 1) / MANY, a.kv.nkv, s.shares - 1), dim3(AC_JOIN),
                           0, st, a, parts);
    else
        hipLaunchKernelGGL((k_attn_chunk_join<TQ, TC, HD, SOME>), dim3((s.rows + SOME - 1) / SOME, a.kv.nkv, s.shares - 1), dim3(AC_JOIN),
                           0, st, a, parts);
}
hipError_t launch_attn_chunk(hipStream_t st, AttnChunkArgs a, void *ws)
{
    a.scale = (float)((double)a.scale * 1.4426950408889634);  // log2 e
    a.by_gqa = page_div((uint32_t)a.gqa);
    with_kernel(a.kv.f16, a.q_f16, a.kv.hd, a.kv.n_seq, (int64_t)a.chunk.n_rows * a.gqa, [&](auto tq, auto tc, auto hd, auto rg) {
        launch_chunk<decltype(tq), decltype(tc), hd(), rg()>(st, a, ws);
        return 0;
    });
    return hipGetLastError();
}

}  // namespace styx
