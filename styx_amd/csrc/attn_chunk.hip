// attn_chunk.hip -- causal attention of the new tokens of a batch over their
// sequences' slots of a paged KV cache.
//
// Token i of sequence b with n = len[b] rows, query head h of kv head j:
//   s_t = scale q . K[t], t <= n + i (and t > n + i - window), pages in the pool
//   M = max s_t, L = sum e^(s_t - M), out = sum e^(s_t - M) V[t] / L, lse = M + ln L
//
// A workgroup takes a tile of query rows -- a row is a token and one of a kv
// head's gqa heads, token by token -- and goes once over the slots that they see,
// in blocks that lie in LDS for its four waves, the next block under way
// meanwhile.  Scores are formed transposed, slots x queries: lane (n = lane & 31,
// h = lane >> 5) then has its own query's scores of slots 8 (i / 4) + 4 h + i % 4
// of each 32, the softmax factors are lane-local, and they are the operand of
// the value product as they stand.
#include <algorithm>
#include <type_traits>

#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int AC_WG = 256, AC_WAVES = AC_WG / 64;
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

// 16 bytes a lane from memory to LDS at off + 16 lane (off uniform), in the
// background: the caller waits (landed) before it reads them.  Not the builtin:
// behind that the compiler waits for all of them before any read of LDS.
__device__ __forceinline__ void to_lds(const void *from, uint32_t off)
{
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(off), "v"(from) : "memory");
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

template <typename TQ, typename TC, int HD> struct Wave;

// f16 caches: v_mfma_f32_32x32x16_f16.  f32 queries and their factors are two
// f16 pieces each, hi + lo with |x - hi - lo| <= 2^-22 |x|, queries brought to
// [2^9, 2^10) by a power of two per row so that the low pieces of all that
// counts are normal numbers.  f16 queries take factors rounded to f16: an
// error of at most 2^-11 of each, as large as the output's own rounding.
template <typename TQ, int HD> struct Wave<TQ, _Float16, HD> {
    using TC = _Float16;
    using La = Lay<TC, HD>;
    static constexpr int NP = sizeof(TQ) == 4 ? 2 : 1;  // pieces
    static constexpr int QT = 1, KT = 64, NK = HD / 16, ND = HD / 32;
    static constexpr int PER_CU = HD == 256 ? 1 : 2;
    h8 q[QT][NP][NK], p[QT][NP][KT / 16];
    f16v s[KT / 32][QT], o[QT][ND];
    float mul[QT];

    __device__ __forceinline__ void init(int qt, const TQ *row, float scale)
    {
        const int h = (threadIdx.x & 63) >> 5;
        // (a scale of 0 goes into q: -infinity times it would be NaN)
        const float a = scale == 0.0f ? 1.0f : fabsf(scale), sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
        if constexpr (NP == 1) {
            mul[qt] = a;
#pragma unroll
            for (int i = 0; i < NK; i++) {
                const h8 v = *(const h8 *)(row + 16 * i + 8 * h);
#pragma unroll
                for (int e = 0; e < 8; e++) q[qt][0][i][e] = v[e] * (_Float16)sign;
            }
        } else {
            styx_f4 v[NK][2];
            float m = 0.0f;
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
            mul[qt] = a / up;
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const float y = v[i][x >> 2][x & 3] * (up * sign);
                    const _Float16 hi = (_Float16)y;
                    q[qt][0][i][x] = hi;
                    q[qt][NP - 1][i][x] = (_Float16)(y - (float)hi);
                }
        }
    }
    __device__ __forceinline__ void scores(const char *kb)
    {
        const int lane = threadIdx.x & 63, m = lane & 31, h = lane >> 5;
        const f16v zero = {};
        const int at = m * La::ROW + ((h ^ La::perm(m)) << 4);
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int kt = 0; kt < KT / 32; kt++) {
                // (piece 2 i + h: its bits above 256 bytes are not permuted)
                const h8 k = *(const h8 *)(kb + (at ^ ((32 * i) & 255)) + ((32 * i) & ~255) + kt * 32 * La::ROW);
#pragma unroll
                for (int x = 0; x < NP; x++)
#pragma unroll
                    for (int qt = 0; qt < QT; qt++)
                        s[kt][qt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[qt][x][i], i + x == 0 ? zero : s[kt][qt], 0, 0, 0);
            }
    }
    // factors from s, which holds them unrounded
    __device__ __forceinline__ void factors(int qt)
    {
#pragma unroll
        for (int k = 0; k < KT / 16; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = s[k / 2][qt][8 * (k & 1) + i];
                const _Float16 hi = (_Float16)v;
                p[qt][0][k][i] = hi;
                if constexpr (NP == 2) p[qt][1][k][i] = (_Float16)(v - (float)hi);
            }
    }
    __device__ __forceinline__ void values(const char *vb)
    {
        const int lane = threadIdx.x & 63, h = lane >> 5, u = (lane >> 4) & 1, kk = (lane & 15) >> 2;
        // piece of dims 16 u + 4 (lane & 3) .. of the first 32, row kk + 4 (h + 2 r)
        auto at = [&](int r) {
            const int t = kk + 4 * h + 8 * r;
            return t * La::ROW + (((2 * u + ((lane & 3) >> 1)) ^ La::perm(t)) << 4) + 8 * (lane & 1);
        };
        const int at0 = at(0), at1 = at(1);
        typedef __attribute__((address_space(3))) s4 *lds4;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int k = 0; k < KT / 16; k++) {
                const int flip = (64 * d) & (La::ROW < 256 ? La::ROW - 1 : 255), far = ((64 * d) & ~255) + k * 16 * La::ROW;
                union {
                    s4 part[2];
                    h8 v;
                } x;
                x.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vb + (at0 ^ flip) + far));
                x.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vb + (at1 ^ flip) + far));
#pragma unroll
                for (int y = 0; y < NP; y++)
#pragma unroll
                    for (int qt = 0; qt < QT; qt++)
                        o[qt][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.v, p[qt][y][k], o[qt][d], 0, 0, 0);
            }
    }
};

// f32 caches: v_mfma_f32_32x32x2_f32, dims in fours on both sides of the score
// product for 16-byte reads.
template <int HD> struct Wave<float, float, HD> {
    using TC = float;
    using La = Lay<TC, HD>;
    static constexpr int QT = 1, KT = 32, NK = HD / 8, ND = HD / 32;
    static constexpr int PER_CU = HD == 256 ? 1 : 2;
    styx_f4 q[NK];
    f16v s[1][1], o[1][ND];
    float mul[1];

    __device__ __forceinline__ void init(int, const float *row, float scale)
    {
        const int h = (threadIdx.x & 63) >> 5;
        mul[0] = scale == 0.0f ? 1.0f : fabsf(scale);
        const float sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < NK; i++) q[i] = *(const styx_f4 *)(row + 8 * i + 4 * h) * sign;
    }
    __device__ __forceinline__ void scores(const char *kb)
    {
        const int lane = threadIdx.x & 63, m = lane & 31, h = lane >> 5;
        const f16v zero = {};
        const int at = m * La::ROW + ((h ^ La::perm(m)) << 4);
        f16v c[2];  // two chains: a product follows the one before on its sum at once otherwise
#pragma unroll
        for (int i = 0; i < NK; i++) {
            const styx_f4 k = *(const styx_f4 *)(kb + (at ^ ((32 * i) & 255)) + ((32 * i) & ~255));
#pragma unroll
            for (int e = 0; e < 4; e++)
                c[e & 1] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[i][e], i == 0 && e < 2 ? zero : c[e & 1], 0, 0, 0);
        }
        s[0][0] = c[0] + c[1];
    }
    __device__ __forceinline__ void factors(int) {}
    __device__ __forceinline__ void values(const char *vb)
    {
        const int lane = threadIdx.x & 63, m = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int t = 8 * (i >> 2) + 4 * h + (i & 3);
            const int at = t * La::ROW + (((m >> 2) ^ La::perm(t)) << 4) + 4 * (m & 3);
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const float v = *(const float *)(vb + (at ^ ((128 * d) & 255)) + ((128 * d) & ~255));
                o[0][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[0][0][i], o[0][d], 0, 0, 0);
            }
        }
    }
};

// ------------------------------------------------------------- the split ---
// Tiles of query rows in the order sequence, last tokens first; the slots of a
// tile are cut into pieces of `share` blocks where the tiles alone are fewer
// than the workgroups that run at once.
struct Cut {
    int share;      // blocks of a piece; 0: tiles are not cut
    int64_t items;  // of all sequences, kv heads aside
};
struct SeqWork {
    int tiles, pieces;
};
constexpr int AC_SLOTS_CU = 256;  // CUs
constexpr int AC_LEAST = 4;       // blocks of a piece at least

template <int BM, int KT> __device__ __forceinline__ SeqWork seq_work(const AttnChunkArgs &a, const ChunkSeq &s, int share)
{
    if (s.count == 0) return {0, 0};
    const int64_t rows = (int64_t)s.count * a.gqa;
    const int tiles = (int)((rows + BM - 1) / BM);
    int blocks = (s.len + s.count + KT - 1) / KT;
    if (a.window) blocks = min(blocks, (int)min((int64_t)1 << 30, ((int64_t)a.window + BM / a.gqa + 1) / KT + 2));
    return {tiles, share ? (blocks + share - 1) / share : blocks};
}

template <int BM, int KT> __device__ __forceinline__ Cut cut_chunk(const AttnChunkArgs &a, int slots)
{
    const int lane = threadIdx.x & 63;
    int64_t tiles = 0, work = 0;
    for (int b0 = 0; b0 < a.kv.n_seq; b0 += 64) {
        const SeqWork w = seq_work<BM, KT>(a, chunk_seq(a.chunk, a.kv, b0 + lane), 0);
        tiles += w.tiles;
        work += (int64_t)w.tiles * w.pieces;
    }
    tiles = wave_total(tiles) * a.kv.nkv;
    work = wave_total(work) * a.kv.nkv;
    if (4 * tiles > 3 * slots) return {0, tiles};
    const int64_t room = slots - tiles;
    return {(int)min((int64_t)1 << 30, max((int64_t)AC_LEAST, (work + room - 1) / room)), tiles};
}

// Item `item` of the batch (kv heads aside): sequence, tile, piece; b < 0: past
// the last.
struct Item {
    int b, tile, tiles, piece, pieces;
    int64_t first;  // pieces of the batch before this tile's
    ChunkSeq s;
};
template <int BM, int KT> __device__ __forceinline__ Item find_item(const AttnChunkArgs &a, int share, int64_t item)
{
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.kv.n_seq; b0 += 64) {
        const ChunkSeq s = chunk_seq(a.chunk, a.kv, b0 + lane);
        SeqWork w = seq_work<BM, KT>(a, s, share);
        if (!share) w.pieces = 1;
        const int64_t mine = (int64_t)w.tiles * w.pieces, upto = base + wave_upto(mine);
        if (const unsigned long long hit = __ballot(upto > item)) {
            const int l = __builtin_ctzll(hit);
            const int tiles = __builtin_amdgcn_readlane(w.tiles, l), pieces = __builtin_amdgcn_readlane(w.pieces, l);
            const int64_t before = of_lane(upto, l) - of_lane(mine, l);
            const int in = (int)(item - before), tile = in / pieces;
            return {b0 + l, tiles - 1 - tile, tiles, in - tile * pieces, pieces, before + (int64_t)tile * pieces,
                    {(int)__builtin_amdgcn_readlane(s.first, l), (int)__builtin_amdgcn_readlane(s.count, l),
                     (int)__builtin_amdgcn_readlane(s.len, l)}};
        }
        base = of_lane(upto, 63);
    }
    return {-1, 0, 0, 0, 0, 0, {0, 0, 0}};
}

// -------------------------------------------------------------- a piece ----
template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(AC_WG, (Wave<TQ, TC, HD>::PER_CU)) k_attn_chunk(AttnChunkArgs a, float *part_ml, float *part_o, int part_rows)
{
    using W = Wave<TQ, TC, HD>;
    using La = Lay<TC, HD>;
    constexpr int QT = W::QT, KT = W::KT, BM = 32 * QT * AC_WAVES, ND = W::ND;
    constexpr int BLOCK = KT * La::ROW, PER_WAVE = KT / AC_WAVES, NI = PER_WAVE / La::RPI;
    __shared__ __align__(1024) char s_k[2][BLOCK];
    __shared__ __align__(1024) char s_v[2][BLOCK];
    const KvView &kv = a.kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const Cut sp = cut_chunk<BM, KT>(a, AC_SLOTS_CU * W::PER_CU);
    const int kvh = blockIdx.x % kv.nkv;
    const Item it = find_item<BM, KT>(a, sp.share, blockIdx.x / kv.nkv);
    if (it.b < 0) return;
    const ChunkSeq &s = it.s;
    const int64_t rows = (int64_t)s.count * a.gqa, row0 = (int64_t)it.tile * BM;
    // tokens of the tile, the slots that any of them sees, the piece's blocks
    const int tok0 = (int)(row0 / a.gqa), tok1 = (int)(min(row0 + BM, rows) - 1) / a.gqa;
    const int t1 = s.len + tok1 + 1, t0 = a.window && s.len + tok0 >= a.window ? s.len + tok0 - a.window + 1 : 0;
    int b0 = t0 / KT, b1 = (t1 + KT - 1) / KT;
    if (sp.share) {
        b0 += min((int64_t)it.piece * sp.share, (int64_t)(b1 - b0));
        b1 = (int)min((int64_t)b1, (int64_t)b0 + sp.share);
    }
    const int32_t *tab = kv.table + (int64_t)it.b * kv.table_len;
    const int64_t stride = (int64_t)kv.nkv * La::ROW;
    const char *kp = (const char *)kv.kpool + kvh * La::ROW, *vp = (const char *)kv.vpool + kvh * La::ROW;

    // this lane's queries
    W x;
    int at[QT];                // last slot seen, -1: no such row
    int64_t orow[QT];          // row of q and out
    int head[QT];
    float m[QT], l[QT];
    uint32_t nan_at[QT][HD / 64];  // dims that are NaN whatever the sums are
    const int wrow0 = 32 * QT * wave;
    const bool works = row0 + wrow0 < rows;
#pragma unroll
    for (int qt = 0; qt < QT; qt++) {
        const int64_t r = row0 + wrow0 + 32 * qt + n, rr = min(r, rows - 1);
        const int tok = (int)(rr / a.gqa);
        head[qt] = kvh * a.gqa + (int)(rr - (int64_t)tok * a.gqa);
        orow[qt] = s.first + tok;
        at[qt] = r < rows ? s.len + tok : -1;
        m[qt] = -INFINITY;
        l[qt] = 0.0f;
#pragma unroll
        for (int w = 0; w < HD / 64; w++) nan_at[qt][w] = 0;
        x.init(qt, (const TQ *)a.q + orow[qt] * a.ldq + (int64_t)head[qt] * HD, a.scale);
#pragma unroll
        for (int d = 0; d < ND; d++) x.o[qt][d] = f16v{};
    }
    // slots that all of the wave's queries see, and those that none sees
    const int wtok0 = (int)(min(row0 + wrow0, rows - 1) / a.gqa), wtok1 = (int)(min(row0 + wrow0 + 32 * QT, rows) - 1) / a.gqa;
    const int all_hi = s.len + wtok0, any_hi = s.len + wtok1;
    const int all_lo = a.window ? s.len + wtok1 - a.window + 1 : 0, any_lo = a.window ? s.len + wtok0 - a.window + 1 : 0;

    // rows of the pools: a lane's slot of a block (KT = 32: both halves alike)
    const int my = lane & (KT - 1);
    auto entry_of = [&](int blk) { return kv.entry(tab, min(blk * KT + my, t1 - 1)); };
    auto row_of = [&](int e, int blk) { return blk * KT + my < t1 ? kv.row_of(e, min(blk * KT + my, t1 - 1)) : -1; };
    const uint32_t lk = lds_at(&s_k[0][0]), lv = lds_at(&s_v[0][0]);
    auto fetch = [&](int buf, int row) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int t = wave * PER_WAVE + i * La::RPI + lane / La::LPR;
            const int64_t r = max(__shfl(row, t), 0);
            const int c = (lane & (La::LPR - 1)) ^ La::perm(t);
            const int to = (wave * PER_WAVE + i * La::RPI) * La::ROW;
            to_lds(kp + r * stride + 16 * c, __builtin_amdgcn_readfirstlane(lk + buf * BLOCK + to));
            to_lds(vp + r * stride + 16 * c, __builtin_amdgcn_readfirstlane(lv + buf * BLOCK + to));
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
        // (uniform over the workgroup: whether every query of the tile sees the block)
        const bool plain = seen == full && tb + KT - 1 <= s.len + tok0 && (!a.window || tb > s.len + tok1 - a.window);
        // the slots of the block that each query sees
        uint32_t vis[QT][KT / 32];
        if (!plain) {
#pragma unroll
            for (int kt = 0; kt < KT / 32; kt++)
#pragma unroll
                for (int qt = 0; qt < QT; qt++) {
                    const int last = at[qt] - (tb + 32 * kt), before = a.window ? last - a.window : -1;
                    uint32_t v = (uint32_t)(seen >> (32 * kt));
                    v &= last < 0 ? 0u : last > 30 ? ~0u : (2u << last) - 1u;
                    v &= before < 0 ? ~0u : before > 30 ? 0u : ~0u << (before + 1);
                    vis[qt][kt] = v;
                }
            // A value that is not finite must not reach those that do not see
            // it, whose factor is 0: where there is one, the dims of those that
            // do see it are noted to be NaN, and the value becomes 0.
            char *mine = s_v[buf] + threadIdx.x * (BLOCK / AC_WG);
            bool odd = false;
#pragma unroll
            for (int i = 0; i < BLOCK / AC_WG; i += 16) {
                const styx_u4 v = *(const styx_u4 *)(mine + i);
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= not_finite<TC>(v[e]) != 0;
            }
            if (__syncthreads_or(odd)) {
#pragma unroll 1
                for (int t = 0; t < KT; t++) {
                    uint32_t see[QT];
#pragma unroll
                    for (int qt = 0; qt < QT; qt++) see[qt] = 0u - (vis[qt][KT == 64 ? t >> 5 : 0] >> (t & 31) & 1);
                    // bits 4 j + e: dims 8 j + 4 h + e
#pragma unroll 1
                    for (int j = 0; j < HD / 8; j++) {
                        const TC *v = (const TC *)(vb + La::at(t, 8 * j + 4 * h));
                        uint32_t bad = 0;
#pragma unroll
                        for (int e = 0; e < 4; e++) bad |= (uint32_t) !(fabsf((float)v[e]) < INFINITY) << e;
                        if (bad)
#pragma unroll
                            for (int w = 0; w < HD / 64; w++)
#pragma unroll
                                for (int qt = 0; qt < QT; qt++)
                                    nan_at[qt][w] |= w == j >> 3 ? (bad & see[qt]) << (4 * (j & 7)) : 0;
                    }
                }
                __syncthreads();
                for (int i = 0; i < BLOCK / AC_WG; i += 4) {
                    uint32_t *v = (uint32_t *)(mine + i);
                    *v &= ~not_finite<TC>(*v);
                }
                __syncthreads();
            }
        }
        if (!works || tb > any_hi || tb + KT <= any_lo) continue;
        x.scores(kb);
        if (seen != full || tb + KT - 1 > all_hi || tb < all_lo) {
#pragma unroll
            for (int kt = 0; kt < KT / 32; kt++)
#pragma unroll
                for (int qt = 0; qt < QT; qt++) {
                    const uint32_t mine = vis[qt][kt] >> (4 * h);
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (!(mine >> (8 * (i >> 2) + (i & 3)) & 1)) x.s[kt][qt][i] = -INFINITY;
                }
        }
#pragma unroll
        for (int qt = 0; qt < QT; qt++) {
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT / 32; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++) mx = fmaxf(mx, x.s[kt][qt][i]);
            mx = fmaxf(mx, other_half(mx)) * x.mul[qt];
            if (__ballot(mx > m[qt] + AC_LAG)) {
                const float mn = fmaxf(m[qt], mx), corr = mn == -INFINITY ? 1.0f : exp2_(m[qt] - mn);
                m[qt] = mn;
                l[qt] *= corr;
#pragma unroll
                for (int d = 0; d < ND; d++) x.o[qt][d] *= corr;
            }
            const float ref = (m[qt] == -INFINITY ? 0.0f : m[qt]) - AC_OFF;
            float sum[4] = {};
#pragma unroll
            for (int kt = 0; kt < KT / 32; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float v = exp2_(fmaf(x.s[kt][qt][i], x.mul[qt], -ref));
                    x.s[kt][qt][i] = v;
                    sum[i & 3] += v;
                }
            l[qt] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            x.factors(qt);
        }
        x.values(vb);
    }
    if (!works) return;
#pragma unroll
    for (int qt = 0; qt < QT; qt++) {
        if (at[qt] < 0) continue;
        l[qt] += other_half(l[qt]);
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (nan_at[qt][d / 2] >> (16 * (d & 1) + i) & 1) x.o[qt][d][i] = NAN;
        if (sp.share) {
            // a partial result: M, L and the sums
            const int64_t p = ((it.first + it.piece) * kv.nkv + kvh) * part_rows + wrow0 + 32 * qt + n;
            if (h == 0) {
                part_ml[2 * p] = m[qt];
                part_ml[2 * p + 1] = l[qt];
            }
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(styx_f4 *)(part_o + p * HD + 32 * d + 2 * i + 4 * h) =
                        styx_f4{x.o[qt][d][i], x.o[qt][d][i + 1], x.o[qt][d][i + 2], x.o[qt][d][i + 3]};
            continue;
        }
        // no slot with a weight (m = -inf): 0, or NaN
        const bool none = m[qt] == -INFINITY;
        const float r = none ? 1.0f : 1.0f / l[qt], add = none ? l[qt] : 0.0f;
        TQ *out = (TQ *)a.out + orow[qt] * a.ldo + (int64_t)head[qt] * HD;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                TQ *dst = out + 32 * d + 2 * i + 4 * h;
                if constexpr (sizeof(TQ) == 2) {
                    h4 v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = (_Float16)(x.o[qt][d][i + e] * r + add);
                    *(h4 *)dst = v;
                } else {
                    styx_f4 v;
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = x.o[qt][d][i + e] * r + add;
                    *(styx_f4 *)dst = v;
                }
            }
        if (a.lse && h == 0)
            a.lse[orow[qt] * a.nh + head[qt]] =
                none ? (l[qt] == 0.0f ? -INFINITY : l[qt]) : (m[qt] - AC_OFF + __builtin_amdgcn_logf(l[qt])) * 0.69314718056f;
    }
}

// The pieces of a tile joined: a workgroup for 16 of its rows, where the split
// cut tiles at all; a wave goes through 4 rows, its lanes through the dims.
template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(AC_WG) k_attn_chunk_join(AttnChunkArgs a, const float *part_ml, const float *part_o, int part_rows)
{
    using W = Wave<TQ, TC, HD>;
    constexpr int KT = W::KT, BM = 32 * W::QT * AC_WAVES, DPL = HD / 64, PARTS = BM / 16, AHEAD = 4;
    const KvView &kv = a.kv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Cut sp = cut_chunk<BM, KT>(a, AC_SLOTS_CU * W::PER_CU);
    if (!sp.share) return;
    const int kvh = blockIdx.x / PARTS % kv.nkv, part = blockIdx.x % PARTS;
    const int64_t nth = blockIdx.x / PARTS / kv.nkv;  // tile of the batch
    if (nth * kv.nkv >= sp.items) return;
    // the tile: found among tiles of one piece, then counted in pieces
    Item it = find_item<BM, KT>(a, 0, nth);
    if (it.b < 0) return;
    const SeqWork w = seq_work<BM, KT>(a, it.s, sp.share);
    int64_t before = 0;
    for (int b0 = 0; b0 <= it.b; b0 += 64) {
        const SeqWork y = seq_work<BM, KT>(a, chunk_seq(a.chunk, kv, b0 + lane), sp.share);
        before += wave_total(b0 + lane < it.b ? (int64_t)y.tiles * y.pieces : (int64_t)0);
    }
    const int64_t first = before + (int64_t)(w.tiles - 1 - it.tile) * w.pieces;
    const int64_t rows = (int64_t)it.s.count * a.gqa;
    for (int i = 0; i < 4; i++) {
        const int in = 16 * part + 4 * wave + i;
        const int64_t r = (int64_t)it.tile * BM + in;
        if (r >= rows) return;
        float m = -INFINITY, l = 0.0f, o[DPL] = {};
        for (int c0 = 0; c0 < w.pieces; c0 += AHEAD) {
            float pm[AHEAD], pl[AHEAD], po[AHEAD][DPL], mn = m;
#pragma unroll
            for (int c = 0; c < AHEAD; c++) {
                const int64_t p = ((first + min(c0 + c, w.pieces - 1)) * kv.nkv + kvh) * part_rows + in;
                pm[c] = part_ml[2 * p];
                pl[c] = part_ml[2 * p + 1];
#pragma unroll
                for (int d = 0; d < DPL; d++) po[c][d] = part_o[p * HD + lane + 64 * d];
            }
#pragma unroll
            for (int c = 0; c < AHEAD; c++) {
                if (c0 + c >= w.pieces) pm[c] = -INFINITY, pl[c] = 0.0f;
                mn = fmaxf(mn, pm[c]);
            }
            const float f = m == -INFINITY ? 0.0f : exp2_(m - mn);
            l *= f;
#pragma unroll
            for (int d = 0; d < DPL; d++) o[d] *= f;
#pragma unroll
            for (int c = 0; c < AHEAD; c++) {
                // a piece without a slot that counts has sums of 0, or of NaN
                const float g = pm[c] == -INFINITY ? (pl[c] == 0.0f ? 0.0f : 1.0f) : exp2_(pm[c] - mn);
                l += pl[c] * g;
                if (c0 + c < w.pieces) {
#pragma unroll
                    for (int d = 0; d < DPL; d++) o[d] += po[c][d] * g;
                }
            }
            m = mn;
        }
        const int tok = (int)(r / a.gqa), head = kvh * a.gqa + (int)(r - (int64_t)tok * a.gqa);
        const int64_t row = it.s.first + tok;
        const bool none = m == -INFINITY;
#pragma unroll
        for (int d = 0; d < DPL; d++)
            ((TQ *)a.out)[row * a.ldo + (int64_t)head * HD + lane + 64 * d] = (TQ)(none ? o[d] + l : o[d] / l);
        if (a.lse && lane == 0)
            a.lse[row * a.nh + head] =
                none ? (l == 0.0f ? -INFINITY : l) : (m - AC_OFF + __builtin_amdgcn_logf(l)) * 0.69314718056f;
    }
}

// ----------------------------------------------------------------- launch ---
struct ChunkShape {
    int bm, slots;
    int64_t tiles, items;  // at most
};
static ChunkShape shape_of(int bm, int per_cu, int n_seq, int nkv, int gqa, int n_rows)
{
    ChunkShape s{bm, AC_SLOTS_CU * per_cu, 0, 0};
    // (a sequence has at least a row, and its last tile may be partly filled)
    const int64_t seqs = std::min(n_seq, n_rows);
    s.tiles = (((int64_t)n_rows * gqa + bm - 1) / bm + seqs) * nkv;
    // tiles that are cut are at most 3/4 of the slots, and make at most `slots` pieces
    s.items = std::max(s.tiles, (int64_t)s.slots);
    return s;
}
template <typename F> static auto with_kernel(bool f16, bool q16, int hd, F f)
{
    auto by_hd = [&](auto tq, auto tc) {
        switch (hd) {
        case 64: return f(tq, tc, std::integral_constant<int, 64>{});
        case 128: return f(tq, tc, std::integral_constant<int, 128>{});
        default: return f(tq, tc, std::integral_constant<int, 256>{});
        }
    };
    if (!f16) return by_hd(float{}, float{});
    return q16 ? by_hd(_Float16{}, _Float16{}) : by_hd(float{}, _Float16{});
}
int64_t attn_chunk_grid(int n_seq, int nkv, int gqa, int n_rows)
{
    return shape_of(128, 2, n_seq, nkv, gqa, n_rows).items;
}
// Rows of a piece's partial results, and floats of all pieces'.
static int part_rows(const ChunkShape &s, int gqa, int n_rows) { return (int)std::min<int64_t>(s.bm, (int64_t)n_rows * gqa); }
static int64_t part_floats(const ChunkShape &s, int gqa, int n_rows, int hd)
{
    return (int64_t)s.slots * part_rows(s, gqa, n_rows) * (hd + 2);
}
uint64_t attn_chunk_ws_bytes(int n_seq, int nkv, int hd, int gqa, int n_rows)
{
    // the types that the call may bring
    int64_t floats = 4;
    for (int t = 0; t < 3; t++)
        with_kernel(t > 0, t > 1, hd, [&](auto tq, auto tc, auto n) {
            using W = Wave<decltype(tq), decltype(tc), decltype(n)::value>;
            const ChunkShape s = shape_of(32 * W::QT * AC_WAVES, W::PER_CU, n_seq, nkv, gqa, n_rows);
            floats = std::max(floats, part_floats(s, gqa, n_rows, hd));
            return 0;
        });
    return 4ull * floats;
}

hipError_t launch_attn_chunk(hipStream_t st, AttnChunkArgs a, void *ws)
{
    a.scale = (float)((double)a.scale * 1.4426950408889634);  // log2 e
    with_kernel(a.kv.f16, a.q_f16, a.kv.hd, [&](auto tq, auto tc, auto hd) {
        using TQ = decltype(tq);
        using TC = decltype(tc);
        constexpr int HD = decltype(hd)::value;
        using W = Wave<TQ, TC, HD>;
        const ChunkShape s = shape_of(32 * W::QT * AC_WAVES, W::PER_CU, a.kv.n_seq, a.kv.nkv, a.gqa, a.chunk.n_rows);
        const int pr = part_rows(s, a.gqa, a.chunk.n_rows);
        float *o = (float *)ws, *ml = o + (int64_t)s.slots * pr * HD;
        hipLaunchKernelGGL((k_attn_chunk<TQ, TC, HD>), dim3((unsigned)s.items), dim3(AC_WG), 0, st, a, ml, o, pr);
        const int64_t joins = std::min(s.tiles, (int64_t)s.slots) * (s.bm / 16);
        hipLaunchKernelGGL((k_attn_chunk_join<TQ, TC, HD>), dim3((unsigned)joins), dim3(AC_WG), 0, st, a, ml, o, pr);
        return 0;
    });
    return hipGetLastError();
}

}  // namespace styx
