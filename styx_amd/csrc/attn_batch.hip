// attn_batch.hip -- decode attention of one new token for each sequence of a
// batch over one paged KV cache of f32 or f16 rows, which also adds every
// row's attention weight to an accumulator (what kv_evict.hip goes by).
//
// Per sequence b with n = len[b] rows, new token at position p = pos[b], and
// query head h of kv head j = h / gqa:
//   q^ = rope_p(rmsnorm(q)), k^ = rope_p(rmsnorm(k)), rows K[n] = k^, V[n] = v
//   s_t = scale q^ . K[t], M = max_t s_t, L = sum_t e^(s_t - M), t = 0 .. n
//   out = sum_t e^(s_t - M) V[t] / L
//   acc_out[j][t] = decay acc_in[j][t] + sum_{h of j} e^(s_t - M_h) / L_h
//
// Bound: HBM.  A row of a kv head is read once for its gqa query heads, 2 to
// 16 flop per byte in f32 and twice that in f16, far below what the matrix
// cores give.  All products are on the matrix cores all the same, 16 query
// rows at a time (fewer heads are padded): they take the per-row reductions
// away, which would cost the VALU more than the products.
//
// Split: the rows of all sequences and kv heads, in units of 64, lie one
// after another and every workgroup takes the same number of them, as many
// workgroups as run at once: a ragged batch keeps the whole chip busy to the
// end, where a split by sequence waits for the longest, or for the rounds of
// a grid that does not fit.  A workgroup's share may end one (sequence, head)
// and go on with the next; each such piece is a partial result (M, L, o).
// A second launch merges the pieces and turns the stored scores into
// weights: these need M and L of the whole context, and the scores (4 gqa
// bytes per row) are cheaper to keep than K is to read again (up to 1024).
// (A tile's scores stored together instead of head by head measured the same
// in the first launch and 1 to 4 us slower in the second.)
//
// Measured, both launches: one context of 32767 f32 rows, 16 query heads for
// each of 4 kv heads, 34 + 6 us (135 MB, 3.4 TB/s); six of up to 20011 f32
// rows, head_dim 256, without weights 62 + 5 us (302 MB, 4.5 TB/s); 24
// conversations of up to 4096 f16 rows 29 + 6.5 us (102 MB, 2.9 TB/s); 40 of
// up to 8192, head_dim 64, 76 + 8 us (327 MB, 3.9 TB/s); one of 37 rows 8 +
// 3.5 us, the chain lengths, page table, rows, and the second launch.
#include <algorithm>
#include <type_traits>

#include "attn16.h"
#include "attn_batch.h"
#include "lanes.h"

namespace styx {

constexpr int AB_WG = 256, AB_WAVES = AB_WG / 64;
// Workgroups of a 256-CU chip that run at once: three, two and one of four
// waves per CU, as k_attn_batch's registers (at most 168, 256 and 512 per
// lane by its launch bounds) allow.
__host__ __device__ constexpr int ab_slots(int hd) { return hd == 64 ? 768 : hd == 128 ? 512 : 256; }
// Rows of a unit: a 16-row tile (f32), or half of a 32-row one, per wave.
constexpr int AB_UNIT = 64;
// Slots of a thread in a step of the joining launch's weights: with its query
// heads (4, 8 or 16 per kv head) 32 scores in flight.
__host__ __device__ constexpr int ab_wper(int gqa) { return gqa <= 4 ? 8 : gqa <= 8 ? 4 : 2; }
// Pieces whose partials a thread of the joining launch has in flight.
constexpr int AB_BATCH = 8;

// Scores are in units of ln 2 (the caller's scale times log2 e, one rounding):
// v_exp_f32 is then the exponential, good to a unit in the last place.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// What a part (M, L, o) of a softmax is multiplied by where the maximum of all
// parts is `all`.  No part is left out of a sum for a factor of 0, or for a
// maximum of -infinity: that is where nothing was seen (L and o are 0), but
// also where every score was NaN (a maximum takes no NaN; L is one then), and
// a value that is not finite has to be so in the sum.
__device__ __forceinline__ float part_factor(float m, float all) { return m == -INFINITY ? 0.0f : exp2_(m - all); }

typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Rows that the new token of sequence b sees, itself among them; 0: skipped.
__device__ __forceinline__ int rows_of(const AttnBatchArgs &a, int b)
{
    if (b >= a.kv.n_seq) return 0;
    const int n = a.len[b], p = a.pos[b];
    return n >= 0 && n < a.kv.cap && p >= 0 && p < a.n_rope ? n + 1 : 0;
}

// The batch's split.  Unit u of the batch belongs to workgroup u / share.
// A share that ends one head and begins another costs its workgroup a second
// start and end, about 10 us on a busy chip; where a slightly larger share
// does without, every head is padded to whole shares (24 ragged f16
// conversations, 8 units instead of 7: 25 us against 36; six f32 documents,
// 10 instead of 9: 62 against 68).  It does not pay where the heads are too
// many for the workgroups (40 sequences of 8 heads, 45 units instead of 27:
// 105 us against 81).  AB_MORE: units of a share that cost about as much as
// a second start, from these three batches (no others were measured).
// `mine`, `upto`: rows of sequence `lane` and units of the sequences up to it.
constexpr int AB_MORE_F16 = 3, AB_MORE_F32 = 1;
struct RowSplit {
    uint32_t units, share, upto;
    int mine, padded;
};
__device__ __forceinline__ uint32_t head_units(const RowSplit &sp, int rows)
{
    const uint32_t u = (uint32_t)(rows + AB_UNIT - 1) / AB_UNIT;
    return sp.padded ? (u + sp.share - 1) / sp.share * sp.share : u;
}
__device__ __forceinline__ RowSplit split_rows(const AttnBatchArgs &a)
{
    const int lane = threadIdx.x & 63;
    const uint32_t nkv = a.kv.nkv, slots = ab_slots(a.kv.hd);
    RowSplit sp;
    sp.padded = 0;
    sp.mine = rows_of(a, lane);
    if (a.kv.n_seq == 1) {
        sp.mine = __builtin_amdgcn_readfirstlane(sp.mine);
        const uint32_t u = (uint32_t)(sp.mine + AB_UNIT - 1) / AB_UNIT;
        // whole shares for every head, if there are workgroups for the heads
        sp.padded = nkv <= slots;
        sp.share = sp.padded ? (u + slots / nkv - 1) / (slots / nkv) : (u * nkv + slots - 1) / slots;
        sp.share += sp.share == 0;
        sp.units = sp.upto = head_units(sp, sp.mine) * nkv;
        return sp;
    }
    const uint32_t u = head_units(sp, sp.mine);
    uint32_t all = u, seqs = sp.mine > 0;
    for (int b = lane + 64; b < a.kv.n_seq; b += 64) {
        const int r = rows_of(a, b);
        all += head_units(sp, r);
        seqs += r > 0;
    }
    all = wave_total(all) * nkv;
    const uint32_t heads = wave_total(seqs) * nkv, least = (all + slots - 1) / slots;
    sp.share = least + (least == 0);
    if (heads < slots) {
        // at most all / share and one for every head
        const uint32_t most = (all + slots - heads - 1) / (slots - heads);
        const uint32_t worth = least + (a.kv.f16 ? AB_MORE_F16 : AB_MORE_F32);
        uint32_t at = max(most, 1u);  // (1: no rows at all)
        // (looked for only as far as it is worth taking: with nearly as many
        // heads as slots `most` is hundreds of steps away, each a division and
        // a sum over the wave; 59 sequences of 13 heads, one of 64K rows and
        // the others of one, took 328 us so, and 95 now)
        if (a.kv.n_seq <= 64)
            for (at = sp.share; at < most && at <= worth && wave_total((u + at - 1) / at) * nkv > slots; at++)
                ;
        if (at <= worth) {
            sp.padded = 1;
            sp.share = at;
        }
    }
    sp.upto = wave_upto(head_units(sp, sp.mine) * nkv);
    sp.units = __builtin_amdgcn_readlane(sp.upto, 63);
    if (a.kv.n_seq > 64) {
        uint32_t more = 0;
        for (int b = lane + 64; b < a.kv.n_seq; b += 64) more += head_units(sp, rows_of(a, b)) * nkv;
        sp.units += wave_total(more);
    }
    return sp;
}

// A sequence, its rows, and the unit at which its first kv head begins.
struct SeqAt {
    int b, rows;
    uint32_t first;
};
// The sequence of unit u.
__device__ __forceinline__ SeqAt seq_find(const AttnBatchArgs &a, const RowSplit &sp, uint32_t u)
{
    if (a.kv.n_seq == 1) return {0, sp.mine, 0};
    const int lane = threadIdx.x & 63;
    uint32_t base = 0;
    for (int b0 = 0;; b0 += 64) {
        const int rows = b0 ? rows_of(a, b0 + lane) : sp.mine;
        const uint32_t upto = b0 ? base + wave_upto(head_units(sp, rows) * a.kv.nkv) : sp.upto;
        if (const unsigned long long hit = __ballot(upto > u)) {
            const int l = __builtin_ctzll(hit), r = __builtin_amdgcn_readlane(rows, l);
            return {b0 + l, r, __builtin_amdgcn_readlane(upto, l) - head_units(sp, r) * a.kv.nkv};
        }
        base = __builtin_amdgcn_readlane(upto, 63);
    }
}

// The split for the joining launch, by one wave: a.plan = {share, padded,
// first unit of every sequence}.
__device__ __forceinline__ void split_store(const AttnBatchArgs &a, const RowSplit &sp)
{
    const int lane = threadIdx.x & 63;
    if (lane == 0) {
        a.plan[0] = sp.share;
        a.plan[1] = sp.padded;
    }
    if (a.kv.n_seq == 1) {
        if (lane == 0) a.plan[2] = 0;
        return;
    }
    uint32_t base = 0;
    for (int b0 = 0; b0 < a.kv.n_seq; b0 += 64) {
        const int rows = b0 ? rows_of(a, b0 + lane) : sp.mine;
        const uint32_t mine = head_units(sp, rows) * a.kv.nkv;
        const uint32_t upto = b0 ? base + wave_upto(mine) : sp.upto;
        if (b0 + lane < a.kv.n_seq) a.plan[2 + b0 + lane] = upto - mine;
        base = __builtin_amdgcn_readlane(upto, 63);
    }
}
__device__ __forceinline__ SeqAt seq_load(const AttnBatchArgs &a, RowSplit &sp, int b)
{
    sp.share = a.plan[0];
    sp.padded = (int)a.plan[1];
    return {b, rows_of(a, b), a.plan[2 + b]};
}

// One head's RMSNorm and rotation by a wave, in f64 to the end, so that the
// cache's rounding of k does not depend on how a sum was ordered.  In two
// phases, so that all of a wave's heads are in flight at once.  Lane l has
// the rope pairs (i, i + HD/2), i = l + 64 j.
template <int HD> struct HeadRow {
    static constexpr int HALF = HD / 2, PPL = (HALF + 63) / 64;
    float x0[PPL], x1[PPL];
    __device__ __forceinline__ void load(const float *x, int lane)
    {
#pragma unroll
        for (int j = 0; j < PPL; j++) {
            const int i = HALF < 64 ? min(lane, HALF - 1) : lane + 64 * j;
            x0[j] = x[i];
            x1[j] = x[i + HALF];
        }
    }
    // emit(dim, value) once per dimension
    template <typename Emit>
    __device__ __forceinline__ void turn(const HeadRow &w, bool norm, const double2 *cs, float eps, int lane, Emit emit) const
    {
        double f = 1.0;
        if (norm) {
            double ss = 0.0;
#pragma unroll
            for (int j = 0; j < PPL; j++)
                if (HALF >= 64 || lane < HALF) ss += (double)x0[j] * x0[j] + (double)x1[j] * x1[j];
            f = 1.0 / sqrt(wave_total(ss) * (1.0 / HD) + (double)eps);
        }
#pragma unroll
        for (int j = 0; j < PPL; j++) {
            if (HALF < 64 && lane >= HALF) continue;
            const int i = lane + 64 * j;
            const double a = norm ? x0[j] * f * w.x0[j] : x0[j], b = norm ? x1[j] * f * w.x1[j] : x1[j];
            // (kept apart from a conversion to f16 that may follow: contracted
            // with it, the f64 value would be rounded to f16 directly, which
            // differs for one value of some 15000 and takes a dozen instructions)
            float lo = (float)(a * cs[j].x - b * cs[j].y), hi = (float)(a * cs[j].y + b * cs[j].x);
            asm volatile("" : "+v"(lo), "+v"(hi));
            emit(i, lo);
            emit(i + HALF, hi);
        }
    }
};

// A row's piece; ONCE: one that nothing will find in a cache again.
template <bool ONCE, typename V> __device__ __forceinline__ V row_piece(const void *p)
{
    if constexpr (ONCE)
        return __builtin_nontemporal_load((const V *)p);
    else
        return *(const V *)p;
}

// Lane (n = lane & 15, g = lane >> 4) holds query row n.  Scores are formed
// transposed, keys x queries, so a lane has its own query's scores of keys
// 4 g + i of a 16-key tile: the softmax factors are lane-local, and the
// scores already are the operand of the value product.
template <typename T, int HD, bool WIDE, bool ONCE> struct Tile;

// f32 rows: v_mfma_f32_16x16x4_f32, 16 keys a step.  The head's dimensions
// are permuted alike on both sides of each product, for 16-byte loads.
template <int HD, bool WIDE, bool ONCE> struct Tile<float, HD, WIDE, ONCE> {
    static constexpr int KEYS = 16, NS = 4, NQ = HD / 16, NV = HD / 64, QROWS = 16;
    int lane;
    f4 q[NQ], kf[NQ], vf[4][NV], o[NV][4];

    __device__ __forceinline__ void init(const float *qs, const float *)  // qs [16][HD + 4]
    {
        const int n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int i = 0; i < NQ; i++) q[i] = *(const f4 *)(qs + n * (HD + 4) + 16 * i + 4 * g);
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[j][e] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ int key_of(int i) const { return 4 * (lane >> 4) + i; }
    // row[0]: the pool row of key n
    __device__ __forceinline__ void load_k(const float *pool, const int *row, int64_t stride)
    {
        const float *p = pool + max(row[0], 0) * stride + 4 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < NQ; i++) kf[i] = row_piece<ONCE, f4>(p + 16 * i);
    }
    __device__ __forceinline__ void load_v(const float *pool, const int *row, int64_t stride)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float *p = pool + max(__shfl(row[0], key_of(i)), 0) * stride + 4 * (lane & 15);
#pragma unroll
            for (int j = 0; j < NV; j++) vf[i][j] = row_piece<ONCE, f4>(p + 64 * j);
        }
    }
    // the new row, at key `at` of the tile, from LDS; values of keys that
    // are not seen become 0 (their factor is 0, but 0 times an infinity that
    // a stale row may hold is not)
    __device__ __forceinline__ void patch_k(const float *knew, int at)
    {
        if ((lane & 15) != at) return;
        const int g = lane >> 4;
#pragma unroll
        for (int i = 0; i < NQ; i++) kf[i] = *(const f4 *)(knew + 16 * i + 4 * g);
    }
    __device__ __forceinline__ void patch_v(const float *vnew, int at, uint32_t seen)
    {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < NV; j++) {
                if (key_of(i) == at) vf[i][j] = *(const f4 *)(vnew + 64 * j + 4 * (lane & 15));
                if (!((seen >> key_of(i)) & 1u)) vf[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            }
    }
    __device__ __forceinline__ void scores(float (&s)[NS], float scale)
    {
        const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        f4 c[4];
#pragma unroll
        for (int i = 0; i < NQ; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                c[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[i][e], q[i][e], i ? c[e] : zero, 0, 0, 0);
        const f4 t = (c[0] + c[1]) + (c[2] + c[3]);
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = t[i] * scale;
    }
    __device__ __forceinline__ void values(const float (&p)[NS], float corr)
    {
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                o[j][e] *= corr;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][j][e], p[i], o[j][e], 0, 0, 0);
            }
    }
    // values 64 j + 4 (4 g + r) .. + 3 of query n, r < 4
    __device__ __forceinline__ void put(int j, float *dst) const  // dst: 64 values of query n
    {
        const int g = lane >> 4;
#pragma unroll
        for (int r = 0; r < 4; r++)
            *(f4 *)(dst + 4 * (4 * g + r)) = f4{o[j][0][r], o[j][1][r], o[j][2][r], o[j][3][r]};
    }
};

// f16 rows: v_mfma_f32_16x16x32_f16, 32 keys a step.  Queries and factors are
// f32 values in two f16 pieces, hi + lo with |x - hi - lo| <= 2^-22 |x| (each
// rounding is off by half a step, 2^-11, of what it rounds), so the products
// are as exact as f32 ones; queries are brought to [2^9, 2^10) by a power of
// two per head and factors (at most 1) to 2^10, so that the low pieces of
// all that count are normal numbers.  With up to 8 query heads the two
// pieces are the two halves of the 16 query rows (WIDE: two products).
// Lane group g's keys are 4 g + i and 16 + 4 g + i on both sides of the value
// product; its V operand, 8 keys of one dimension, is made of 16-byte pieces
// of 8 rows by lane-local byte permutes.
template <int HD, bool WIDE, bool ONCE> struct Tile<_Float16, HD, WIDE, ONCE> {
    static constexpr int KEYS = 32, NS = 8, NQ = HD / 32, DPL = HD / 16, QROWS = WIDE ? 16 : 8;
    static constexpr int NB = DPL > 8 ? DPL / 8 : 1, ND = DPL > 8 ? 4 : DPL / 2;  // 16-byte blocks, dwords of each
    static constexpr int EB = 2 * ND;  // dims of a lane in a block
    static constexpr float PSCALE = 1024.0f;
    h8 q[NQ], ql[WIDE ? NQ : 1], kf[2][NQ];
    uint32_t vf[8][NB][ND];
    f4 o[NB][EB];
    float qscale;
    int lane;

    __device__ __forceinline__ void init(const float *qs, const float *qmax)
    {
        const int n = lane & 15, g = lane >> 4, row = n & (QROWS - 1);
        const float m = qmax[row];
        const int e = m > 0.0f && m < INFINITY ? (int)((__float_as_uint(m) >> 23) & 255) - 127 : 9;
        // 2^(9 - e), in range for every exponent: 9 - e within [-118, 136]
        const float up = e < -100 ? ldexpf(1.0f, 109) : ldexpf(1.0f, 9 - e);
        qscale = 1.0f / up;
#pragma unroll
        for (int i = 0; i < NQ; i++)
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const float v = qs[row * (HD + 4) + 32 * i + 8 * g + x] * up;
                const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
                q[i][x] = WIDE || n < 8 ? hi : lo;
                if constexpr (WIDE) ql[i][x] = lo;
            }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e2 = 0; e2 < EB; e2++) o[b][e2] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ int key_of(int i) const
    {
        return (i & 4) * 4 + 4 * (lane >> 4) + (i & 3);
    }
    // row[0], row[1]: the pool rows of keys n and 16 + n
    __device__ __forceinline__ void load_k(const _Float16 *pool, const int *row, int64_t stride)
    {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const _Float16 *p = pool + max(row[t], 0) * stride + 8 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < NQ; i++) kf[t][i] = row_piece<ONCE, h8>(p + 32 * i);
        }
    }
    template <bool NT> __device__ __forceinline__ void load_v_row(int i, const _Float16 *p)
    {
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t *s = (const uint32_t *)(p + 128 * b + EB * (lane & 15));
            if constexpr (ND == 4) {
                const styx_u4 v = row_piece<NT, styx_u4>(s);
#pragma unroll
                for (int d = 0; d < 4; d++) vf[i][b][d] = v[d];
            } else {
                const styx_u2 v = row_piece<NT, styx_u2>(s);
                vf[i][b][0] = v[0];
                vf[i][b][1] = v[1];
            }
        }
    }
    __device__ __forceinline__ void load_v(const _Float16 *pool, const int *row, int64_t stride)
    {
#pragma unroll
        for (int i = 0; i < 8; i++)
            load_v_row<ONCE>(i, pool + max(__shfl(row[i >> 2], key_of(i & 3)), 0) * stride);
    }
    __device__ __forceinline__ void patch_k(const _Float16 *knew, int at)
    {
        const int n = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < 2; t++)
            if (16 * t + n == at) {
#pragma unroll
                for (int i = 0; i < NQ; i++) kf[t][i] = *(const h8 *)(knew + 32 * i + 8 * g);
            }
    }
    __device__ __forceinline__ void patch_v(const _Float16 *vnew, int at, uint32_t seen)
    {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (key_of(i) == at) load_v_row<false>(i, vnew);
            if (!((seen >> key_of(i)) & 1u)) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int d = 0; d < ND; d++) vf[i][b][d] = 0;
            }
        }
    }
    __device__ __forceinline__ void scores(float (&s)[NS], float scale)
    {
        const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        scale *= qscale;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            f4 c = zero, d = zero;
#pragma unroll
            for (int i = 0; i < NQ; i++) {
                c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][i], q[i], c, 0, 0, 0);
                if constexpr (WIDE) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][i], ql[i], d, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // rows n and n + 8 (row_ror:8) are the two pieces of a query
                const float other = WIDE ? d[i] : dpp_f<0x128>(c[i]);
                s[4 * t + i] = (c[i] + other) * scale;
            }
        }
    }
    __device__ __forceinline__ void values(const float (&p)[NS], float corr)
    {
        const bool low = !WIDE && (lane & 8);
        h8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = p[i] * PSCALE;
            const _Float16 h = (_Float16)v, l = (_Float16)(v - (float)h);
            hi[i] = low ? l : h;
            lo[i] = l;
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < EB; e++) {
                // 8 keys of dimension e: halves e & 1 of dword e / 2 of 8 rows
                const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                styx_u4 w;
#pragma unroll
                for (int x = 0; x < 4; x++)
                    w[x] = __builtin_amdgcn_perm(vf[2 * x + 1][b][e >> 1], vf[2 * x][b][e >> 1], sel);
                const h8 vo = __builtin_bit_cast(h8, w);
                o[b][e] *= corr;
                o[b][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vo, hi, o[b][e], 0, 0, 0);
                if constexpr (WIDE) o[b][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vo, lo, o[b][e], 0, 0, 0);
            }
    }
    // values 64 j .. + 63 of query n; a lane has dims 128 b + EB (4 g + r) + e
    __device__ __forceinline__ void put(int j, float *dst) const
    {
        const int g = lane >> 4;
        constexpr int PER = 64 / EB;  // lanes' rows (4 g + r) that make 64 values
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int m = 4 * g + r;
#pragma unroll
                for (int e = 0; e < EB; e++) {
                    float v = o[b][e][r];
                    if constexpr (!WIDE) v += dpp_f<0x128>(v);
                    if (128 * b / 64 + m / PER == j) dst[m % PER * EB + e] = v * (1.0f / PSCALE);
                }
            }
    }
};

// LARGE: pools larger than the Infinity Cache (launch_ab).
template <typename T, int HD, bool WIDE, bool SCORED, bool LARGE>
__global__ void __launch_bounds__(AB_WG, ab_slots(HD) / 256) k_attn_batch(AttnBatchArgs a)
{
    using Any = Tile<T, HD, WIDE, false>;
    constexpr int KEYS = Any::KEYS, NS = Any::NS, QROWS = Any::QROWS, NR = KEYS / 16;
    __shared__ __align__(16) float s_q[QROWS][HD + 4];
    __shared__ float s_qmax[QROWS];
    __shared__ __align__(16) T s_k[HD], s_v[HD];
    constexpr int DR = HD < 128 ? HD : 128;  // dimensions merged at a time
    __shared__ __align__(16) float s_o[AB_WAVES][QROWS][DR + 4];
    __shared__ float s_m[AB_WAVES][16], s_l[AB_WAVES][16];
    const KvView &kv = a.kv;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const RowSplit sp = split_rows(a);
    if (blockIdx.x == 0 && wave == 0) split_store(a, sp);
    const uint32_t end = min(sp.units, (blockIdx.x + 1) * sp.share);
    auto pieces = [&](auto once) __attribute__((always_inline)) {
    using Tl = Tile<T, HD, WIDE, decltype(once)::value>;
    for (uint32_t u = blockIdx.x * sp.share; u < end;) {
    // (a lane number that the compiler takes for a new one in every trip:
    // what is computed from it would else be kept in registers over the
    // trips, a wave less of them per SIMD)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int n = lane & 15, g = lane >> 4;
    const SeqAt at = seq_find(a, sp, u);
    const int b = at.b, rows = at.rows, last = rows - 1;
    const uint32_t per_head = head_units(sp, rows), in_seq = u - at.first;
    const int kvh = in_seq / per_head, u0 = in_seq - kvh * per_head, nu = min(per_head - u0, end - u);
    u += nu;
    const int t0 = u0 * AB_UNIT, t1 = min(rows, t0 + nu * AB_UNIT);
    const int32_t *tab = kv.table + (int64_t)b * kv.table_len;
    const int64_t stride = (int64_t)kv.nkv * HD;
    const T *kp = (const T *)kv.kpool + kvh * HD, *vp = (const T *)kv.vpool + kvh * HD;
    Tl x;
    x.lane = lane;
    // pool rows of this lane's keys of a tile: page-table entries are asked
    // for one tile ahead of the rows, the rows one tile ahead of their use
    int entry[NR], row[NR];
    auto entries_at = [&](int tb) {
#pragma unroll
        for (int r = 0; r < NR; r++) entry[r] = kv.entry(tab, min(tb + 16 * r + n, last));
    };
    auto rows_at = [&](int tb) {
#pragma unroll
        for (int r = 0; r < NR; r++) row[r] = kv.row_of(entry[r], min(tb + 16 * r + n, last));
    };
    const int step = AB_WAVES * KEYS;
    int tb = t0 + wave * KEYS;
    const bool own = t1 == rows;  // this piece holds the new row
    // Everything that does not wait for the page table is asked for behind
    // it: loads are counted in order, and the rows of K and V after them
    // then do not hold up the heads.
    entries_at(tb);
    constexpr int PPL = HeadRow<HD>::PPL;
    const int pos = a.pos[b];
    double2 cs[PPL];
    HeadRow<HD> hq[QROWS / AB_WAVES], qw, hk, kw, hv;
#pragma unroll
    for (int j = 0; j < PPL; j++) cs[j] = a.rope[(int64_t)pos * (HD / 2) + (HD < 128 ? lane & (HD / 2 - 1) : lane + 64 * j)];
    const float *qb = a.q + ((int64_t)b * a.nh + kvh * a.gqa) * HD;
#pragma unroll
    for (int i = 0; i < QROWS / AB_WAVES; i++) hq[i].load(qb + min(wave + AB_WAVES * i, a.gqa - 1) * HD, lane);
    qw.load(a.q_norm ? a.q_norm : qb, lane);
    const int64_t in = ((int64_t)b * kv.nkv + kvh) * HD;
    if (own && wave == AB_WAVES - 1) {
        hk.load(a.k + in, lane);
        kw.load(a.k_norm ? a.k_norm : a.k + in, lane);
        hv.load(a.v + in, lane);
    }
    rows_at(tb);
    x.load_k(kp, row, stride);
    x.load_v(vp, row, stride);
    entries_at(tb + step);
#pragma unroll
    for (int i = 0; i < QROWS / AB_WAVES; i++) {
        const int h = wave + AB_WAVES * i;
        float big = 0.0f;
        if (h < a.gqa)
            hq[i].turn(qw, a.q_norm != nullptr, cs, a.eps, lane, [&](int d, float v) {
                s_q[h][d] = v;
                big = fmaxf(big, fabsf(v));
            });
        else
            for (int d = lane; d < HD; d += 64) s_q[h][d] = 0.0f;
        if constexpr (!std::is_same<T, float>::value) {
            big = wave_max(big);
            if (lane == 0) s_qmax[h] = big;
        }
    }
    if (own && wave == AB_WAVES - 1) {
        hk.turn(kw, a.k_norm != nullptr, cs, a.eps, lane, [&](int d, float v) { s_k[d] = (T)v; });
#pragma unroll
        for (int j = 0; j < PPL; j++)
            if (HD >= 128 || lane < HD / 2) {
                s_v[lane + 64 * j] = (T)hv.x0[j];
                s_v[lane + 64 * j + HD / 2] = (T)hv.x1[j];
            }
    }
    __syncthreads();
    x.init(&s_q[0][0], s_qmax);
    float m = -INFINITY, l = 0.0f;  // l: this lane group's share
    float *score = nullptr;
    if constexpr (SCORED)
        score = a.score + (((int64_t)b * kv.nkv + kvh) * a.gqa + min(n, a.gqa - 1)) * a.stride;
    for (; tb < t1; tb += step) {
        // keys seen: of the tile's, those of the piece whose page is there
        uint32_t seen = 0;
#pragma unroll
        for (int r = 0; r < NR; r++)
            seen |= (uint32_t)(__ballot(row[r] >= 0 && tb + 16 * r + n < t1) & 0xFFFFu) << (16 * r);
        const bool whole = seen == (KEYS == 32 ? 0xFFFFFFFFu : 0xFFFFu) && !(own && last < tb + KEYS);
        const int fresh = own ? last - tb : -1;
        if (!whole) x.patch_k(s_k, fresh);
        float s[NS], mn = m;
        x.scores(s, a.scale);
        // the next tile's K (issued after the last tile too, of clamped rows:
        // every trip then issues the same loads)
        const int tn = tb + step;
        rows_at(tn);
        x.load_k(kp, row, stride);
        entries_at(tn + step);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < NS; i++)
                if (!((seen >> x.key_of(i)) & 1u)) s[i] = -INFINITY;
            x.patch_v(s_v, fresh, seen);
        }
        if constexpr (SCORED) {
            if (n < a.gqa) {
#pragma unroll
                for (int r = 0; r < NR; r++)
                    *(f4 *)(score + tb + 16 * r + 4 * g) = f4{s[4 * r], s[4 * r + 1], s[4 * r + 2], s[4 * r + 3]};
            }
        }
#pragma unroll
        for (int i = 0; i < NS; i++) mn = fmaxf(mn, s[i]);
        mn = groups_max(mn);
        const float mz = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet
        const float corr = exp2_(m - mz);
        m = mn;
        float lb = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            s[i] = exp2_(s[i] - mz);
            lb += s[i];
        }
        l = l * corr + lb;
        x.values(s, corr);
        x.load_v(vp, row, stride);
    }
    // the new row goes to the pools (the tiles took it from LDS)
    if (own && wave == 0) {
        const int r = kv.row(tab, last);
        if (r >= 0)
            for (int i = lane; i < HD; i += 64) {
                ((T *)kv.kpool)[r * stride + kvh * HD + i] = s_k[i];
                ((T *)kv.vpool)[r * stride + kvh * HD + i] = s_v[i];
            }
        if (a.slot_pos && lane == 0) a.slot_pos[((int64_t)b * kv.nkv + kvh) * kv.cap + last] = pos;
    }
    // the waves' results of each head merged, one partial per piece and head
    l = groups_sum(l);
    if (g == 0 && n < QROWS) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
    const int64_t pc = ((int64_t)blockIdx.x + b * kv.nkv + kvh) * a.gqa;
#pragma unroll
    for (int d0 = 0; d0 < HD; d0 += DR) {
        __syncthreads();
        // (every lane takes part: pieces of a query come from two lanes)
#pragma unroll
        for (int j = 0; j < DR / 64; j++) x.put(d0 / 64 + j, s_o[wave][n & (QROWS - 1)] + 64 * j);
        __syncthreads();
        for (int i = threadIdx.x; i < a.gqa * DR; i += AB_WG) {
            const int h = i / DR, d = i % DR;
            float M = s_m[0][h];
#pragma unroll
            for (int w = 1; w < AB_WAVES; w++) M = fmaxf(M, s_m[w][h]);
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < AB_WAVES; w++) {
                const float f = part_factor(s_m[w][h], M);
                L += s_l[w][h] * f;
                O += s_o[w][h][d] * f;
            }
            a.part_o[(pc + h) * HD + d0 + d] = O;
            if (d0 == 0 && d == 0) {
                a.part_ml[2 * (pc + h)] = M;
                a.part_ml[2 * (pc + h) + 1] = L;
            }
        }
    }
    }
    };
    if constexpr (LARGE) {
        if (__builtin_amdgcn_readfirstlane(sp.units) > a.once_units) {
            pieces(std::true_type{});
            return;
        }
    }
    pieces(std::false_type{});
}

// The pieces of one kv head: their partials lie one after another (piece i of
// the batch is workgroup w's of the p-th head with w + p = i).
struct Pieces {
    int64_t first;
    int count;
};
__device__ __forceinline__ Pieces pieces_of(const AttnBatchArgs &a, const RowSplit &sp, const SeqAt &at, int kvh)
{
    const uint32_t per_head = head_units(sp, at.rows), u = at.first + kvh * per_head;
    const uint32_t w0 = u / sp.share, w1 = (u + per_head - 1) / sp.share;
    return {(int64_t)w0 + at.b * a.kv.nkv + kvh, (int)(w1 - w0) + 1};
}

// Partials of every STEP-th piece from c0 on of one head merged by a thread:
// the loads of AB_BATCH pieces in flight at once, their maximum first, then
// independent factors.  O: of the value at dim; else M and L alone.
template <int STEP, bool O>
__device__ __forceinline__ void merge_pieces(const AttnBatchArgs &a, const Pieces &at, int c0, int hg, int dim,
                                             float &m, float &l, float &o)
{
    m = -INFINITY;
    l = o = 0.0f;
    for (int c = c0; c < at.count; c += STEP * AB_BATCH) {
        float2 ml[AB_BATCH];
        float oc[AB_BATCH];
#pragma unroll
        for (int i = 0; i < AB_BATCH; i++) {
            const int cc = min(c + STEP * i, at.count - 1);
            const int64_t p = (at.first + cc) * a.gqa + hg;
            ml[i] = ((const float2 *)a.part_ml)[p];
            if (O) oc[i] = a.part_o[p * a.kv.hd + dim];
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < AB_BATCH; i++) {
            if (c + STEP * i >= at.count) {
                ml[i] = float2{-INFINITY, 0.0f};
                oc[i] = 0.0f;
            }
            mn = fmaxf(mn, ml[i].x);
        }
        const float fa = part_factor(m, mn);
        l *= fa;
        o *= fa;
#pragma unroll
        for (int i = 0; i < AB_BATCH; i++) {
            const float f = part_factor(ml[i].x, mn);
            l += ml[i].y * f;
            if (O) o += oc[i] * f;
        }
        m = mn;
    }
}

// The pieces joined.  Workgroups below n_merge: one query head of one
// sequence and DIMS of its dimensions, each part of the workgroup taking
// every AB_WG / DIMS-th piece.  The others: every a.tiles-th step of one kv
// head's weights, M and L of its heads formed from the pieces' first (16
// lanes a head), the first step's scores in flight meanwhile.
template <int DIMS, int HM>
__global__ void __launch_bounds__(AB_WG) k_attn_batch_join(AttnBatchArgs a)
{
    constexpr int PARTS = AB_WG / DIMS, PER = ab_wper(HM);
    __shared__ float s_o[PARTS][DIMS], s_m[PARTS], s_l[PARTS], s_M[16], s_R[16];
    const KvView &kv = a.kv;
    const int tid = threadIdx.x;
    RowSplit sp;
    if ((int)blockIdx.x < a.n_merge) {
        const int nd = kv.hd / DIMS, bh = blockIdx.x / nd, d0 = blockIdx.x % nd * DIMS;
        const int b = bh / a.nh, h = bh % a.nh, kvh = h / a.gqa, hg = h % a.gqa;
        const SeqAt at = seq_load(a, sp, b);
        if (at.rows == 0) return;
        const int part = tid / DIMS, d = tid % DIMS;
        float m, l, o;
        merge_pieces<PARTS, true>(a, pieces_of(a, sp, at, kvh), part, hg, d0 + d, m, l, o);
        s_o[part][d] = o;
        if (d == 0) {
            s_m[part] = m;
            s_l[part] = l;
        }
        __syncthreads();
        if (tid < DIMS) {
            float M = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < PARTS; w++) M = fmaxf(M, s_m[w]);
#pragma unroll
            for (int w = 0; w < PARTS; w++) {
                const float f = part_factor(s_m[w], M);
                L += s_l[w] * f;
                O += s_o[w][tid] * f;
            }
            // no row with a weight (M = -inf): 0, or NaN
            a.out[((int64_t)b * a.nh + h) * kv.hd + d0 + tid] = M == -INFINITY ? O + L : O / L;
        }
        return;
    }
    const int w = blockIdx.x - a.n_merge, tile = w % a.tiles, bk = w / a.tiles;
    const int b = bk / kv.nkv, kvh = bk % kv.nkv;
    const SeqAt at = seq_load(a, sp, b);
    constexpr int STEP = PER * AB_WG;
    if (tile * STEP >= at.rows) return;
    const int64_t base = (int64_t)b * kv.nkv + kvh;
    const float *sc = a.score + base * a.gqa * a.stride;
    // (every load on every path: heads past the last read it again, and without
    // weights to add to, those that are to be written are read and dropped)
    const float *acc = (a.acc_in ? a.acc_in : a.acc_out) + base * kv.cap;
    float s[PER][HM], old[PER];
    auto load = [&](int t0) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int t = min(t0 + tid + AB_WG * j, at.rows - 1);
#pragma unroll
            for (int h = 0; h < HM; h++) s[j][h] = sc[(int64_t)min(h, a.gqa - 1) * a.stride + t];
            old[j] = acc[t];
        }
    };
    load(tile * STEP);
    {
        const int h = tid >> 4;
        float m = -INFINITY, l = 0.0f, o;
        if (h < a.gqa) merge_pieces<16, false>(a, pieces_of(a, sp, at, kvh), tid & 15, h, 0, m, l, o);
        const float M = bfly<16>(m, [](float x, float y) { return fmaxf(x, y); });
        const float L = bfly_sum<16>(l * part_factor(m, M));
        if ((tid & 15) == 0) {
            s_M[h] = M == -INFINITY ? 0.0f : M;
            s_R[h] = M == -INFINITY ? L : 1.0f / L;
        }
    }
    __syncthreads();
    for (int t0 = tile * STEP;;) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int t = t0 + tid + AB_WG * j;
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < HM; h++)
                if (h < a.gqa) sum += exp2_(s[j][h] - s_M[h]) * s_R[h];
            if (t < at.rows) a.acc_out[base * kv.cap + t] = (a.acc_in && t < at.rows - 1 ? a.decay * old[j] : 0.0f) + sum;
        }
        t0 += a.tiles * STEP;
        if (t0 >= at.rows) break;
        load(t0);
    }
}

// Dimensions of a merging workgroup: all of a head's where that makes two
// workgroups per CU, else as few as it takes (32 at least), so that many
// pieces of few heads are read by many.
static int merge_dims(int64_t heads, int hd)
{
    int d = hd;
    while (d > 32 && heads * (hd / d) < 512) d /= 2;
    return d;
}

AttnBatchWs attn_batch_ws(int n_seq, int nkv, int hd, int cap, int gqa, bool scored)
{
    AttnBatchWs w{};
    const int64_t heads = (int64_t)n_seq * nkv;
    w.units = ((int64_t)cap + AB_UNIT - 1) / AB_UNIT * heads;
    w.grid = std::min<int64_t>(w.units, ab_slots(hd));
    const int64_t pieces = w.grid + heads;
    w.stride = (cap + 63) / 64 * 64;
    w.ml = (2 * pieces * gqa + 63) / 64 * 64;
    w.o = pieces * gqa * hd;
    w.plan = ((int64_t)n_seq + 2 + 63) / 64 * 64;
    w.score = scored ? heads * gqa * w.stride : 0;
    w.dims = merge_dims(heads * gqa, hd);
    // weights: eight workgroups per CU, or one for every step
    const int step = ab_wper(gqa) * AB_WG;
    w.tiles = scored ? (int)std::min<int64_t>((cap - 1) / step + 1, std::max<int64_t>(1, 2048 / heads)) : 0;
    w.join = heads * gqa * (hd / w.dims) + heads * w.tiles;
    return w;
}

template <typename T, int HD, bool WIDE>
static void launch_ab(hipStream_t st, AttnBatchArgs a, int64_t grid)
{
    const dim3 g((unsigned)grid), wg(AB_WG);
    // Rows past the Infinity Cache come from HBM, and loads that leave nothing
    // behind stream them 5-9% faster (40 f16 sequences of 8 heads, 327 MB: 83
    // -> 76 us); fewer may be found there by the next call, which such loads
    // would spoil (24 conversations, 102 MB, call after call: 32 us against
    // 38).  What counts are the rows that the call reads, which the device
    // knows (those of shared pages count for each sequence), and no more than
    // there are: a kernel that looks carries both loops, of which a call of few
    // rows notices the length (eight conversations: 21.0 us without, 21.7
    // with), and is taken only where the pools are larger.
    const KvView &kv = a.kv;
    constexpr double ROW = 2.0 * sizeof(T) * HD, CACHE = 256.0 * (1 << 20);
    const bool large = ROW * kv.nkv * kv.n_pages * kv.page_tokens > CACHE;
    a.once_units = (uint32_t)(CACHE / (ROW * AB_UNIT));
    if (a.acc_out) {
        if (large)
            hipLaunchKernelGGL((k_attn_batch<T, HD, WIDE, true, true>), g, wg, 0, st, a);
        else
            hipLaunchKernelGGL((k_attn_batch<T, HD, WIDE, true, false>), g, wg, 0, st, a);
    } else {
        if (large)
            hipLaunchKernelGGL((k_attn_batch<T, HD, WIDE, false, true>), g, wg, 0, st, a);
        else
            hipLaunchKernelGGL((k_attn_batch<T, HD, WIDE, false, false>), g, wg, 0, st, a);
    }
}

template <int HD> static void launch_ab_hd(hipStream_t st, const AttnBatchArgs &a, int64_t grid)
{
    if (!a.kv.f16)
        launch_ab<float, HD, true>(st, a, grid);
    else if (a.gqa > 8)
        launch_ab<_Float16, HD, true>(st, a, grid);
    else
        launch_ab<_Float16, HD, false>(st, a, grid);
}

template <int DIMS> static void launch_join(hipStream_t st, const AttnBatchArgs &a, int64_t grid)
{
    if (a.gqa <= 4)
        hipLaunchKernelGGL((k_attn_batch_join<DIMS, 4>), dim3((unsigned)grid), dim3(AB_WG), 0, st, a);
    else if (a.gqa <= 8)
        hipLaunchKernelGGL((k_attn_batch_join<DIMS, 8>), dim3((unsigned)grid), dim3(AB_WG), 0, st, a);
    else
        hipLaunchKernelGGL((k_attn_batch_join<DIMS, 16>), dim3((unsigned)grid), dim3(AB_WG), 0, st, a);
}

hipError_t launch_attn_batch(hipStream_t st, AttnBatchArgs a, float *ws)
{
    const KvView &kv = a.kv;
    const AttnBatchWs w = attn_batch_ws(kv.n_seq, kv.nkv, kv.hd, kv.cap, a.gqa, a.acc_out != nullptr);
    a.stride = w.stride;
    a.scale = (float)((double)a.scale * 1.4426950408889634);  // log2 e
    a.n_merge = kv.n_seq * a.nh * (kv.hd / w.dims);
    a.tiles = w.tiles;
    a.part_ml = ws;
    a.part_o = a.part_ml + w.ml;
    a.plan = (uint32_t *)(a.part_o + w.o);
    a.score = a.part_o + w.o + w.plan;
    switch (kv.hd) {
    case 64: launch_ab_hd<64>(st, a, w.grid); break;
    case 128: launch_ab_hd<128>(st, a, w.grid); break;
    default: launch_ab_hd<256>(st, a, w.grid); break;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    switch (w.dims) {
    case 32: launch_join<32>(st, a, w.join); break;
    case 64: launch_join<64>(st, a, w.join); break;
    case 128: launch_join<128>(st, a, w.join); break;
    default: launch_join<256>(st, a, w.join); break;
    }
    return hipGetLastError();
}

}  // namespace styx
