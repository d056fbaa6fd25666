// kv_append.hip -- per-head RMSNorm and rotary positions of new tokens' q and
// k, and their k and v into the rows of a paged KV cache.
//
//   x^ = x / sqrt(mean x^2 + eps) * w, then for each pair (a, b) of the first
//   n_rot dims, (i, i + n_rot/2) or (2i, 2i+1), with (c, s) = table[pos][i]:
//   a' = a c - b s, b' = a s + b c
// in f64 to the end and rounded to f32 and then to the type.  Another order of
// the f64 sums (the single-token operator's) gives the same bits but for the rare
// value that lies at a rounding's border, which is a step of the type away.
//
// Bound: HBM, each value read once and written once.  A head is 16 bytes a lane;
// a wave takes heads of one row, the next under way while one is turned, and
// keeps the row's sines and cosines.  The partner of a dim is in the same lane
// where pairs are neighbours, else it is read back from LDS (for a part of a
// head it may lie anywhere).  A row's heads go to several workgroups where rows
// are few: 48 tokens 5.5 us a call.  8192 f16 tokens of
// 40 heads, 172 MB: 41 us in the kernel (4.2 TB/s), 51 where neither side is in
// a cache; 4 parts of documents, f32 heads of 256, 125 MB: 27 and 30 us.  A
// workgroup lives for a row, whose position, angles and turn wait for one
// another, so that few bytes are under way.  By types, 8192 tokens as above
// under norms, all of each head turned: f32 to f16 69 us, to an f16 cache and
// f32 queries 76, f16 to an f16 cache and f32 queries 120 (a lane then stores 32
// bytes in two pieces, lines half by half); 56, 70 and 52 at a copy's rate.
// Loads and stores are plain: with non-temporal loads the prompt takes 50 us from
// memory, but 49 instead of 41 where the Infinity Cache holds what the product
// before has just written, as it does in use.
#include <algorithm>

#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int KA_WG = 256;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <typename T, int N> struct Piece;
template <> struct Piece<float, 4> { typedef styx_f4 V; };
template <> struct Piece<_Float16, 4> { typedef _Float16 V __attribute__((ext_vector_type(4))); };
template <> struct Piece<_Float16, 8> { typedef h8 V; };

// N consecutive values, and from floats, in pieces of 16 bytes at most
template <typename T, int N> __device__ __forceinline__ void store_row(T *p, const float (&x)[N])
{
    constexpr int M = sizeof(T) == 4 ? 4 : N < 8 ? N : 8;
#pragma unroll
    for (int i = 0; i < N; i += M) {
        typename Piece<T, M>::V v;
#pragma unroll
        for (int e = 0; e < M; e++) v[e] = (T)x[i + e];
        *(typename Piece<T, M>::V *)(p + i) = v;
    }
}

template <typename TI, typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(KA_WG, 4) k_kv_append(KvAppendArgs a)
{
    constexpr int VEC = sizeof(TI) == 2 ? 8 : 4, LPH = HD / VEC, HPW = 64 / LPH;  // heads of a wave at once
    __shared__ __align__(16) float s_x[KA_WG / 64][HPW][HD + 4];
    const KvView &kv = a.kv;
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = lane / LPH, d0 = lane % LPH * VEC;
    const int pos = a.row_pos ? a.row_pos[row] : 0;
    const int at = a.k ? a.row_at[row] : -1;
    // (a row of no sequence has a position below 0, with a table or without)
    if (a.rope ? (uint32_t)pos >= (uint32_t)a.n_pos : pos < 0) return;
    const bool store = at >= 0 && at < kv.n_pages * kv.page_tokens;
    // groups of heads: q's, then k's, then v's
    const int gq = (a.nh + HPW - 1) / HPW, gk = (kv.nkv + HPW - 1) / HPW, groups = gq + (store ? 2 * gk : 0);
    const int step = gridDim.y * (KA_WG / 64);
    struct Head {
        int kind, h;  // 0 q, 1 k, 2 v; head
    };
    auto head_of = [&](int g) {
        const int kind = g < gq ? 0 : g < gq + gk ? 1 : 2;
        return Head{kind, (kind == 0 ? g : kind == 1 ? g - gq : g - gq - gk) * HPW + slot};
    };
    typedef typename Piece<TI, VEC>::V Raw;
    auto load = [&](int g) {
        const Head o = head_of(min(g, groups - 1));
        const TI *p = o.kind == 0   ? (const TI *)a.q + row * a.ldq + (int64_t)min(o.h, a.nh - 1) * HD
                      : o.kind == 1 ? (const TI *)a.k + row * a.ldk + (int64_t)min(o.h, kv.nkv - 1) * HD
                                    : (const TI *)a.v + row * a.ldv + (int64_t)min(o.h, kv.nkv - 1) * HD;
        return *(const Raw *)(p + d0);
    };
    int g = blockIdx.y * (KA_WG / 64) + wave;
    if (g >= groups) return;
    Raw next = load(g);  // (two or three ahead measured the same or slower)
    // of this lane's dims: cosine, and the partner's sine with its sign, times
    // the norm's weights; the partner
    double c[VEC], s[VEC];
    const int half = a.n_rot / 2;
    auto other = [&](int d) { return d >= a.n_rot ? d : a.interleaved ? d ^ 1 : d >= half ? d - half : d + half; };
    int kind = -1;
    for (; g < groups; g += step) {
        const Head o = head_of(g);
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = (float)next[e];
        next = load(g + step);
        const bool is = o.h < (o.kind ? kv.nkv : a.nh);
        if (o.kind < 2) {
            const float *w = o.kind ? a.k_norm : a.q_norm;
            if (o.kind != kind) {
                kind = o.kind;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const int d = d0 + e;
                    double2 cs = {1.0, 0.0};
                    if (d < a.n_rot) cs = a.rope[(int64_t)pos * half + (a.interleaved ? d >> 1 : d >= half ? d - half : d)];
                    c[e] = cs.x;
                    s[e] = (a.interleaved ? d & 1 : d >= half) ? cs.y : -cs.y;
                }
                if (w)
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        c[e] *= w[d0 + e];
                        s[e] *= w[other(d0 + e)];
                    }
            }
            double f = 1.0;
            if (w) {
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < VEC; e++) ss += (double)x[e] * x[e];
#pragma unroll
                for (int m = 1; m < LPH; m <<= 1) ss += __shfl_xor(ss, m);
                f = 1.0 / sqrt(ss * (1.0 / HD) + (double)a.eps);
            }
            float xo[VEC];
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < VEC; e++) xo[e] = x[e ^ 1];
            } else {
                // (a wave's LDS operations are carried out in order)
#pragma unroll
                for (int e = 0; e < VEC; e += 4) *(styx_f4 *)&s_x[wave][slot][d0 + e] = styx_f4{x[e], x[e + 1], x[e + 2], x[e + 3]};
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int e = 0; e < VEC; e++) xo[e] = s_x[wave][slot][other(d0 + e)];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const double me = x[e] * c[e];
                // (a dim that is not turned keeps its value, whatever it is)
                float v = (float)(f * (d0 + e < a.n_rot ? me + xo[e] * s[e] : me));
                // (kept apart from a conversion to f16 that may follow:
                // contracted with it, the f64 value would be rounded to f16 directly)
                asm volatile("" : "+v"(v));
                x[e] = v;
            }
        }
        if (!is) continue;
        if (o.kind == 0)
            store_row<TQ, VEC>((TQ *)a.q_out + row * a.ldo + (int64_t)o.h * HD + d0, x);
        else
            store_row<TC, VEC>((TC *)(o.kind == 1 ? kv.kpool : kv.vpool) + ((int64_t)at * kv.nkv + o.h) * HD + d0, x);
    }
}

// Workgroups of a row: as many as its heads make where rows are few, so that
// the chip is filled, else one, whose waves keep the row's sines and cosines.
static int row_groups(const KvAppendArgs &a)
{
    const int vec = a.in_f16 ? 8 : 4, hpw = 64 / (a.kv.hd / vec);
    const int64_t groups = (a.nh + hpw - 1) / hpw + (a.k ? 2 * ((a.kv.nkv + hpw - 1) / hpw) : 0), most = (groups + 3) / 4;
    return (int)std::min<int64_t>(std::max<int64_t>(1, std::min<int64_t>(most, 2048 / std::max(a.n_rows, 1))), 65535);
}
int64_t kv_append_grid(const KvAppendArgs &a) { return (int64_t)a.n_rows * row_groups(a); }

template <typename TI, typename TQ, typename TC> static void launch_hd(hipStream_t st, const KvAppendArgs &a)
{
    const dim3 g((unsigned)a.n_rows, (unsigned)row_groups(a)), wg(KA_WG);
    switch (a.kv.hd) {
    case 64: hipLaunchKernelGGL((k_kv_append<TI, TQ, TC, 64>), g, wg, 0, st, a); break;
    case 128: hipLaunchKernelGGL((k_kv_append<TI, TQ, TC, 128>), g, wg, 0, st, a); break;
    default: hipLaunchKernelGGL((k_kv_append<TI, TQ, TC, 256>), g, wg, 0, st, a); break;
    }
}
template <typename TI, typename TQ> static void launch_c(hipStream_t st, const KvAppendArgs &a)
{
    a.kv.f16 ? launch_hd<TI, TQ, _Float16>(st, a) : launch_hd<TI, TQ, float>(st, a);
}
template <typename TI> static void launch_q(hipStream_t st, const KvAppendArgs &a)
{
    a.q_f16 ? launch_c<TI, _Float16>(st, a) : launch_c<TI, float>(st, a);
}
hipError_t launch_kv_append(hipStream_t st, const KvAppendArgs &a)
{
    a.in_f16 ? launch_q<_Float16>(st, a) : launch_q<float>(st, a);
    return hipGetLastError();
}

}  // namespace styx
