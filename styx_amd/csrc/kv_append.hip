// kv_append.hip -- per-head RMSNorm and rotary positions of new tokens' q and
// k, and their k and v into the rows of a paged KV cache.
//
//   x^ = x / sqrt(mean x^2 + eps) * w, then for each pair (a, b) of the first
//   n_rot dims, (i, i + n_rot/2) or (2i, 2i+1), with (c, s) = table[pos][i]:
//   a' = a c - b s, b' = a s + b c
// in f64 to the end and rounded to f32 and then to the type, so that a cache
// holds the same bits whatever the order of a sum.
//
// Bound: HBM, each value read once and written once.  A head is VEC values a
// lane; the partner of a dim, which for a part of a head may lie anywhere, is
// read back from LDS.
#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int KA_WG = 256;
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <typename T, int N> struct Piece;
template <> struct Piece<float, 4> { typedef styx_f4 V; };
template <> struct Piece<_Float16, 4> { typedef _Float16 V __attribute__((ext_vector_type(4))); };
template <> struct Piece<_Float16, 8> { typedef h8 V; };

// N consecutive values as floats / from floats, in pieces of 16 bytes at most
template <typename T, int N> __device__ __forceinline__ void load_row(const T *p, float (&x)[N])
{
    constexpr int M = sizeof(T) == 4 ? 4 : N < 8 ? N : 8;
#pragma unroll
    for (int i = 0; i < N; i += M) {
        const auto v = *(const typename Piece<T, M>::V *)(p + i);
#pragma unroll
        for (int e = 0; e < M; e++) x[i + e] = (float)v[e];
    }
}
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
__global__ void __launch_bounds__(KA_WG) k_kv_append(KvAppendArgs a)
{
    constexpr int VEC = sizeof(TI) == 2 ? 8 : 4, LPH = HD / VEC, HEADS = KA_WG / LPH;
    __shared__ float s_x[HEADS][HD + 4];
    const KvView &kv = a.kv;
    const int row = blockIdx.x, tid = threadIdx.x, slot = tid / LPH, d0 = tid % LPH * VEC;
    const int pos = a.rope ? a.row_pos[row] : 0;
    if (a.rope && (uint32_t)pos >= (uint32_t)a.n_pos) return;
    const int at = a.k ? a.row_at[row] : -1;
    const bool store = at >= 0 && at < kv.n_pages * kv.page_tokens;
    // this lane's dims: (cos, sin), the sign of the partner's sine, its dim
    const int half = a.n_rot / 2;
    double c[VEC], s[VEC];
    int other[VEC];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const int d = d0 + e;
        c[e] = 1.0;
        s[e] = 0.0;
        other[e] = d;
        if (d < a.n_rot) {
            const bool hi = a.interleaved ? d & 1 : d >= half;
            const double2 cs = a.rope[(int64_t)pos * half + (a.interleaved ? d >> 1 : hi ? d - half : d)];
            other[e] = a.interleaved ? d ^ 1 : hi ? d - half : d + half;
            c[e] = cs.x;
            s[e] = hi ? cs.y : -cs.y;
        }
    }
    const int heads = a.nh + (store ? 2 * kv.nkv : 0);
    for (int h0 = 0; h0 < heads; h0 += HEADS) {
        const int h = h0 + slot;
        const bool is = h < heads, is_q = h < a.nh, is_v = h >= a.nh + kv.nkv;
        float x[VEC];
        if (is) {
            const TI *p = is_q    ? (const TI *)a.q + row * a.ldq + (int64_t)h * HD
                          : is_v ? (const TI *)a.v + row * a.ldv + (int64_t)(h - a.nh - kv.nkv) * HD
                                 : (const TI *)a.k + row * a.ldk + (int64_t)(h - a.nh) * HD;
            load_row<TI, VEC>(p + d0, x);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = 0.0f;
        }
        const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        double f = 1.0, ss = 0.0;
#pragma unroll
        for (int e = 0; e < VEC; e++) ss += (double)x[e] * x[e];
#pragma unroll
        for (int m = 1; m < LPH; m <<= 1) ss += __shfl_xor(ss, m);
        if (w) f = 1.0 / sqrt(ss * (1.0 / HD) + (double)a.eps);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; e++) s_x[slot][d0 + e] = x[e];
        __syncthreads();
        if (!is) continue;
        if (!is_v) {
            float y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const double me = w ? x[e] * f * w[d0 + e] : x[e];
                const float xo = s_x[slot][other[e]];
                const double you = w ? xo * f * w[other[e]] : xo;
                // (a dim that is not turned keeps its value, whatever it is)
                float v = (float)(d0 + e < a.n_rot ? me * c[e] + you * s[e] : me);
                // (kept apart from a conversion to f16 that may follow:
                // contracted with it, the f64 value would be rounded to f16 directly)
                asm volatile("" : "+v"(v));
                y[e] = v;
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) x[e] = y[e];
        }
        if (is_q) {
            store_row<TQ, VEC>((TQ *)a.q_out + row * a.ldo + (int64_t)h * HD + d0, x);
        } else {
            TC *pool = (TC *)(is_v ? kv.vpool : kv.kpool);
            store_row<TC, VEC>(pool + ((int64_t)at * kv.nkv + (h - a.nh) % kv.nkv) * HD + d0, x);
        }
    }
}

int64_t kv_append_grid(const KvAppendArgs &a) { return a.n_rows; }

template <typename TI, typename TQ, typename TC> static void launch_hd(hipStream_t st, const KvAppendArgs &a)
{
    const dim3 g((unsigned)kv_append_grid(a)), wg(KA_WG);
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
