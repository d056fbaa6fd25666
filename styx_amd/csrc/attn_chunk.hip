// attn_chunk.hip -- causal attention of the new tokens of a batch over their
// sequences' slots of a paged KV cache.
//
// Token i of sequence b with n = len[b] rows, query head h of kv head j:
//   s_t = scale q . K[t], t <= n + i (and t > n + i - window), pages in the pool
//   M = max s_t, L = sum e^(s_t - M), out = sum e^(s_t - M) V[t] / L, lse = M + ln L
//
// The plain kernel: a wave for a token and head, 64 slots at a time, one for
// each lane's score, then the running maximum and sum, then the lanes take the
// head's dims.
#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int AC_WG = 256, AC_WAVES = AC_WG / 64;

// The sequence of a row, by a wave: -1 for a row of none.
__device__ __forceinline__ int seq_of_row(const ChunkView &c, const KvView &kv, int row, ChunkSeq &s)
{
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < kv.n_seq; b0 += 64) {
        const ChunkSeq mine = chunk_seq(c, kv, b0 + lane);
        const bool hit = mine.count > 0 && row >= mine.first && row - mine.first < mine.count;
        if (const unsigned long long m = __ballot(hit)) {
            const int l = __builtin_ctzll(m);
            s = {(int)__builtin_amdgcn_readlane(mine.first, l), (int)__builtin_amdgcn_readlane(mine.count, l),
                 (int)__builtin_amdgcn_readlane(mine.len, l)};
            return b0 + l;
        }
    }
    return -1;
}

template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(AC_WG) k_attn_chunk(AttnChunkArgs a)
{
    __shared__ float s_q[AC_WAVES][HD];
    __shared__ float s_p[AC_WAVES][64];
    __shared__ int s_row[AC_WAVES][64];
    constexpr int DPL = HD / 64;
    const KvView &kv = a.kv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t item = (int64_t)blockIdx.x * AC_WAVES + wave;
    const int row = (int)(item / a.nh), h = (int)(item % a.nh), kvh = h / a.gqa;
    ChunkSeq s{};
    const int b = row < a.chunk.n_rows ? seq_of_row(a.chunk, kv, row, s) : -1;
    const bool is = b >= 0;
    if (is)
        for (int d = lane; d < HD; d += 64) s_q[wave][d] = (float)((const TQ *)a.q)[row * a.ldq + (int64_t)h * HD + d];
    __syncthreads();
    if (!is) return;
    const int at = s.len + row - s.first, t1 = at + 1, t0 = a.window && t1 > a.window ? t1 - a.window : 0;
    const int32_t *tab = kv.table + (int64_t)b * kv.table_len;
    const int64_t stride = (int64_t)kv.nkv * HD;
    const TC *kp = (const TC *)kv.kpool + kvh * HD, *vp = (const TC *)kv.vpool + kvh * HD;
    float m = -INFINITY, l = 0.0f, o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; j++) o[j] = 0.0f;
    for (int tb = t0; tb < t1; tb += 64) {
        const int t = tb + lane, r = t < t1 ? kv.row(tab, t) : -1;
        float x = -INFINITY;
        if (r >= 0) {
            float sum = 0.0f;
            for (int d = 0; d < HD; d++) sum += s_q[wave][d] * (float)kp[r * stride + d];
            x = sum * a.scale;
        }
        const float mn = fmaxf(m, wave_all(x, [](float p, float q) { return fmaxf(p, q); }));
        const float mz = mn == -INFINITY ? 0.0f : mn, corr = __expf(m - mz);
        const float p = r >= 0 ? __expf(x - mz) : 0.0f;
        l = l * corr + wave_total(p);
        m = mn;
        s_p[wave][lane] = p;
        s_row[wave][lane] = r;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < DPL; j++) o[j] *= corr;
        for (int i = 0; i < 64; i++) {
            const int ri = s_row[wave][i];
            if (ri < 0) continue;
            const float pi = s_p[wave][i];
#pragma unroll
            for (int j = 0; j < DPL; j++) o[j] += pi * (float)vp[ri * stride + lane + 64 * j];
        }
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int j = 0; j < DPL; j++)
        ((TQ *)a.out)[row * a.ldo + (int64_t)h * HD + lane + 64 * j] = (TQ)(m == -INFINITY ? o[j] + l : o[j] / l);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.nh + h] = m == -INFINITY && l == 0.0f ? -INFINITY : m + __logf(l);
}

int64_t attn_chunk_grid(int n_seq, int nkv, int gqa, int n_rows)
{
    return ((int64_t)n_rows * nkv * gqa + AC_WAVES - 1) / AC_WAVES;
}
uint64_t attn_chunk_ws_bytes(int n_seq, int nkv, int hd, int gqa, int n_rows) { return 16; }

template <typename TQ, typename TC> static void launch_hd(hipStream_t st, const AttnChunkArgs &a)
{
    const dim3 g((unsigned)attn_chunk_grid(a.kv.n_seq, a.kv.nkv, a.gqa, a.chunk.n_rows)), wg(AC_WG);
    switch (a.kv.hd) {
    case 64: hipLaunchKernelGGL((k_attn_chunk<TQ, TC, 64>), g, wg, 0, st, a); break;
    case 128: hipLaunchKernelGGL((k_attn_chunk<TQ, TC, 128>), g, wg, 0, st, a); break;
    default: hipLaunchKernelGGL((k_attn_chunk<TQ, TC, 256>), g, wg, 0, st, a); break;
    }
}
hipError_t launch_attn_chunk(hipStream_t st, AttnChunkArgs a, void *ws)
{
    if (!a.kv.f16)
        launch_hd<float, float>(st, a);
    else if (a.q_f16)
        launch_hd<_Float16, _Float16>(st, a);
    else
        launch_hd<float, _Float16>(st, a);
    return hipGetLastError();
}

}  // namespace styx
