// kv_weigh.hip -- the attention weights of the last tokens of each sequence's
// chunk, added to the accumulator by which rows are evicted.
//
//   acc_out[j][t] = decay acc_in[j][t] (0 for the new rows)
//                 + sum over the last tokens i that see t and the heads h of j
//                   of e^(scale q_ih . K[t] - lse_ih),  t < len + count
//
// The plain kernel: a wave for 64 slots of a kv head, a slot a lane, the tokens
// and heads one after another.
#include <algorithm>

#include "kv_chunk.h"
#include "lanes.h"

namespace styx {

constexpr int KW_WG = 256, KW_WAVES = KW_WG / 64;

template <typename TQ, typename TC, int HD>
__global__ void __launch_bounds__(KW_WG) k_kv_weigh(KvWeighArgs a, int tiles)
{
    const KvView &kv = a.kv;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bk = blockIdx.x / tiles, b = bk / kv.nkv, kvh = bk % kv.nkv;
    const ChunkSeq s = chunk_seq(a.chunk, kv, b);
    if (s.count == 0) return;
    const int rows = s.len + s.count;
    const int32_t *tab = kv.table + (int64_t)b * kv.table_len;
    const int64_t stride = (int64_t)kv.nkv * HD, base = (int64_t)bk * kv.cap;
    for (int64_t t64 = ((int64_t)(blockIdx.x % tiles) * KW_WAVES + wave) * 64; t64 < rows; t64 += (int64_t)tiles * KW_WG) {
        const int t = (int)t64 + lane, r = t < rows ? kv.row(tab, t) : -1;
        const TC *k = (const TC *)kv.kpool + max(r, 0) * stride + kvh * HD;
        float sum = 0.0f;
        for (int i = max(0, s.count - a.last); i < s.count; i++) {
            const int at = s.len + i;
            if (t > at || (a.window && t <= at - a.window) || r < 0) continue;
            for (int g = 0; g < a.gqa; g++) {
                const int h = kvh * a.gqa + g, row = s.first + i;
                const TQ *q = (const TQ *)a.q + row * a.ldq + (int64_t)h * HD;
                float x = 0.0f;
                for (int d = 0; d < HD; d++) x += (float)q[d] * (float)k[d];
                const float lse = a.lse[(int64_t)row * a.nh + h];
                if (lse != -INFINITY) sum += __expf(x * a.scale - lse);
            }
        }
        if (t >= rows) continue;
        a.acc_out[base + t] = (a.acc_in && t < s.len ? a.decay * a.acc_in[base + t] : 0.0f) + sum;
        if (a.slot_pos && t >= s.len) a.slot_pos[base + t] = a.pos[b] + (t - s.len);
    }
}

static int64_t weigh_tiles(const KvWeighArgs &a)
{
    return std::min<int64_t>(((int64_t)a.kv.cap + KW_WG - 1) / KW_WG,
                             std::max<int64_t>(1, 4096 / ((int64_t)a.kv.n_seq * a.kv.nkv)));
}
int64_t kv_weigh_grid(const KvWeighArgs &a) { return weigh_tiles(a) * a.kv.n_seq * a.kv.nkv; }

template <typename TQ, typename TC> static void launch_hd(hipStream_t st, const KvWeighArgs &a)
{
    const dim3 g((unsigned)kv_weigh_grid(a)), wg(KW_WG);
    const int tiles = (int)weigh_tiles(a);
    switch (a.kv.hd) {
    case 64: hipLaunchKernelGGL((k_kv_weigh<TQ, TC, 64>), g, wg, 0, st, a, tiles); break;
    case 128: hipLaunchKernelGGL((k_kv_weigh<TQ, TC, 128>), g, wg, 0, st, a, tiles); break;
    default: hipLaunchKernelGGL((k_kv_weigh<TQ, TC, 256>), g, wg, 0, st, a, tiles); break;
    }
}
hipError_t launch_kv_weigh(hipStream_t st, KvWeighArgs a)
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
