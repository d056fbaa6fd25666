// kv_evict.hip -- the rows of least accumulated attention weight leave a
// batch's paged KV cache.
//
// Per sequence with n = len > trigger rows and kv head: the `keep` rows of
// the largest weight stay, rows of the `recent` newest positions and of the
// first `sinks` positions before all others, ties to the lower slot.  The
// attention does not ask in which order rows lie, so nothing is compacted:
// a row that leaves a slot below `keep` makes a hole, a row that stays at or
// past `keep` moves into one (both ascending), and no other row is touched.
// Sources and targets of the moves are apart, so they need no order among
// them and the call may be made again on the same lists.
//
// Bound: latency (a selection has to see all weights before its first
// move) and, for long caches, HBM: 8 bytes of weight and position per row
// read, 2 rows of K and V read and written per move.
#include <algorithm>

#include "attn_batch.h"

namespace styx {

constexpr int EV_WG = 1024, EV_WAVES = EV_WG / 64;
constexpr int MV_WG = 256, MV_SLOTS = 256;

// A row's key: weights in order, NaN below all; rows that stay anyway above all.
__device__ __forceinline__ uint32_t evict_key(const KvEvictArgs &a, int64_t base, int t, int64_t newest)
{
    const int64_t p = a.pos_in[base + t];
    const float w = a.acc_in[base + t] + 0.0f;  // -0 is 0
    if (p > newest - a.recent || p < a.sinks) return 0xFFFFFFFFu;
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Over a workgroup's threads in order: how many of those before this one
// have f set, and the total.  Every thread takes part.
struct Before {
    int rank, total;
};
__device__ __forceinline__ Before count_before(bool f, int *s)  // s [EV_WAVES]
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned long long m = __ballot(f);
    __syncthreads();
    if (lane == 0) s[wave] = __popcll(m);
    __syncthreads();
    Before r{(int)__popcll(m & ((1ull << lane) - 1)), 0};
    for (int w = 0; w < EV_WAVES; w++) {
        if (w < wave) r.rank += s[w];
        r.total += s[w];
    }
    return r;
}

// One workgroup per sequence and kv head: the keep-th largest key by a radix
// selection of 8 bits a pass, then holes and movers in slot order.
__global__ void __launch_bounds__(EV_WG) k_evict_select(KvEvictArgs a)
{
    __shared__ uint32_t hist[256];
    __shared__ int cnt[EV_WAVES];
    __shared__ uint32_t s_digit;
    __shared__ int s_above;
    const KvView &kv = a.kv;
    const int bk = blockIdx.x, b = bk / kv.nkv, n = a.len[b], tid = threadIdx.x;
    if (n <= a.trigger || n > kv.cap) return;
    const int64_t base = (int64_t)bk * kv.cap, newest = a.pos[b];
    uint32_t prefix = 0, mask = 0;
    int need = a.keep;  // the need-th largest of the keys that match the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += EV_WG) {
            const uint32_t k = evict_key(a, base, t, newest);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            int above = 0, d = 255;
            for (; d > 0 && above + (int)hist[d] < need; d--) above += hist[d];
            s_digit = d;
            s_above = above;
        }
        __syncthreads();
        prefix |= s_digit << shift;
        mask |= 255u << shift;
        need -= s_above;
        __syncthreads();
    }
    // keys above the prefix stay, and the first `need` that equal it
    int32_t *map = a.map + (int64_t)bk * a.keep, *holes = a.holes + (int64_t)bk * a.keep;
    int ties = 0, n_holes = 0, n_moved = 0;
    for (int t0 = 0; t0 < n; t0 += EV_WG) {
        const int t = t0 + tid;
        const uint32_t k = t < n ? evict_key(a, base, t, newest) : 0;
        const Before eq = count_before(t < n && k == prefix, cnt);
        const bool stays = t < n && (k > prefix || (k == prefix && ties + eq.rank < need));
        ties += eq.total;
        const bool hole = t < a.keep && !stays, mover = stays && t >= a.keep;
        const Before h = count_before(hole, cnt);
        if (hole) holes[n_holes + h.rank] = t;
        if (t < a.keep && stays) map[t] = t;
        n_holes += h.total;
        // (a mover's hole is below keep, so it has been written: in an
        // earlier round, or in this one before the barrier)
        const Before mv = count_before(mover, cnt);
        if (mover) map[holes[n_moved + mv.rank]] = t;
        n_moved += mv.total;
    }
}

// 256 places of one kv head: weights and positions, then the rows of the
// places whose row changes, one after another by a wave.
template <int ROW16>  // 16-byte pieces of a row
__global__ void __launch_bounds__(MV_WG) k_evict_move(KvEvictArgs a)
{
    const KvView &kv = a.kv;
    const int bk = blockIdx.x / a.copy_tiles, tile = blockIdx.x % a.copy_tiles;
    const int b = bk / kv.nkv, kvh = bk % kv.nkv, n = a.len[b];
    const bool act = n > a.trigger && n <= kv.cap;
    const int left = act ? a.keep : n > kv.cap ? 0 : n;
    const int lane = threadIdx.x & 63, s = tile * MV_SLOTS + threadIdx.x;
    if (tile * MV_SLOTS >= left) return;
    const int64_t base = (int64_t)bk * kv.cap;
    int src = s;
    if (s < left) {
        if (act) src = a.map[(int64_t)bk * a.keep + s];
        a.acc_out[base + s] = a.acc_in[base + src];
        a.pos_out[base + s] = a.pos_in[base + src];
    }
    const int32_t *tab = kv.table + (int64_t)b * kv.table_len;
    int from = -1, to = -1;
    if (src != s) {
        from = kv.row(tab, src);
        to = kv.row(tab, s);
    }
    unsigned long long todo = __ballot(from >= 0 && to >= 0);
    const int64_t stride = (int64_t)kv.nkv * ROW16;
    while (todo) {
        const int l = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int64_t f = __builtin_amdgcn_readlane(from, l) * stride + kvh * ROW16;
        const int64_t d = __builtin_amdgcn_readlane(to, l) * stride + kvh * ROW16;
        if (lane < ROW16) {
            const styx_u4 k = ((const styx_u4 *)kv.kpool)[f + lane], v = ((const styx_u4 *)kv.vpool)[f + lane];
            ((styx_u4 *)kv.kpool)[d + lane] = k;
            ((styx_u4 *)kv.vpool)[d + lane] = v;
        }
    }
}

// Last, when no workgroup reads the lengths any more: they may be the
// caller's own.
__global__ void __launch_bounds__(256) k_evict_len(KvEvictArgs a)
{
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= a.kv.n_seq) return;
    const int n = a.len[b];
    a.len_out[b] = n > a.trigger && n <= a.kv.cap ? a.keep : n;
}

static int copy_tiles(const KvEvictArgs &a)
{
    // sequences that stay as they are are copied only into other buffers
    const bool apart = a.acc_out != a.acc_in || a.pos_out != a.pos_in;
    const int most = apart && a.trigger > a.keep ? std::min(a.trigger, a.kv.cap) : a.keep;
    return (most - 1) / MV_SLOTS + 1;
}
int64_t kv_evict_grid(const KvEvictArgs &a) { return (int64_t)a.kv.n_seq * a.kv.nkv * copy_tiles(a); }

hipError_t launch_kv_evict(hipStream_t st, KvEvictArgs a, void *ws)
{
    const KvView &kv = a.kv;
    const int heads = kv.n_seq * kv.nkv;
    a.copy_tiles = copy_tiles(a);
    a.map = (int32_t *)ws;
    a.holes = a.map + (int64_t)heads * a.keep;
    hipLaunchKernelGGL(k_evict_select, dim3(heads), dim3(EV_WG), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)(heads * a.copy_tiles));
    switch (kv.hd * (kv.f16 ? 2 : 4) / 16) {
    case 8: hipLaunchKernelGGL(k_evict_move<8>, grid, dim3(MV_WG), 0, st, a); break;
    case 16: hipLaunchKernelGGL(k_evict_move<16>, grid, dim3(MV_WG), 0, st, a); break;
    case 32: hipLaunchKernelGGL(k_evict_move<32>, grid, dim3(MV_WG), 0, st, a); break;
    default: hipLaunchKernelGGL(k_evict_move<64>, grid, dim3(MV_WG), 0, st, a); break;
    }
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_evict_len, dim3((kv.n_seq + 255) / 256), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace styx
