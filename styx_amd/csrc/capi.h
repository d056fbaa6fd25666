// capi.h -- what the entry points of the C ABI share: their first lines, the
// current device, and the checks of a paged cache and of a workspace
// (capi.cpp, capi_chunk.cpp).
#pragma once

#include <string>

#include "attn_batch.h"
#include "runtime.h"

#define OP_GPU(g)                                                         \
    do {                                                                  \
        if (!(g)) return fail(STYX_E_INVALID, "NULL gpu");                \
    } while (0)
#define OP_RUN(expr, what)                                                \
    do {                                                                  \
        hipError_t _e = (expr);                                           \
        if (_e == hipErrorInvalidValue)                                   \
            return fail(STYX_E_INVALID, std::string(what) + ": unsupported shape or type"); \
        if (_e != hipSuccess) return hip_fail(_e, what);                  \
    } while (0)

namespace styx {

// The gpu's device current for a call, whatever device the caller has current.
struct DeviceScope {
    int before = -1, now;
    explicit DeviceScope(int device) : now(device)
    {
        if (hipGetDevice(&before) == hipSuccess && before != now) hipSetDevice(now);
    }
    ~DeviceScope()
    {
        if (before >= 0 && before != now) hipSetDevice(before);
    }
};

// A launch's workgroups times its threads stay below 2^32.
constexpr int64_t MAX_WG_256 = (1 << 24) - 1;

inline bool kv_shape_ok(const styx_kv_cache *kv)
{
    return kv && (kv->type == STYX_F32 || kv->type == STYX_F16) && kv->n_seq >= 1 && kv->nkv >= 1 &&
           (kv->hd == 64 || kv->hd == 128 || kv->hd == 256) && kv->page_tokens >= 1 && kv->n_pages >= 1 &&
           kv->table_len >= 1 && (int64_t)kv->table_len * kv->page_tokens <= (1 << 30) &&
           (int64_t)kv->n_pages * kv->page_tokens <= INT32_MAX && (int64_t)kv->n_seq * kv->nkv <= MAX_WG_256 / 4;
}

inline int kv_view(const styx_kv_cache *kv, KvView *v, const char *who)
{
    if (!kv_shape_ok(kv))
        return fail(STYX_E_INVALID, std::string(who) + ": unsupported cache type or shape");
    if (!kv->kpool || !kv->vpool || !kv->page_table)
        return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer in the cache");
    if (((uintptr_t)kv->kpool | (uintptr_t)kv->vpool) & 15)
        return fail(STYX_E_INVALID, std::string(who) + ": pools must be 16-byte aligned");
    *v = KvView{kv->kpool, kv->vpool, kv->page_table, kv->type == STYX_F16, kv->n_seq, kv->nkv, kv->hd,
                kv->page_tokens, kv->n_pages, kv->table_len, kv->table_len * kv->page_tokens,
                page_div((uint32_t)kv->page_tokens)};
    return STYX_OK;
}

inline int ws_ok(const void *ws, uint64_t have, uint64_t need, const char *who)
{
    if (!ws || have < need)
        return fail(STYX_E_INVALID, std::string(who) + ": workspace of " + std::to_string(have) + " bytes, " +
                                        std::to_string(need) + " needed");
    if ((uintptr_t)ws & 15) return fail(STYX_E_INVALID, std::string(who) + ": workspace must be 16-byte aligned");
    return STYX_OK;
}

}  // namespace styx
