// capi_chunk.cpp -- C ABI of the operators that bring new tokens of a batch
// into its paged KV cache (no counterpart in the reference, which decodes one
// sequence into a cache of fixed length).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "capi.h"
#include "kv_chunk.h"

using namespace styx;

static int chunk_view(const styx_kv_chunk *c, ChunkView *v, const char *who)
{
    if (!c || c->n_rows < 0) return fail(STYX_E_INVALID, std::string(who) + ": bad chunk");
    if (!c->first || !c->count || !c->len) return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer in the chunk");
    *v = ChunkView{c->n_rows, c->first, c->count, c->len};
    return STYX_OK;
}

// Rows of `heads` heads of hd values of a type, ld values apart: 16-byte pieces.
static int rows_ok(const void *p, int type, int64_t ld, int64_t width, const char *name, const char *who)
{
    const int64_t bytes = type == STYX_F16 ? 2 : 4;
    if (ld < width || ld > INT32_MAX)
        return fail(STYX_E_INVALID, std::string(who) + ": rows of " + name + " are " + std::to_string(ld) +
                                        " values apart, " + std::to_string(width) + " each");
    if (((uintptr_t)p | (uintptr_t)(ld * bytes)) & 15)
        return fail(STYX_E_INVALID, std::string(who) + ": rows of " + name + " must be 16-byte aligned");
    return STYX_OK;
}

static int heads_ok(const styx_kv_cache *kv, int nh, int type_q, const char *who)
{
    if (nh < 1 || nh % kv->nkv || nh / kv->nkv > 16)
        return fail(STYX_E_INVALID, std::string(who) + ": nh must be 1 to 16 times nkv");
    if (type_q != STYX_F32 && !(type_q == STYX_F16 && kv->type == STYX_F16))
        return fail(STYX_E_INVALID, std::string(who) + ": q must be f32, or f16 with an f16 cache");
    return STYX_OK;
}

extern "C" {

int styx_rope_table_scaled(float base, int n_rot, int n_pos, const styx_rope_scaling *s, double *out)
{
    const char *who = "styx_rope_table_scaled";
    if (!out || n_rot < 2 || n_rot % 2 || n_pos < 1 || !(base > 0.0f) || !std::isfinite(base))
        return fail(STYX_E_INVALID, std::string(who) + ": bad table, base or sizes");
    styx_rope_scaling z{};
    if (s) z = *s;
    if (z.kind < STYX_ROPE_PLAIN || z.kind > STYX_ROPE_BANDS) return fail(STYX_E_INVALID, std::string(who) + ": unknown kind");
    if (z.kind != STYX_ROPE_PLAIN && !(z.factor > 0.0f && std::isfinite(z.factor)))
        return fail(STYX_E_INVALID, std::string(who) + ": factor must be above 0");
    if (z.kind == STYX_ROPE_BASE && n_rot < 4) return fail(STYX_E_INVALID, std::string(who) + ": a stretched base needs two pairs");
    const bool two = z.kind == STYX_ROPE_PARTS || z.kind == STYX_ROPE_BANDS;
    const double fast = z.fast != 0.0f ? z.fast : z.kind == STYX_ROPE_PARTS ? 32.0 : 4.0, slow = z.slow != 0.0f ? z.slow : 1.0;
    if (two && (z.n_orig < 1 || !(fast > slow && slow > 0.0) || !std::isfinite(fast)))
        return fail(STYX_E_INVALID, std::string(who) + ": needs n_orig and fast > slow > 0");
    if (z.kind == STYX_ROPE_PARTS && !(base > 1.0f)) return fail(STYX_E_INVALID, std::string(who) + ": base must be above 1");
    if (!std::isfinite(z.gain)) return fail(STYX_E_INVALID, std::string(who) + ": gain must be finite");

    const int half = n_rot / 2;
    const double pi2 = 6.283185307179586476925286766559, factor = z.factor;
    double b = base, gain = z.gain != 0.0f ? z.gain : 1.0;
    if (z.kind == STYX_ROPE_BASE) b = base * std::pow(factor, (double)n_rot / (n_rot - 2));
    const double ts = std::pow(b, -2.0 / (double)n_rot);
    double low = 0.0, high = 0.0;  // PARTS: the ramp's pairs
    if (z.kind == STYX_ROPE_PARTS) {
        // the pair that makes `turns` turns over n_orig positions
        auto pair_of = [&](double turns) { return n_rot * std::log(z.n_orig / (turns * pi2)) / (2.0 * std::log(b)); };
        low = std::max(0.0, std::floor(pair_of(fast)));
        high = std::min(n_rot - 1.0, std::ceil(pair_of(slow)));
        if (high <= low) high = low + 0.001;  // a step
        if (z.gain == 0.0f && factor > 1.0) gain = 0.1 * std::log(factor) + 1.0;
    }
    // The frequencies lie in the table's first row until that, the last, is
    // written: there is no other memory, whose allocation could throw.
    for (int i = 0; i < half; i++) {
        double f = std::pow(ts, (double)i);
        if (z.kind == STYX_ROPE_LINEAR) f /= factor;
        if (z.kind == STYX_ROPE_PARTS) {
            const double r = std::min(1.0, std::max(0.0, (i - low) / (high - low)));
            f = f * (1.0 - r) + f / factor * r;
        }
        if (z.kind == STYX_ROPE_BANDS) {
            const double turns = z.n_orig * f / pi2;
            const double r = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            f = f / factor * (1.0 - r) + f * r;
        }
        out[(size_t)i * 2] = f;
    }
    for (int p = n_pos - 1; p >= 0; p--)
        for (int i = 0; i < half; i++) {
            const double th = (double)p * out[(size_t)i * 2];
            out[((size_t)p * half + i) * 2] = gain * std::cos(th);
            out[((size_t)p * half + i) * 2 + 1] = gain * std::sin(th);
        }
    return STYX_OK;
}

int styx_op_kv_plan(styx_gpu *g, const styx_kv_cache *kv, const styx_kv_pages *in, const styx_kv_pages *out,
                    const int32_t *shared, const int32_t *len, const int32_t *n_new, const int32_t *pos, int n_rows,
                    int32_t *first, int32_t *count, int32_t *row_seq, int32_t *row_pos, int32_t *row_at)
{
    const char *who = "styx_op_kv_plan";
    OP_GPU(g);
    if (!kv_shape_ok(kv)) return fail(STYX_E_INVALID, std::string(who) + ": unsupported cache type or shape");
    for (const styx_kv_pages *p : {in, out})
        if (!p || !p->page_table || !p->held || !p->free_pages || !p->n_free)
            return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer in the pages");
    const int same = (in->page_table == out->page_table) + (in->held == out->held) +
                     (in->free_pages == out->free_pages) + (in->n_free == out->n_free);
    if (same != 0 && same != 4)
        return fail(STYX_E_INVALID, std::string(who) + ": all arrays of the pages in place, or none");
    if (!len || !n_new || !first || !count || (row_pos && !pos)) return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer");
    if (n_rows < 0) return fail(STYX_E_INVALID, std::string(who) + ": n_rows must not be negative");
    if ((int64_t)kv->n_seq * kv->table_len > INT32_MAX)
        return fail(STYX_E_INVALID, std::string(who) + ": more than 2^31 page-table entries");
    KvPlanArgs a{};
    a.kv = KvView{nullptr, nullptr, nullptr, 0, kv->n_seq, kv->nkv, kv->hd, kv->page_tokens, kv->n_pages,
                  kv->table_len, kv->table_len * kv->page_tokens, page_div((uint32_t)kv->page_tokens)};
    a.in = KvPages{in->page_table, in->held, in->free_pages, in->n_free};
    a.out = KvPages{out->page_table, out->held, out->free_pages, out->n_free};
    a.shared = shared;
    a.len = len;
    a.n_new = n_new;
    a.pos = pos;
    a.n_rows = n_rows;
    a.first = first;
    a.count = count;
    a.row_seq = row_seq;
    a.row_pos = row_pos;
    a.row_at = row_at;
    if (kv_plan_grid(a) > MAX_WG_256) return fail(STYX_E_INVALID, std::string(who) + ": too many sequences, rows or pages");
    const DeviceScope on(g->device);
    OP_RUN(launch_kv_plan(g->stream, a), who);
    return STYX_OK;
}

int styx_op_kv_append(styx_gpu *g, const styx_kv_cache *kv, int n_rows, const int32_t *row_pos, const int32_t *row_at,
                      int nh, int type_in, const void *q, int64_t ldq, const void *k, int64_t ldk, const void *v,
                      int64_t ldv, const float *q_norm, const float *k_norm, float eps, const styx_rope *rope,
                      int type_q, void *q_out, int64_t ldo)
{
    const char *who = "styx_op_kv_append";
    OP_GPU(g);
    KvAppendArgs a{};
    if (int r = kv_view(kv, &a.kv, who)) return r;
    auto is_f = [](int t) { return t == STYX_F32 || t == STYX_F16; };
    if (!is_f(type_in) || !is_f(type_q)) return fail(STYX_E_INVALID, std::string(who) + ": rows must be f32 or f16");
    if (n_rows < 0) return fail(STYX_E_INVALID, std::string(who) + ": n_rows must not be negative");
    if (!q != !q_out || !k != !v || (!q && !k))
        return fail(STYX_E_INVALID, std::string(who) + ": q goes with q_out and k with v, and one pair must be there");
    if ((k && !row_at) || (rope && !row_pos)) return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer");
    if (rope && (!rope->table || rope->n_pos < 1 || rope->n_rot < 2 || rope->n_rot % 2 || rope->n_rot > kv->hd ||
                 ((uintptr_t)rope->table & 15)))
        return fail(STYX_E_INVALID, std::string(who) + ": bad rope table");
    const int64_t kw = (int64_t)kv->nkv * kv->hd, qw = (int64_t)nh * kv->hd;
    if (q) {
        if (nh < 1 || nh > 65536) return fail(STYX_E_INVALID, std::string(who) + ": nh must be 1 to 65536");
        if (int r = rows_ok(q, type_in, ldq, qw, "q", who)) return r;
        if (int r = rows_ok(q_out, type_q, ldo, qw, "q_out", who)) return r;
        if (q == q_out && (type_in != type_q || ldq != ldo))
            return fail(STYX_E_INVALID, std::string(who) + ": q in place needs one type and row length");
    }
    if (k) {
        if (int r = rows_ok(k, type_in, ldk, kw, "k", who)) return r;
        if (int r = rows_ok(v, type_in, ldv, kw, "v", who)) return r;
    }
    a.n_rows = n_rows;
    a.nh = q ? nh : 0;
    a.row_pos = row_pos;
    a.row_at = row_at;
    a.in_f16 = type_in == STYX_F16;
    a.q_f16 = type_q == STYX_F16;
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.ldo = ldo;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    if (rope) {
        a.rope = (const double2 *)rope->table;
        a.n_pos = rope->n_pos;
        a.n_rot = rope->n_rot;
        a.interleaved = rope->interleaved != 0;
    }
    a.q_out = q_out;
    if (kv_append_grid(a) > MAX_WG_256) return fail(STYX_E_INVALID, std::string(who) + ": too many rows or heads");
    if (n_rows == 0) return STYX_OK;
    const DeviceScope on(g->device);
    OP_RUN(launch_kv_append(g->stream, a), who);
    return STYX_OK;
}

uint64_t styx_op_attn_chunk_ws_bytes(const styx_kv_cache *kv, int n_rows, int nh)
{
    if (!kv_shape_ok(kv) || nh < 1 || nh % kv->nkv || nh / kv->nkv > 16 || n_rows < 0) return 0;
    if (attn_chunk_grid(kv->n_seq, kv->nkv, nh / kv->nkv, n_rows) > MAX_WG_256) return 0;
    return attn_chunk_ws_bytes(kv->n_seq, kv->nkv, kv->hd, nh / kv->nkv, n_rows);
}

int styx_op_attn_chunk(styx_gpu *g, const styx_kv_cache *kv, const styx_kv_chunk *chunk, int nh, int type_q,
                       const void *q, int64_t ldq, float scale, int window, void *out, int64_t ldo, float *lse,
                       void *ws, uint64_t ws_bytes)
{
    const char *who = "styx_op_attn_chunk";
    OP_GPU(g);
    AttnChunkArgs a{};
    if (int r = kv_view(kv, &a.kv, who)) return r;
    if (int r = chunk_view(chunk, &a.chunk, who)) return r;
    if (int r = heads_ok(kv, nh, type_q, who)) return r;
    if (!q || !out) return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer");
    if (window < 0) return fail(STYX_E_INVALID, std::string(who) + ": window must not be negative");
    if (int r = rows_ok(q, type_q, ldq, (int64_t)nh * kv->hd, "q", who)) return r;
    if (int r = rows_ok(out, type_q, ldo, (int64_t)nh * kv->hd, "out", who)) return r;
    const uint64_t need = styx_op_attn_chunk_ws_bytes(kv, chunk->n_rows, nh);
    if (!need) return fail(STYX_E_INVALID, std::string(who) + ": too many sequences, heads or rows");
    if (int r = ws_ok(ws, ws_bytes, need, who)) return r;
    a.nh = nh;
    a.gqa = nh / kv->nkv;
    a.q_f16 = type_q == STYX_F16;
    a.window = window < a.kv.cap ? window : 0;  // (all of a sequence: none)
    a.q = q;
    a.ldq = ldq;
    a.ldo = ldo;
    a.scale = scale;
    a.out = out;
    a.lse = lse;
    if (chunk->n_rows == 0) return STYX_OK;
    const DeviceScope on(g->device);
    OP_RUN(launch_attn_chunk(g->stream, a, ws), who);
    return STYX_OK;
}

int styx_op_kv_weigh(styx_gpu *g, const styx_kv_cache *kv, const styx_kv_chunk *chunk, const int32_t *pos, int nh,
                     int type_q, const void *q, int64_t ldq, float scale, int window, const float *lse, int last,
                     float decay, const float *acc_in, float *acc_out, int32_t *slot_pos)
{
    const char *who = "styx_op_kv_weigh";
    OP_GPU(g);
    KvWeighArgs a{};
    if (int r = kv_view(kv, &a.kv, who)) return r;
    if (int r = chunk_view(chunk, &a.chunk, who)) return r;
    if (int r = heads_ok(kv, nh, type_q, who)) return r;
    if (!q || !lse || !acc_out || (slot_pos && !pos)) return fail(STYX_E_INVALID, std::string(who) + ": NULL pointer");
    if (window < 0 || last < 0) return fail(STYX_E_INVALID, std::string(who) + ": window and last must not be negative");
    if (int r = rows_ok(q, type_q, ldq, (int64_t)nh * kv->hd, "q", who)) return r;
    a.pos = pos;
    a.nh = nh;
    a.gqa = nh / kv->nkv;
    a.q_f16 = type_q == STYX_F16;
    a.window = window < a.kv.cap ? window : 0;  // (all of a sequence: none)
    a.last = last;
    a.q = q;
    a.ldq = ldq;
    a.scale = scale;
    a.decay = decay;
    a.lse = lse;
    a.acc_in = acc_in;
    a.acc_out = acc_out;
    a.slot_pos = slot_pos;
    if ((int64_t)chunk->n_rows * a.gqa > (1 << 28) || kv_weigh_grid(a) > MAX_WG_256) return fail(STYX_E_INVALID, std::string(who) + ": too many sequences, heads, rows or slots");
    if (chunk->n_rows == 0) return STYX_OK;
    const DeviceScope on(g->device);
    OP_RUN(launch_kv_weigh(g->stream, a), who);
    return STYX_OK;
}

}  // extern "C"
