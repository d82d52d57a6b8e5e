// s3e_kv.cpp — the entry points of the quantized key/value cache: checks of
// arguments and the split of attention over key ranges.  Nothing here
// allocates or synchronises.
#include <algorithm>
#include <cmath>

#include "k_kv.h"
#include "s3e_rt.h"

using namespace s3e;

namespace {

#define KV_HIP(expr)                                                  \
    do {                                                              \
        const hipError_t e_ = (expr);                                 \
        if (e_ != hipSuccess) {                                       \
            set_error("%s: %s", fn, hipGetErrorString(e_));           \
            return S3E_ERR_HIP;                                       \
        }                                                             \
    } while (0)

#define KV_REFUSE(status, ...)    \
    do {                          \
        set_error(__VA_ARGS__);   \
        return status;            \
    } while (0)

int check_cache(const char *fn, const s3e_kv_cache *c, bool data) {
    if (!c) KV_REFUSE(S3E_ERR_INVALID, "%s: NULL cache", fn);
    if (c->type != S3E_TYPE_Q4_0 && c->type != S3E_TYPE_Q8_0)
        KV_REFUSE(S3E_ERR_UNSUPPORTED, "%s: a cache of type %d (Q4_0 or Q8_0)", fn, c->type);
    const int D = c->head_dim;
    if (D != 32 && D != 64 && D != 96 && D != 128 && D != 256)
        KV_REFUSE(S3E_ERR_UNSUPPORTED, "%s: head dim %d (32, 64, 96, 128 or 256)", fn, D);
    if (c->page != 32 && c->page != 64 && c->page != 128 && c->page != 256)
        KV_REFUSE(S3E_ERR_UNSUPPORTED, "%s: pages of %d tokens (32, 64, 128 or 256)", fn, c->page);
    if (c->n_heads < 1 || c->n_heads > 65535) KV_REFUSE(S3E_ERR_INVALID, "%s: %d key/value heads", fn, c->n_heads);
    if (c->n_pages < 1 || c->n_pages > INT32_MAX / c->page)
        KV_REFUSE(S3E_ERR_INVALID, "%s: %lld pages of %d tokens", fn, (long long)c->n_pages, c->page);
    if (data && !c->data) KV_REFUSE(S3E_ERR_INVALID, "%s: the cache has no memory", fn);
    if ((uintptr_t)c->data % 16 != 0) KV_REFUSE(S3E_ERR_INVALID, "%s: the cache's memory must be 16-byte aligned", fn);
    return S3E_OK;
}

size_t cache_bytes(const s3e_kv_cache *c) {
    return (size_t)c->n_pages * (size_t)c->page * (size_t)c->n_heads * (size_t)c->head_dim / 8 *
           (c->type == S3E_TYPE_Q4_0 ? 9 : 17);
}

KvCache on_device(const s3e_kv_cache *c) {
    KvCache k;
    k.data = (uint8_t *)c->data;
    k.slots = c->n_pages * c->page;
    k.type = c->type;
    k.heads = c->n_heads;
    k.D = c->head_dim;
    while ((1 << k.page_shift) < c->page) k.page_shift++;
    return k;
}

// Rows of a call: a grid's threads along one dimension stay below 2^32.
constexpr int64_t KV_MAX_ROWS = 1 << 29;

int check_type(const char *fn, int type) {
    if (type != S3E_TYPE_F32 && type != S3E_TYPE_F16) KV_REFUSE(S3E_ERR_UNSUPPORTED, "%s: rows of type %d (F32 or F16)", fn, type);
    return S3E_OK;
}

// n rows of `heads` times D values by element strides: whether they lie on their
// type's alignment, whether 16-byte loads may read them, and the bytes from the
// first to the last.
int check_rows(const char *fn, const char *what, const void *p, const int64_t nb[2], int64_t n, int64_t heads, int64_t D,
               int64_t esize, int *vec, size_t *bytes) {
    if (nb[0] < 0 || nb[1] < 0) KV_REFUSE(S3E_ERR_INVALID, "%s: a negative stride of %s", fn, what);
    if ((uintptr_t)p % (uintptr_t)esize != 0) KV_REFUSE(S3E_ERR_INVALID, "%s: %s is not aligned to its type", fn, what);
    const __int128 span = n <= 0 ? 0 : ((__int128)(n - 1) * nb[0] + (__int128)(heads - 1) * nb[1] + D) * esize;
    if (span > INT64_MAX) KV_REFUSE(S3E_ERR_INVALID, "%s: strides of %s past any memory", fn, what);
    // (a stride that no row takes says nothing)
    const bool rows_vec = n <= 1 || nb[0] * esize % 16 == 0, heads_vec = heads <= 1 || nb[1] * esize % 16 == 0;
    *vec = (uintptr_t)p % 16 == 0 && rows_vec && heads_vec;
    *bytes = (size_t)span;
    return S3E_OK;
}

bool meets(const void *a, size_t an, const void *b, size_t bn) {
    return an && bn && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

int check_batch(const char *fn, const s3e_kv_cache *c, const s3e_kv_batch *b, int64_t nh) {
    if (!b) KV_REFUSE(S3E_ERR_INVALID, "%s: NULL batch", fn);
    if (nh < 1 || nh > 65535 || nh % c->n_heads != 0)
        KV_REFUSE(S3E_ERR_INVALID, "%s: %lld query heads on %d key/value heads", fn, (long long)nh, c->n_heads);
    if (b->n_seq < 0 || b->n_seq > 65535 || b->n_tokens < 0 || b->max_q < 0 || b->max_kv < 0 || b->pages_ld < 0)
        KV_REFUSE(S3E_ERR_INVALID, "%s: a count of the batch is negative or has over 65535 sequences", fn);
    if (b->n_tokens > INT32_MAX / nh || b->max_q > INT32_MAX / nh)
        KV_REFUSE(S3E_ERR_INVALID, "%s: %lld rows of %lld heads", fn, (long long)std::max(b->n_tokens, b->max_q), (long long)nh);
    if (b->pages_ld > INT32_MAX || b->max_kv > b->pages_ld * c->page || b->max_kv > 1 << 30)
        KV_REFUSE(S3E_ERR_INVALID, "%s: %lld keys in rows of %lld pages of %d", fn, (long long)b->max_kv,
                  (long long)b->pages_ld, c->page);
    return S3E_OK;
}

// Fewest keys a work-group is worth starting for (µs at 128, 256, 512, 1024: one
// query over 4096 keys of 16 heads of 64 10.0, 9.6, 11.2, 13.3; 7 × 5 in fp32
// under a mask over up to 1733 19.7, 21.3, 26.3, 37.0).
constexpr int64_t KV_MIN_KEYS = 256;

// The kernel, its column tiles and the split over keys: by the host's bounds
// alone, so that a captured call is the same for any lengths.
void plan(const s3e_kv_cache *c, const s3e_kv_batch *b, int64_t nh, bool f32, KvAttnArgs &a) {
    a.n_seq = (int)b->n_seq;
    a.c.type = c->type;
    const int64_t G = nh / c->n_heads;
    kv_attn_columns(a, c->head_dim, f32, std::min(b->max_q, b->n_tokens) * G, b->n_tokens * G);
    const int64_t wgs = c->n_heads * (a.tiles ? a.tiles : b->n_seq * a.ctiles);
    // (to the nearest: 64 sequences of up to 4096 keys, 16 heads of 64, Q8_0, whose
    // 1024 work-groups are two thirds of the goal, take 64 µs in one range, 70 in two)
    int64_t ns = (a.goal + (a.tile ? 0 : (wgs - 1) / 2)) / wgs;
    ns = std::max<int64_t>(1, std::min(ns, (b->max_kv + KV_MIN_KEYS - 1) / KV_MIN_KEYS));
    a.chunk = std::max<int64_t>(128, round_up((b->max_kv + ns - 1) / ns, 128));
    a.nsplit = (int)std::max<int64_t>(1, (b->max_kv + a.chunk - 1) / a.chunk);
}

size_t partial_bytes(const s3e_kv_cache *c, const s3e_kv_batch *b, int64_t nh, const KvAttnArgs &a) {
    return a.nsplit > 1 ? (size_t)a.nsplit * (size_t)b->n_tokens * (size_t)nh * (size_t)(c->head_dim + 2) * 4 : 0;
}

}  // namespace

extern "C" int s3e_kv_cache_bytes(const s3e_kv_cache *c, size_t *bytes) try {
    if (!bytes) { set_error("s3e_kv_cache_bytes: NULL argument"); return S3E_ERR_INVALID; }
    const int rc = check_cache("s3e_kv_cache_bytes", c, false);
    if (rc == S3E_OK) *bytes = cache_bytes(c);
    return rc;
} S3E_CATCH("s3e_kv_cache_bytes")

extern "C" int s3e_kv_write(s3e_ctx *ctx, const s3e_kv_cache *c, int type, const void *k, const int64_t k_nb[2],
                            const void *v, const int64_t v_nb[2], const int32_t *slots, int64_t n) try {
    const char *fn = "s3e_kv_write";
    if (!ctx || !k || !k_nb || !v || !v_nb || !slots) { set_error("%s: NULL argument", fn); return S3E_ERR_INVALID; }
    int rc = check_cache(fn, c, true);
    if (rc == S3E_OK) rc = check_type(fn, type);
    if (rc != S3E_OK) return rc;
    if (n < 0 || n > KV_MAX_ROWS) { set_error("%s: %lld rows", fn, (long long)n); return S3E_ERR_INVALID; }
    KvWriteArgs a;
    const int64_t esize = type == S3E_TYPE_F32 ? 4 : 2;
    size_t k_bytes = 0, v_bytes = 0;
    rc = check_rows(fn, "k", k, k_nb, n, c->n_heads, c->head_dim, esize, &a.vec[0], &k_bytes);
    if (rc == S3E_OK) rc = check_rows(fn, "v", v, v_nb, n, c->n_heads, c->head_dim, esize, &a.vec[1], &v_bytes);
    if (rc != S3E_OK) return rc;
    if (n == 0) return S3E_OK;
    const size_t cb = cache_bytes(c);
    if (meets(k, k_bytes, c->data, cb) || meets(v, v_bytes, c->data, cb) || meets(slots, (size_t)n * 4, c->data, cb)) {
        set_error("%s: k, v or slots overlap the cache", fn);
        return S3E_ERR_INVALID;
    }
    a.x[0] = k, a.x[1] = v;
    a.st[0] = k_nb[0], a.sh[0] = k_nb[1];
    a.st[1] = v_nb[0], a.sh[1] = v_nb[1];
    a.slots = slots;
    a.n = (int)n;
    a.c = on_device(c);
    KV_HIP(hipSetDevice(ctx->device));
    KV_HIP(launch_kv_write(a, type == S3E_TYPE_F32, ctx->stream));
    return S3E_OK;
} S3E_CATCH("s3e_kv_write")

extern "C" int s3e_kv_read(s3e_ctx *ctx, const s3e_kv_cache *c, const int32_t *slots, int64_t n, int type, void *k,
                           void *v) try {
    const char *fn = "s3e_kv_read";
    if (!ctx || !slots || (!k && !v)) { set_error("%s: NULL argument", fn); return S3E_ERR_INVALID; }
    int rc = check_cache(fn, c, true);
    if (rc == S3E_OK) rc = check_type(fn, type);
    if (rc != S3E_OK) return rc;
    if (n < 0 || n > KV_MAX_ROWS) { set_error("%s: %lld rows", fn, (long long)n); return S3E_ERR_INVALID; }
    if ((uintptr_t)k % 16 != 0 || (uintptr_t)v % 16 != 0) { set_error("%s: k and v must be 16-byte aligned", fn); return S3E_ERR_INVALID; }
    if (n == 0) return S3E_OK;
    const size_t cb = cache_bytes(c), yb = (size_t)n * c->n_heads * c->head_dim * (type == S3E_TYPE_F32 ? 4 : 2);
    const size_t kb = k ? yb : 0, vb = v ? yb : 0;
    if (meets(k, kb, v, vb) || meets(k, kb, c->data, cb) || meets(v, vb, c->data, cb) || meets(k, kb, slots, (size_t)n * 4) ||
        meets(v, vb, slots, (size_t)n * 4)) {
        set_error("%s: k and v overlap each other, the cache or the slots", fn);
        return S3E_ERR_INVALID;
    }
    KvReadArgs a;
    a.y[0] = k, a.y[1] = v;
    a.slots = slots;
    a.n = (int)n;
    a.c = on_device(c);
    KV_HIP(hipSetDevice(ctx->device));
    KV_HIP(launch_kv_read(a, type == S3E_TYPE_F32, ctx->stream));
    return S3E_OK;
} S3E_CATCH("s3e_kv_read")

extern "C" int s3e_kv_attn_workspace(const s3e_kv_cache *c, const s3e_kv_batch *b, int64_t nh, int type,
                                     size_t *bytes) try {
    const char *fn = "s3e_kv_attn_workspace";
    if (!bytes) { set_error("%s: NULL argument", fn); return S3E_ERR_INVALID; }
    int rc = check_cache(fn, c, false);
    if (rc == S3E_OK) rc = check_type(fn, type);
    if (rc == S3E_OK) rc = check_batch(fn, c, b, nh);
    if (rc != S3E_OK) return rc;
    *bytes = 0;
    if (b->n_seq == 0 || b->n_tokens == 0 || b->max_q == 0) return S3E_OK;
    KvAttnArgs a;
    plan(c, b, nh, type == S3E_TYPE_F32, a);
    *bytes = partial_bytes(c, b, nh, a);
    return S3E_OK;
} S3E_CATCH("s3e_kv_attn_workspace")

extern "C" int s3e_kv_attn(s3e_ctx *ctx, const s3e_kv_cache *c, const s3e_kv_batch *b, int type, const void *q,
                           const int64_t q_nb[2], int64_t nh, float scale, int causal, const uint16_t *mask,
                           int64_t mask_ld, void *o, void *ws, size_t ws_bytes) try {
    const char *fn = "s3e_kv_attn";
    if (!ctx || !q || !q_nb || !o) { set_error("%s: NULL argument", fn); return S3E_ERR_INVALID; }
    int rc = check_cache(fn, c, true);
    if (rc == S3E_OK) rc = check_type(fn, type);
    if (rc == S3E_OK) rc = check_batch(fn, c, b, nh);
    if (rc != S3E_OK) return rc;
    if (!std::isfinite(scale)) { set_error("%s: the scale is not finite", fn); return S3E_ERR_INVALID; }
    const bool f32 = type == S3E_TYPE_F32;
    const int64_t esize = f32 ? 4 : 2;
    KvAttnArgs a;
    const int64_t D = c->head_dim;
    size_t qb = 0;
    rc = check_rows(fn, "q", q, q_nb, b->n_tokens, nh, D, esize, &a.q_vec, &qb);
    if (rc != S3E_OK) return rc;
    if ((uintptr_t)o % 16 != 0) { set_error("%s: o must be 16-byte aligned", fn); return S3E_ERR_INVALID; }
    if (mask && (mask_ld < b->max_kv || (uintptr_t)mask % 2 != 0)) {
        set_error("%s: mask rows of %lld for %lld keys, or a mask that is not 2-byte aligned", fn, (long long)mask_ld, (long long)b->max_kv);
        return S3E_ERR_INVALID;
    }
    if (b->n_seq == 0 || b->n_tokens == 0 || b->max_q == 0) return S3E_OK;
    if (!b->q_start || !b->kv_len || !b->pages) { set_error("%s: the batch lacks an array", fn); return S3E_ERR_INVALID; }
    const size_t ob = (size_t)(b->n_tokens * nh * D * esize);
    const __int128 mask_span = mask ? ((__int128)(b->n_tokens - 1) * mask_ld + b->max_kv) * 2 : 0;
    if (mask_span > INT64_MAX) { set_error("%s: mask rows of %lld past any memory", fn, (long long)mask_ld); return S3E_ERR_INVALID; }
    const bool in_place = o == q && q_nb[0] == nh * D && (nh == 1 || q_nb[1] == D);
    if (!in_place && meets(o, ob, q, qb)) { set_error("%s: o overlaps q", fn); return S3E_ERR_INVALID; }
    if (meets(o, ob, c->data, cache_bytes(c))) { set_error("%s: o overlaps the cache", fn); return S3E_ERR_INVALID; }
    // what every work-group reads stays as it is
    struct { const void *p; size_t n; } read[] = {{mask, (size_t)mask_span}, {b->q_start, (size_t)(b->n_seq + 1) * 4},
                                                  {b->kv_len, (size_t)b->n_seq * 4}, {b->pages, (size_t)(b->n_seq * b->pages_ld) * 4}};
    for (const auto &r : read)
        if (meets(o, ob, r.p, r.n)) { set_error("%s: o overlaps the mask or an array of the batch", fn); return S3E_ERR_INVALID; }
    plan(c, b, nh, f32, a);
    const size_t need = partial_bytes(c, b, nh, a);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16 != 0)) {
        set_error("%s: needs %zu bytes of 16-byte aligned workspace, has %zu", fn, need, ws ? ws_bytes : (size_t)0);
        return S3E_ERR_INVALID;
    }
    if (need && (meets(ws, need, o, ob) || meets(ws, need, q, qb) || meets(ws, need, c->data, cache_bytes(c)))) {
        set_error("%s: the workspace overlaps q, o or the cache", fn);
        return S3E_ERR_INVALID;
    }
    for (const auto &r : read)
        if (meets(ws, need, r.p, r.n)) { set_error("%s: the workspace overlaps the mask or an array of the batch", fn); return S3E_ERR_INVALID; }
    a.c = on_device(c);
    a.q = q;
    a.q_st = q_nb[0], a.q_sh = q_nb[1];
    a.q_start = b->q_start, a.kv_len = b->kv_len, a.pages = b->pages;
    a.pages_ld = b->pages_ld;
    a.mask = (const _Float16 *)mask;
    a.mask_ld = mask_ld;
    a.mask_vec = (uintptr_t)mask % 16 == 0 && mask_ld % 8 == 0;
    a.o = o;
    a.sign = scale < 0 ? -1 : (scale > 0 ? 1 : 0);
    // (in log2 units, neither zero nor infinite: a score of 0 stays 0)
    a.scale = a.sign ? (float)std::min(std::max(std::fabs((double)scale) * 1.4426950408889634, 1.17549435e-38), 3.40282347e38) : 1.0f;
    a.causal = causal != 0;
    a.n_tokens = (int)b->n_tokens;
    a.max_q = (int)std::min(b->max_q, b->n_tokens);
    a.nh = (int)nh;
    a.max_kv = b->max_kv;
    if (need) {
        a.part_o = (float *)ws;
        a.part_ml = a.part_o + (size_t)a.nsplit * (size_t)b->n_tokens * (size_t)nh * (size_t)D;
    }
    KV_HIP(hipSetDevice(ctx->device));
    KV_HIP(c->type == S3E_TYPE_Q4_0 ? launch_kv_attn_q4(a, f32, ctx->stream) : launch_kv_attn_q8(a, f32, ctx->stream));
    if (a.nsplit > 1) KV_HIP(launch_kv_combine(a, f32, ctx->stream));
    return S3E_OK;
} S3E_CATCH("s3e_kv_attn")
