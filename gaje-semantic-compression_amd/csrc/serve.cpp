// C entry points of the serving operators: their checks, then the launches.
#include <hip/hip_runtime.h>

#include "common.h"
#include "serve.h"

using namespace gaje;

namespace {

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_heads(const char *what, int dtype, int64_t n_head, int64_t n_head_kv, int64_t head_dim) {
    if (dtype != GAJE_DTYPE_F32 && dtype != GAJE_DTYPE_F16 && dtype != GAJE_DTYPE_BF16)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: dtype %d (0 f32, 1 f16, 2 bf16)", what, dtype);
    if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv || n_head > 1024)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: %lld heads over %lld K/V heads", what, (long long)n_head,
                         (long long)n_head_kv);
    if (head_dim <= 0 || head_dim % 8 || head_dim > 256)
        return set_error(GAJE_ERR_UNSUPPORTED, "%s: head_dim %lld (a multiple of 8 up to 256)", what, (long long)head_dim);
    return GAJE_OK;
}

int check_pages(const char *what, const gaje_hip_kv_pages *c) {
    if (!c) return set_error(GAJE_ERR_INVALID_ARG, "%s: null cache", what);
    GAJE_TRY(check_heads(what, c->dtype, c->n_head_kv, c->n_head_kv, c->head_dim));
    if (!c->k || !c->v || !c->table || !c->len || !c->ref)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: the cache lacks an array", what);
    if (!aligned16(c->k) || !aligned16(c->v))
        return set_error(GAJE_ERR_INVALID_ARG, "%s: the cache's K and V must be 16-byte aligned", what);
    if (c->page < 8 || c->page > 1024 || (c->page & (c->page - 1)))
        return set_error(GAJE_ERR_INVALID_ARG, "%s: page of %d positions (a power of two, 8 to 1024)", what, c->page);
    if (c->n_layer <= 0 || c->n_layer > 65535 || c->n_pages <= 0 || c->n_pages > (int64_t)1 << 26 || c->n_seq <= 0 ||
        c->n_seq > 65536 || c->max_pages <= 0 || c->max_pages * c->page > (int64_t)1 << 24)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: %lld layers of %lld pages, %lld sequences of up to %lld pages", what,
                         (long long)c->n_layer, (long long)c->n_pages, (long long)c->n_seq, (long long)c->max_pages);
    return GAJE_OK;
}

// The arrays a call writes must not overlap the ones it reads.
bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    return (uintptr_t)a < (uintptr_t)b + (uint64_t)nb && (uintptr_t)b < (uintptr_t)a + (uint64_t)na;
}
int check_new(const char *what, const gaje_hip_kv_pages *c, const void *p, int64_t bytes) {
    const int64_t table = c->n_seq * c->max_pages * 4;
    if (((uintptr_t)p & 3) != 0 || overlap(p, bytes, c->table, table) || overlap(p, bytes, c->len, c->n_seq * 4) ||
        overlap(p, bytes, c->ref, c->n_pages * 4))
        return set_error(GAJE_ERR_INVALID_ARG, "%s: the new arrays must be 4-byte aligned and not the cache's own", what);
    return GAJE_OK;
}

int check_layer(const char *what, const gaje_hip_kv_pages *c, int64_t layer) {
    if (layer < 0 || layer >= c->n_layer)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: layer %lld of %lld", what, (long long)layer, (long long)c->n_layer);
    return GAJE_OK;
}

// Rows of `width` elements, ld apart, read or written 16 bytes at a time.
int check_rows(const char *what, const char *name, const void *p, int64_t ld, int64_t width) {
    if (!p) return set_error(GAJE_ERR_INVALID_ARG, "%s: null %s", what, name);
    if (!aligned16(p) || ld % 8 || ld < width || ld > (int64_t)1 << 21)
        return set_error(GAJE_ERR_INVALID_ARG,
                         "%s: %s needs 16-byte aligned rows, a leading dimension of %lld to 2^21 and a multiple of 8 (got %lld)",
                         what, name, (long long)width, (long long)ld);
    return GAJE_OK;
}

int check_count(const char *what, int64_t n_seq, int64_t T) {
    if (n_seq < 0 || n_seq > 65536 || T < 0 || T > (int64_t)1 << 24)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: %lld sequences, %lld rows", what, (long long)n_seq, (long long)T);
    return GAJE_OK;
}

// Rows times heads are counted in 32 bits.
int check_attn_count(const char *what, int64_t n_seq, int64_t T, int n_head) {
    GAJE_TRY(check_count(what, n_seq, T));
    if (T * n_head > (int64_t)1 << 30)
        return set_error(GAJE_ERR_UNSUPPORTED, "%s: %lld rows of %d heads (2^30 at most)", what, (long long)T, n_head);
    return GAJE_OK;
}

int check_scale(const char *what, float scale) {
    if (!(scale > 0.0f) || scale > 1e30f)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: scale %g (positive, 1e30 at most)", what, (double)scale);
    return GAJE_OK;
}

int check_workspace(const char *what, const void *ws, int64_t bytes, int64_t need) {
    if (need > 0 && (!ws || !aligned16(ws)))
        return set_error(GAJE_ERR_INVALID_ARG, "%s: the workspace must be 16-byte aligned device memory", what);
    if (bytes < need)
        return set_error(GAJE_ERR_INVALID_ARG, "%s: workspace of %lld bytes is smaller than the %lld needed", what,
                         (long long)bytes, (long long)need);
    return GAJE_OK;
}

ServeAttnParams packed_params(int dtype, int64_t n_seq, int64_t T, int n_head, int n_head_kv, int head_dim) {
    ServeAttnParams p{};
    p.dtype = dtype;
    p.n_seq = n_seq;
    p.T = T;
    p.n_head = n_head;
    p.n_head_kv = n_head_kv;
    p.head_dim = head_dim;
    return p;
}

ServeAttnParams paged_params(const gaje_hip_kv_pages *c, int64_t layer, int64_t T, int n_head) {
    ServeAttnParams p = packed_params(c->dtype, c->n_seq, T, n_head, c->n_head_kv, c->head_dim);
    p.ldk = p.ldv = (int64_t)c->n_head_kv * c->head_dim;
    const int64_t bytes = c->n_pages * c->page * p.ldk * (c->dtype == GAJE_DTYPE_F32 ? 4 : 2) * layer;
    p.k = (const char *)c->k + bytes;
    p.v = (const char *)c->v + bytes;
    p.table = c->table;
    p.len = c->len;
    p.max_pages = c->max_pages;
    p.n_pages = c->n_pages;
    p.page_shift = __builtin_ctz((unsigned)c->page);
    return p;
}

}  // namespace

// -------------------------------------------------------------- the pages --

extern "C" int64_t gaje_hip_kv_workspace(const gaje_hip_kv_pages *c) {
    if (check_pages("kv_workspace", c) != GAJE_OK) return -1;
    return kv_update_workspace(*c);
}

extern "C" int gaje_hip_kv_update(const gaje_hip_kv_pages *c, const int32_t *source, const int32_t *add,
                                  int32_t *new_table, int32_t *new_len, int32_t *new_ref, int32_t *status,
                                  void *workspace, int64_t workspace_bytes, void *stream) {
    clear_error();
    GAJE_TRY(check_pages("kv_update", c));
    if (!new_table || !new_len || !new_ref || !status) return set_error(GAJE_ERR_INVALID_ARG, "kv_update: null argument");
    GAJE_TRY(check_new("kv_update", c, new_table, c->n_seq * c->max_pages * 4));
    GAJE_TRY(check_new("kv_update", c, new_len, c->n_seq * 4));
    GAJE_TRY(check_new("kv_update", c, new_ref, c->n_pages * 4));
    GAJE_TRY(check_workspace("kv_update", workspace, workspace_bytes, kv_update_workspace(*c)));
    return launch_kv_update(*c, source, add, new_table, new_len, new_ref, status, workspace, (hipStream_t)stream);
}

extern "C" int gaje_hip_kv_compact(const gaje_hip_kv_pages *c, int32_t *new_table, int32_t *new_ref, int32_t *n_live,
                                   void *workspace, int64_t workspace_bytes, void *stream) {
    clear_error();
    GAJE_TRY(check_pages("kv_compact", c));
    if (!new_table || !new_ref || !n_live) return set_error(GAJE_ERR_INVALID_ARG, "kv_compact: null argument");
    GAJE_TRY(check_new("kv_compact", c, new_table, c->n_seq * c->max_pages * 4));
    GAJE_TRY(check_new("kv_compact", c, new_ref, c->n_pages * 4));
    GAJE_TRY(check_workspace("kv_compact", workspace, workspace_bytes, kv_update_workspace(*c)));
    return launch_kv_compact(*c, new_table, new_ref, n_live, workspace, (hipStream_t)stream);
}

extern "C" int gaje_hip_kv_append(const gaje_hip_kv_pages *c, int64_t layer, int source_dtype, const void *k,
                                  int64_t ldk, const void *v, int64_t ldv, const int32_t *seq_off, int64_t T,
                                  void *stream) {
    clear_error();
    GAJE_TRY(check_pages("kv_append", c));
    GAJE_TRY(check_layer("kv_append", c, layer));
    if (source_dtype != GAJE_DTYPE_F32 && source_dtype != c->dtype)
        return set_error(GAJE_ERR_INVALID_ARG, "kv_append: rows of dtype %d into a cache of dtype %d (f32 or the same)",
                         source_dtype, c->dtype);
    GAJE_TRY(check_count("kv_append", c->n_seq, T));
    if (T == 0) return GAJE_OK;
    if (!seq_off) return set_error(GAJE_ERR_INVALID_ARG, "kv_append: null seq_off");
    const int64_t width = (int64_t)c->n_head_kv * c->head_dim;
    GAJE_TRY(check_rows("kv_append", "k", k, ldk, width));
    GAJE_TRY(check_rows("kv_append", "v", v, ldv, width));
    return launch_kv_append(*c, layer, source_dtype, k, ldk, v, ldv, seq_off, T, (hipStream_t)stream);
}

// -------------------------------------------------------------- attention --

extern "C" int64_t gaje_hip_attention_packed_workspace(int64_t T, int64_t n_seq, int n_head, int n_head_kv,
                                                       int head_dim) {
    if (check_heads("attention_packed", GAJE_DTYPE_F32, n_head, n_head_kv, head_dim) != GAJE_OK ||
        check_attn_count("attention_packed", n_seq, T, n_head) != GAJE_OK)
        return -1;
    if (T == 0 || n_seq == 0) return 0;
    int64_t most = 0;  // a workspace serves every dtype
    for (int d : {GAJE_DTYPE_F32, GAJE_DTYPE_F16}) {
        const int64_t b = serve_attn_workspace(packed_params(d, n_seq, T, n_head, n_head_kv, head_dim));
        if (b > most) most = b;
    }
    return most;
}

extern "C" int gaje_hip_attention_packed(int dtype, const void *q, int64_t ldq, const void *k, int64_t ldk,
                                         const void *v, int64_t ldv, const int32_t *seq_off, int64_t n_seq, int64_t T,
                                         int n_head, int n_head_kv, int head_dim, float scale, void *out, int64_t ldo,
                                         void *workspace, int64_t workspace_bytes, void *stream) {
    static const char *const me = "attention_packed";
    clear_error();
    GAJE_TRY(check_heads(me, dtype, n_head, n_head_kv, head_dim));
    GAJE_TRY(check_attn_count(me, n_seq, T, n_head));
    GAJE_TRY(check_scale(me, scale));
    if (T == 0 || n_seq == 0) return GAJE_OK;
    if (!seq_off) return set_error(GAJE_ERR_INVALID_ARG, "%s: null seq_off", me);
    GAJE_TRY(check_rows(me, "q", q, ldq, (int64_t)n_head * head_dim));
    GAJE_TRY(check_rows(me, "k", k, ldk, (int64_t)n_head_kv * head_dim));
    GAJE_TRY(check_rows(me, "v", v, ldv, (int64_t)n_head_kv * head_dim));
    GAJE_TRY(check_rows(me, "out", out, ldo, (int64_t)n_head * head_dim));
    ServeAttnParams p = packed_params(dtype, n_seq, T, n_head, n_head_kv, head_dim);
    p.q = q;
    p.ldq = ldq;
    p.k = k;
    p.ldk = ldk;
    p.v = v;
    p.ldv = ldv;
    p.out = out;
    p.ldo = ldo;
    p.seq_off = seq_off;
    p.scale = scale;
    GAJE_TRY(check_workspace(me, workspace, workspace_bytes, serve_attn_workspace(p)));
    return launch_serve_attn(p, workspace, (hipStream_t)stream);
}

extern "C" int64_t gaje_hip_attention_paged_workspace(const gaje_hip_kv_pages *c, int64_t T, int n_head) {
    static const char *const me = "attention_paged";
    if (check_pages(me, c) != GAJE_OK || check_heads(me, c->dtype, n_head, c->n_head_kv, c->head_dim) != GAJE_OK ||
        check_attn_count(me, c->n_seq, T, n_head) != GAJE_OK)
        return -1;
    return T == 0 ? 0 : serve_attn_workspace(paged_params(c, 0, T, n_head));
}

extern "C" int gaje_hip_attention_paged(const void *q, int64_t ldq, const gaje_hip_kv_pages *c, int64_t layer,
                                        const int32_t *seq_off, int64_t T, int n_head, float scale, void *out,
                                        int64_t ldo, void *workspace, int64_t workspace_bytes, void *stream) {
    static const char *const me = "attention_paged";
    clear_error();
    GAJE_TRY(check_pages(me, c));
    GAJE_TRY(check_layer(me, c, layer));
    GAJE_TRY(check_heads(me, c->dtype, n_head, c->n_head_kv, c->head_dim));
    GAJE_TRY(check_attn_count(me, c->n_seq, T, n_head));
    GAJE_TRY(check_scale(me, scale));
    if (T == 0) return GAJE_OK;
    if (!seq_off) return set_error(GAJE_ERR_INVALID_ARG, "%s: null seq_off", me);
    GAJE_TRY(check_rows(me, "q", q, ldq, (int64_t)n_head * c->head_dim));
    GAJE_TRY(check_rows(me, "out", out, ldo, (int64_t)n_head * c->head_dim));
    ServeAttnParams p = paged_params(c, layer, T, n_head);
    p.q = q;
    p.ldq = ldq;
    p.out = out;
    p.ldo = ldo;
    p.seq_off = seq_off;
    p.scale = scale;
    GAJE_TRY(check_workspace(me, workspace, workspace_bytes, serve_attn_workspace(p)));
    return launch_serve_attn(p, workspace, (hipStream_t)stream);
}

extern "C" int64_t gaje_hip_attention_prefix_workspace(const gaje_hip_kv_pages *c, int64_t prefix_len, int n_head) {
    static const char *const me = "attention_prefix";
    if (check_pages(me, c) != GAJE_OK || check_heads(me, c->dtype, n_head, c->n_head_kv, c->head_dim) != GAJE_OK) return -1;
    if (prefix_len < 0 || prefix_len > c->max_pages * c->page) {
        set_error(GAJE_ERR_INVALID_ARG, "%s: a prefix of %lld positions", me, (long long)prefix_len);
        return -1;
    }
    ServeAttnParams p = paged_params(c, 0, c->n_seq, n_head);
    p.prefix_table = c->table;
    p.prefix_len = prefix_len;
    return serve_attn_workspace(p);
}

extern "C" int gaje_hip_attention_prefix(const void *q, int64_t ldq, const gaje_hip_kv_pages *c, int64_t layer,
                                         const int32_t *prefix_table, int64_t prefix_len, int n_head, float scale,
                                         void *out, int64_t ldo, void *workspace, int64_t workspace_bytes,
                                         void *stream) {
    static const char *const me = "attention_prefix";
    clear_error();
    GAJE_TRY(check_pages(me, c));
    GAJE_TRY(check_layer(me, c, layer));
    GAJE_TRY(check_heads(me, c->dtype, n_head, c->n_head_kv, c->head_dim));
    GAJE_TRY(check_scale(me, scale));
    if (prefix_len < 0 || prefix_len > c->max_pages * c->page || (prefix_len > 0 && !prefix_table))
        return set_error(GAJE_ERR_INVALID_ARG, "%s: a prefix of %lld positions", me, (long long)prefix_len);
    GAJE_TRY(check_rows(me, "q", q, ldq, (int64_t)n_head * c->head_dim));
    GAJE_TRY(check_rows(me, "out", out, ldo, (int64_t)n_head * c->head_dim));
    ServeAttnParams p = paged_params(c, layer, c->n_seq, n_head);
    p.q = q;
    p.ldq = ldq;
    p.out = out;
    p.ldo = ldo;
    p.scale = scale;
    p.prefix_table = prefix_table ? prefix_table : c->table;
    p.prefix_len = prefix_len;
    GAJE_TRY(check_workspace(me, workspace, workspace_bytes, serve_attn_workspace(p)));
    return launch_serve_attn(p, workspace, (hipStream_t)stream);
}
