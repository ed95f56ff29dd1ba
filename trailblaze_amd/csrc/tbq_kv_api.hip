// tbq_kv_api.hip -- the extern "C" API of the paged key/value cache
// (include/tbq_kv.h): checks on the host, all of them before the first HIP
// call, then the gfx950 launchers.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/tbq_kv.h"
#include "tbq_kernels.h"
#include "tbq_paged.hpp"
#include "tbq_serve.hpp"

using namespace tbq;

extern "C" int tbq_host_fail(const char *msg);

namespace {

int fail(const char *fmt, ...) __attribute__((format(printf, 1, 2)));
int fail(const char *fmt, ...) {
    char msg[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    return tbq_host_fail(msg);
}

int hip_ok(hipError_t e, const char *what) { return e == hipSuccess ? 1 : fail("%s: %s", what, hipGetErrorString(e)); }

bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

hipStream_t S(void *s) { return reinterpret_cast<hipStream_t>(s); }

bool cache_type(int t) { return t == TBQ_KV_F16 || t == TBQ_KV_BF16 || t == TBQ_KV_MXFP4; }
bool float_type(int t) { return t == TBQ_KV_F32 || t == TBQ_KV_F16 || t == TBQ_KV_BF16; }
bool head_dim(int d) { return d == 64 || d == 128; }
bool page_size(int n) { return n == 16 || n == 32 || n == 64 || n == 128 || n == 256; }

int check_cache(const char *who, const tbq_kv_cache *c) {
    if (!c) return fail("%s: null cache", who);
    if (!cache_type(c->type)) return fail("%s: cache type %d (F16, BF16 or MXFP4)", who, c->type);
    if (!head_dim(c->head_dim)) return fail("%s: head_dim %d (64 or 128)", who, c->head_dim);
    if (!page_size(c->page_size)) return fail("%s: page_size %d (16, 32, 64, 128 or 256)", who, c->page_size);
    if (c->n_layers < 1 || c->n_layers > 16384 || c->n_pages < 1 || c->n_kv_heads < 1 || c->n_kv_heads > 65535)
        return fail("%s: cache of %d layers, %d pages, %d kv heads", who, c->n_layers, c->n_pages, c->n_kv_heads);
    if ((long long)c->n_pages * c->n_kv_heads * c->page_size > 0x7FFFFFFF)
        return fail("%s: more than 2^31 - 1 rows of kv heads in a layer", who);
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) return fail("%s: null or misaligned cache", who);
    return 1;
}

int check_layer(const char *who, const tbq_kv_cache *c, int layer) {
    return layer >= 0 && layer < c->n_layers ? 1 : fail("%s: layer %d of %d", who, layer, c->n_layers);
}

int check_batch(const char *who, const tbq_kv_batch *b) {
    if (!b) return fail("%s: null batch", who);
    if (b->n_seqs < 0 || b->n_seqs > 65535 || b->n_tokens < 0 || b->max_pages < 1 || b->max_q < 0 || b->max_kv < 0)
        return fail("%s: batch of %d sequences, %d tokens, %d pages, max_q %d, max_kv %d", who, b->n_seqs, b->n_tokens,
                    b->max_pages, b->max_q, b->max_kv);
    if (b->n_seqs && (!b->q_start || !b->kv_len || !b->page_table)) return fail("%s: null batch array", who);
    return 1;
}

long long page_bytes(const tbq_kv_cache *c) {
    return (long long)c->n_kv_heads * c->page_size * pg_row_bytes(c->type, c->head_dim);
}

PgArgs pg_args(const tbq_kv_cache *c, int layer, const tbq_kv_batch *b) {
    PgArgs a = pg_layer(c, layer);
    a.n_seqs = b->n_seqs;
    a.n_tokens = b->n_tokens;
    a.max_pages = b->max_pages;
    a.max_q = b->max_q > 0 && b->max_q < b->n_tokens ? b->max_q : b->n_tokens;
    const long long room = (long long)b->max_pages * c->page_size;
    const int most = room > (1 << 30) ? 1 << 30 : (int)room;   // position arithmetic stays in 32 bits
    a.max_kv = b->max_kv > 0 && b->max_kv < most ? b->max_kv : most;
    a.q_start = b->q_start;
    a.kv_len = b->kv_len;
    a.table = b->page_table;
    return a;
}

}  // namespace

extern "C" {

// For tbq_api.hip (hidden): the checks of a cache.
__attribute__((visibility("hidden"))) int tbq_kv_check_cache(const char *who, const tbq_kv_cache *c) {
    return check_cache(who, c);
}

size_t tbq_kv_head_bytes(int type, int page, int dim) {
    return cache_type(type) && page_size(page) && head_dim(dim) ? (size_t)page * pg_row_bytes(type, dim) : 0;
}

int tbq_rope_init(tbq_rope *r, int rot_dim, int layout, double theta, int scaling, double factor, int orig_ctx,
                  double beta_fast, double beta_slow, const float *factors) {
    if (!r) return fail("tbq_rope_init: null plan");
    if (rot_dim < 8 || rot_dim > 128 || rot_dim % 8) return fail("tbq_rope_init: rot_dim %d (a multiple of 8 up to 128)", rot_dim);
    if (layout != TBQ_ROPE_HALF && layout != TBQ_ROPE_INTERLEAVED) return fail("tbq_rope_init: layout %d", layout);
    if (!(theta > 1) || !isfinite(theta)) return fail("tbq_rope_init: theta %g", theta);
    if (scaling < TBQ_ROPE_NO_SCALING || scaling > TBQ_ROPE_YARN) return fail("tbq_rope_init: scaling %d", scaling);
    if (scaling != TBQ_ROPE_NO_SCALING && (!(factor >= 1) || !isfinite(factor)))
        return fail("tbq_rope_init: factor %g (at least 1)", factor);
    if (beta_fast == 0) beta_fast = 32;
    if (beta_slow == 0) beta_slow = 1;
    if (scaling == TBQ_ROPE_YARN && (orig_ctx < 1 || !(beta_slow > 0) || !(beta_fast >= beta_slow) || !isfinite(beta_fast)))
        return fail("tbq_rope_init: orig_ctx %d, beta_fast %g, beta_slow %g", orig_ctx, beta_fast, beta_slow);
    for (int j = 0; factors && j < rot_dim / 2; j++)
        if (!(factors[j] > 0) || !isfinite(factors[j])) return fail("tbq_rope_init: factors[%d] = %g", j, factors[j]);
    memset(r, 0, sizeof *r);
    r->rot_dim = rot_dim;
    r->layout = layout;
    r->mscale = scaling == TBQ_ROPE_YARN ? 0.1 * log(factor) + 1 : 1;
    // The pair that turns beta times in orig_ctx positions.  (The whole pairs that bound the ramp, their
    // limits 0 and rot_dim - 1 and the 0.001 between equal ones are not the paper's: models are trained
    // with them.)
    auto pair = [&](double beta) { return rot_dim * log(orig_ctx / (beta * 2 * M_PI)) / (2 * log(theta)); };
    double lo = 0, hi = 0;
    if (scaling == TBQ_ROPE_YARN) {
        lo = fmax(floor(pair(beta_fast)), 0);
        hi = fmin(ceil(pair(beta_slow)), rot_dim - 1);
    }
    for (int j = 0; j < rot_dim / 2; j++) {
        double f = pow(theta, -2.0 * j / rot_dim);
        if (factors) f /= factors[j];
        if (scaling == TBQ_ROPE_LINEAR) f /= factor;
        if (scaling == TBQ_ROPE_YARN) {
            const double share = fmin(fmax((j - lo) / fmax(hi - lo, 0.001), 0), 1);
            f = f / factor * share + f * (1 - share);
        }
        r->freq[j] = f;
    }
    return 1;
}

int tbq_kv_append(const tbq_kv_cache *c, int layer, const tbq_kv_batch *b, int n_heads, const tbq_rope *rope,
                  const float *q_norm, const float *k_norm, float eps, const int *positions, int in_type, const void *q,
                  long long qs, const void *k, long long ks, const void *v, long long vs, int q_type, void *q_out,
                  void *stream) {
    const char *who = "tbq_kv_append";
    if (!check_cache(who, c) || !check_layer(who, c, layer) || !check_batch(who, b)) return 0;
    const int D = c->head_dim;
    const bool mx = c->type == TBQ_KV_MXFP4;
    if (mx ? !float_type(in_type) : in_type != TBQ_KV_F32 && in_type != c->type)
        return fail("%s: in_type %d (F32 or the cache's; F32, F16 or BF16 with MXFP4)", who, in_type);
    if (!q != !q_out) return fail("%s: q and q_out go together", who);
    if (q && (mx ? !float_type(q_type) || (in_type != TBQ_KV_F32 && q_type != in_type)
                 : q_type != c->type && !(q_type == TBQ_KV_F32 && in_type == TBQ_KV_F32)))
        return fail("%s: q_type %d with in_type %d and cache type %d", who, q_type, in_type, c->type);
    if (q && (n_heads < 1 || n_heads > 65535)) return fail("%s: n_heads %d", who, n_heads);
    if (rope) {
        if (rope->rot_dim < 8 || rope->rot_dim > D || rope->rot_dim % 8)
            return fail("%s: rot_dim %d (a multiple of 8 up to head_dim)", who, rope->rot_dim);
        if (rope->layout != TBQ_ROPE_HALF && rope->layout != TBQ_ROPE_INTERLEAVED)
            return fail("%s: rope layout %d", who, rope->layout);
    }
    if (b->n_seqs == 0 || b->n_tokens == 0) return 1;
    if (!k || !v) return fail("%s: null k or v", who);
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(q_norm, 16) ||
        !aligned(k_norm, 16))
        return fail("%s: misaligned pointer (16 bytes)", who);
    if ((q && qs % 8) || ks % 8 || vs % 8) return fail("%s: strides must be multiples of 8 elements", who);
    if ((q && qs < (long long)n_heads * D) || ks < (long long)c->n_kv_heads * D || vs < (long long)c->n_kv_heads * D)
        return fail("%s: a stride is shorter than its heads", who);
    if (q && q_out == q && (q_type != in_type || qs != (long long)n_heads * D))
        return fail("%s: q_out is q, but its type or stride differs", who);
    if (!tbq_init()) return 0;
    PgAppend a{};
    a.pg = pg_args(c, layer, b);
    a.q = q;
    a.k = k;
    a.v = v;
    a.qs = qs;
    a.ks = ks;
    a.vs = vs;
    a.qo = q_out;
    a.qn = q_norm;
    a.kn = k_norm;
    a.positions = positions;
    a.eps = eps;
    a.NQ = q ? n_heads : 0;
    a.nsl = 1;
    if (rope) pg_rope(*rope, a.rope);
    return hip_ok(launch_pg_append(a, D, in_type, q ? q_type : mx ? in_type : c->type, c->type, S(stream)),
                  "kv append launch");
}

static int check_attn(const char *who, const tbq_kv_cache *c, const tbq_kv_batch *b, int n_heads, int q_type) {
    if (!check_cache(who, c) || !check_batch(who, b)) return 0;
    if (n_heads < 1 || n_heads > 65535 || n_heads % c->n_kv_heads)
        return fail("%s: n_heads %d, a multiple of the %d kv heads", who, n_heads, c->n_kv_heads);
    if ((long long)b->n_tokens * n_heads >= 1ll << 30) return fail("%s: %d tokens of %d heads", who, b->n_tokens, n_heads);
    if (c->type == TBQ_KV_MXFP4 ? !float_type(q_type) : q_type != c->type && !(q_type == TBQ_KV_F32 && c->type == TBQ_KV_F16))
        return fail("%s: q_type %d with cache type %d (the cache's type, F32 with an F16 cache, any with MXFP4)", who, q_type,
                    c->type);
    return 1;
}

size_t tbq_attn_paged_workspace_size(const tbq_kv_cache *c, const tbq_kv_batch *b, int n_heads, int q_type) {
    if (!check_attn("tbq_attn_paged_workspace_size", c, b, n_heads, q_type)) return 0;
    return pg_attn_workspace_bytes(pg_args(c, 0, b), c->head_dim, n_heads, q_type == TBQ_KV_F32, c->type);
}

int tbq_attn_paged(const tbq_kv_cache *c, int layer, const tbq_kv_batch *b, int n_heads, int q_type, const void *q,
                   long long qs, void *out, int window, int sinks, float scale, void *ws, size_t ws_bytes, void *stream) {
    const char *who = "tbq_attn_paged";
    if (!check_attn(who, c, b, n_heads, q_type) || !check_layer(who, c, layer)) return 0;
    if (window < 0 || sinks < 0) return fail("%s: window %d, sinks %d", who, window, sinks);
    if (!(scale >= 0) || !isfinite(scale)) return fail("%s: scale %g", who, (double)scale);
    if (b->n_seqs == 0 || b->n_tokens == 0) return 1;
    if (!q || !out || !aligned(q, 16) || !aligned(out, 16)) return fail("%s: null or misaligned pointer (16 bytes)", who);
    if (qs % 8 || qs < (long long)n_heads * c->head_dim) return fail("%s: q_stride %lld", who, qs);
    PgAttn a{};
    a.pg = pg_args(c, layer, b);
    const size_t need = pg_attn_workspace_bytes(a.pg, c->head_dim, n_heads, q_type == TBQ_KV_F32, c->type);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 16)))
        return fail("%s: workspace %zu < %zu bytes, or not 16-byte aligned", who, ws ? ws_bytes : 0, need);
    if (!tbq_init()) return 0;
    a.q = q;
    a.qs = qs;
    a.out = out;
    a.NQ = n_heads;
    a.window = pg_window(window);
    a.sinks = window > 0 ? pg_window(sinks) : 0;
    a.scale = pg_scale(scale, c->head_dim);
    return hip_ok(launch_pg_attn(a, c->head_dim, q_type, c->type, ws, S(stream)), "paged attention launch");
}

int tbq_kv_dequant(const tbq_kv_cache *c, int layer, const int *pages, int n, int out_type, void *k_out, void *v_out,
                   void *stream) {
    const char *who = "tbq_kv_dequant";
    if (!check_cache(who, c) || !check_layer(who, c, layer)) return 0;
    if (c->type != TBQ_KV_MXFP4) return fail("%s: cache type %d (MXFP4)", who, c->type);
    if (!float_type(out_type)) return fail("%s: out_type %d (F32, F16 or BF16)", who, out_type);
    // (a workgroup for 16 rows at most: their number, times 256 threads, stays below 2^32)
    if (n < 0 || n > (1 << 20) || (!pages && n > c->n_pages)) return fail("%s: %d pages of %d", who, n, c->n_pages);
    if (n == 0) return 1;
    if (!k_out || !v_out || !aligned(k_out, 16) || !aligned(v_out, 16))
        return fail("%s: null or misaligned output (16 bytes)", who);
    if (!tbq_init()) return 0;
    tbq_kv_batch b{};
    b.max_pages = 1;
    return hip_ok(launch_mx_dequant(pg_args(c, layer, &b), c->head_dim, pages, n, out_type, k_out, v_out, S(stream)),
                  "kv dequant launch");
}

int tbq_kv_copy_pages(const tbq_kv_cache *c, const int *src, const int *dst, int n, void *stream) {
    const char *who = "tbq_kv_copy_pages";
    if (!check_cache(who, c)) return 0;
    if (n < 0 || (n > 0 && (!src || !dst))) return fail("%s: %d pairs", who, n);
    if (n == 0) return 1;
    for (int i = 0; i < n; i++)
        if (src[i] < 0 || src[i] >= c->n_pages || dst[i] < 0 || dst[i] >= c->n_pages)
            return fail("%s: pair %d: page %d -> %d of %d pages", who, i, src[i], dst[i], c->n_pages);
    // one byte a page: 1 a source, 2 a destination
    unsigned char *seen = (unsigned char *)calloc((size_t)c->n_pages, 1);
    if (!seen) return fail("%s: out of host memory", who);
    int bad = -1;
    for (int i = 0; i < n; i++) seen[src[i]] |= 1;
    for (int i = 0; i < n && bad < 0; i++) {
        if (seen[dst[i]]) bad = i;
        seen[dst[i]] |= 2;
    }
    free(seen);
    if (bad >= 0) return fail("%s: page %d is written twice, or read and written", who, dst[bad]);
    if (!tbq_init()) return 0;
    const long long pbytes = page_bytes(c), lbytes = pbytes * c->n_pages;
    for (int i = 0; i < n; i += PG_PAIRS) {
        PgPairs p;
        const int m = n - i < PG_PAIRS ? n - i : PG_PAIRS;
        memcpy(p.src, src + i, m * sizeof(int));
        memcpy(p.dst, dst + i, m * sizeof(int));
        if (!hip_ok(launch_pg_copy(c->k, c->v, c->n_layers, pbytes, lbytes, p, m, S(stream)), "page copy launch")) return 0;
    }
    return 1;
}

int tbq_kv_compact(const tbq_kv_cache *c, int n_seqs, const int *page_table, int max_pages, const int *keep_start,
                   const int *keep, void *stream) {
    const char *who = "tbq_kv_compact";
    if (!check_cache(who, c)) return 0;
    if (n_seqs < 0 || n_seqs > 65535 || max_pages < 1) return fail("%s: %d sequences, %d pages", who, n_seqs, max_pages);
    if (n_seqs == 0) return 1;
    if (!page_table || !keep_start || !keep) return fail("%s: null pointer", who);
    if (!tbq_init()) return 0;
    tbq_kv_batch b{};
    b.n_seqs = n_seqs;
    b.max_pages = max_pages;
    b.page_table = page_table;
    const long long lbytes = page_bytes(c) * c->n_pages;
    const PgArgs a = pg_args(c, 0, &b);
    return hip_ok(c->type == TBQ_KV_MXFP4
                      ? launch_mx_compact(c->k, c->v, c->n_layers, lbytes, c->head_dim, a, keep_start, keep, S(stream))
                      : launch_pg_compact(c->k, c->v, c->n_layers, lbytes / 2, c->head_dim, a, keep_start, keep, S(stream)),
                  "compact launch");
}

int tbq_kv_build_tables(const tbq_kv_tables *t, void *stream) {
    const char *who = "tbq_kv_build_tables";
    if (!t) return fail("%s: null tables", who);
    if (!page_size(t->page_size)) return fail("%s: page_size %d (16, 32, 64, 128 or 256)", who, t->page_size);
    if (t->n_seqs < 0 || t->n_seqs > 65535 || t->n_tokens < 0 || t->n_tokens > 1 << 30 || t->max_pages < 1 ||
        t->n_pages < 1 || (long long)t->max_pages * t->page_size > 1 << 30 ||
        (long long)t->n_seqs * t->max_pages > 0x7FFFFFFF || (long long)t->n_pages * t->page_size > 0x7FFFFFFF)
        return fail("%s: %d sequences of %d pages, %d tokens, %d pages of %d", who, t->n_seqs, t->max_pages, t->n_tokens,
                    t->n_pages, t->page_size);
    if (!t->q_start || !t->free_pages || !t->n_free || !t->free_out || !t->n_free_out ||
        (t->n_seqs && (!t->kv_len || !t->n_new || !t->page_table || !t->kv_len_out || !t->page_table_out)))
        return fail("%s: null array", who);
    if ((t->free_out == t->free_pages) != (t->n_free_out == t->n_free))
        return fail("%s: free_out and n_free_out go together: both in place, or neither", who);
    if (!tbq_init()) return 0;
    return hip_ok(launch_tables({*t, pg_log2(t->page_size)}, S(stream)), "tables launch");
}

static int check_verify(const char *who, int n_seqs, int n_rows, int vocab, int type, bool draft) {
    if (n_seqs < 0 || n_seqs > 65535 || n_rows < 0 || vocab < 1 || vocab > 1 << 28)
        return fail("%s: %d sequences, %d rows of %d", who, n_seqs, n_rows, vocab);
    if (!float_type(type)) return fail("%s: type %d (F32, F16 or BF16)", who, type);
    // a workgroup of 256 a chunk: their threads stay below 2^32
    const long long chunks = (vocab + DV_CHUNK - 1) / DV_CHUNK;
    if (chunks * (n_rows > n_seqs ? n_rows : n_seqs) * (draft ? 2 : 1) > (1 << 24) - 1)
        return fail("%s: %d rows of %d", who, n_rows, vocab);
    return 1;
}

size_t tbq_draft_verify_workspace_size(int n_seqs, int n_rows, int vocab, int type, int draft) {
    if (!check_verify("tbq_draft_verify_workspace_size", n_seqs, n_rows, vocab, type, draft)) return 0;
    return verify_workspace_bytes(n_seqs, n_rows, vocab, draft);
}

int tbq_draft_verify(int n_seqs, int n_rows, int vocab, int type, const int *q_start, const int *tokens,
                     const void *logits, long long stride, const void *draft, long long dstride, const float *temperature,
                     const float *u_accept, const float *u_next, int *n_accept, int *next, int *n_drop, void *ws,
                     size_t ws_bytes, void *stream) {
    const char *who = "tbq_draft_verify";
    if (!check_verify(who, n_seqs, n_rows, vocab, type, draft != nullptr)) return 0;
    if (n_seqs == 0) return 1;
    if (!q_start || !u_next || !n_accept || !next || (n_rows && (!tokens || !logits || !u_accept)))
        return fail("%s: null pointer", who);
    const unsigned size = type == TBQ_KV_F32 ? 4 : 2;
    if (!aligned(logits, size) || !aligned(draft, size)) return fail("%s: misaligned logits", who);
    if (n_rows && (stride < vocab || (draft && dstride < vocab))) return fail("%s: a stride is shorter than its row", who);
    const size_t need = verify_workspace_bytes(n_seqs, n_rows, vocab, draft != nullptr);
    if (need && (!ws || ws_bytes < need || !aligned(ws, 16)))
        return fail("%s: workspace %zu < %zu bytes, or not 16-byte aligned", who, ws ? ws_bytes : 0, need);
    if (!tbq_init()) return 0;
    SvVerify a{};
    a.n_seqs = n_seqs;
    a.n_rows = n_rows;
    a.vocab = vocab;
    a.chunks = (vocab + DV_CHUNK - 1) / DV_CHUNK;
    a.q_start = q_start;
    a.tokens = tokens;
    a.logits = logits;
    a.draft = draft;
    a.stride = stride;
    a.dstride = dstride;
    a.temperature = temperature;
    a.u_accept = u_accept;
    a.u_next = u_next;
    a.n_accept = n_accept;
    a.next = next;
    a.n_drop = n_drop;
    return hip_ok(launch_verify(a, type, ws, S(stream)), "draft verify launch");
}

}  // extern "C"
