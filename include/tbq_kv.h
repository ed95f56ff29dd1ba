/*
 * tbq_kv.h -- a paged key/value cache for many sequences, and the operators
 * that work on it: rotary positions with the append of new keys and values,
 * causal attention of new tokens over the pages (whole, or a sliding window
 * with sinks), page copies, row compaction, a host-side page pool, and the
 * dense model's forward over such a cache.  No counterpart in the reference,
 * whose cache is one contiguous fp32 buffer of one sequence
 * (layer1/tb_tensor.c:229-291).
 *
 * Conventions are tbq.h's: device pointers, `stream` a hipStream_t, calls
 * enqueue work and return 1, or 0 with tbq_last_error().  Nothing here
 * allocates device memory, and every call with device inputs can be captured
 * into a graph.
 */
#ifndef TBQ_KV_H
#define TBQ_KV_H

#include <stddef.h>

#include "tbq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types, as tbq.h's ids: 0 F32, 1 F16 (IEEE halves), 30 BF16. */
#define TBQ_KV_F32 0
#define TBQ_KV_F16 1
#define TBQ_KV_BF16 30

/* The cache: K and V are [n_layers][n_pages][n_kv_heads][page_size][head_dim]
 * of `type` (F16 or BF16), 16-byte aligned.  head_dim 64 or 128; page_size
 * 16, 32, 64, 128 or 256 positions.  Position p of a sequence is row
 * p % page_size of the page that its page table names at p / page_size. */
typedef struct {
    int n_layers, n_pages, n_kv_heads, page_size, head_dim, type;
    void *k, *v;
} tbq_kv_cache;

/* New tokens of n_seqs sequences side by side (device arrays of int, which a
 * captured call reads again at every replay).  Sequence s has the token rows
 * q_start[s] .. q_start[s + 1] - 1 (none, one or many; q_start[0] = 0,
 * non-decreasing), and kv_len[s] positions with them: its i-th new token is
 * at position kv_len[s] - (q_start[s + 1] - q_start[s]) + i.  page_table is
 * [n_seqs][max_pages].  Token rows at or behind q_start[n_seqs] belong to no
 * sequence: no call reads or writes anything for them.
 * n_tokens: rows of q, k, v and the outputs.  max_q, max_kv: what no
 * sequence's number of new tokens and of positions exceeds; launches are sized
 * by them, and 0 stands for n_tokens and max_pages * page_size.  Lengths
 * above them (or above 2^30 positions) are an error that the device does not
 * report: what lies beyond is left out.  A page number outside the cache is
 * never followed: keys there are not written and not visible. */
typedef struct {
    int n_seqs, n_tokens, max_pages, max_q, max_kv;
    const int *q_start;    /* [n_seqs + 1] */
    const int *kv_len;     /* [n_seqs] */
    const int *page_table; /* [n_seqs][max_pages] */
} tbq_kv_batch;

/* ---- rotary positions --------------------------------------------------- */
#define TBQ_ROPE_HALF 0         /* pairs (j, j + rot_dim / 2) */
#define TBQ_ROPE_INTERLEAVED 1  /* pairs (2j, 2j + 1) */
#define TBQ_ROPE_NO_SCALING 0
#define TBQ_ROPE_LINEAR 1       /* every frequency divided by factor */
#define TBQ_ROPE_YARN 2         /* arXiv 2309.00071 */

/* A plan: pair j of the first rot_dim elements of a head turns by freq[j]
 * radians per position and is scaled by mscale; the elements behind rot_dim
 * stay as they are.  tbq_rope_init fills it; a caller may fill or change it
 * too. */
typedef struct {
    int rot_dim;    /* a multiple of 8, at most head_dim */
    int layout;
    double mscale;
    double freq[64];
} tbq_rope;

/* freq[j] = theta^(-2j / rot_dim), scaled.  LINEAR: / factor.  YARN: the
 * share 1 - r_j kept and the share r_j divided by factor, where r_j rises
 * from 0 to 1 between the pairs that turn beta_fast and beta_slow times in
 * orig_ctx positions (0 for either: 32 and 1), and mscale = 0.1 ln(factor) +
 * 1.  factors: NULL, or rot_dim / 2 host floats that each frequency is
 * divided by first (the rope_freqs tensor of a GGUF file).  Host only. */
int tbq_rope_init(tbq_rope *rope, int rot_dim, int layout, double theta, int scaling, double factor, int orig_ctx,
                  double beta_fast, double beta_slow, const float *factors);

/* ---- append --------------------------------------------------------------- */
/* For every token row t of a sequence: q and k heads RMS-normalised (where
 * q_norm / k_norm, [head_dim] fp32, is not NULL: x * (1 / sqrt(mean(x^2) +
 * eps)) * w), rotated by the token's position (rope NULL: not rotated), q
 * written to q_out [n_tokens][n_heads][head_dim] and k and v to the token's
 * row of its page in `layer`.  The arithmetic is fp32 (angles reduced in
 * fp64), rounded once.
 * q, k, v: heads of row t side by side at base + t * stride elements (strides
 * multiples of 8, 16-byte aligned bases).  in_type is theirs, q_type q_out's:
 * in_type F32 with q_type F32 or the cache's type, or both the cache's type.
 * q (with q_out) may be NULL; q_out may be q itself where types and strides
 * agree (q_stride = n_heads * head_dim), and must overlap no other input.
 * positions: NULL, or [n_tokens] ints that rotate in place of the positions in
 * the cache (rows that an earlier compaction moved keep their own).
 * A token at a negative position is skipped whole; one whose position has no
 * page gets its q, and its k and v are dropped.  No two tokens may share a
 * position of a page. */
int tbq_kv_append(const tbq_kv_cache *c, int layer, const tbq_kv_batch *b, int n_heads, const tbq_rope *rope,
                  const float *q_norm, const float *k_norm, float eps, const int *positions, int in_type,
                  const void *q, long long q_stride, const void *k, long long k_stride, const void *v,
                  long long v_stride, int q_type, void *q_out, void *stream);

/* ---- attention ------------------------------------------------------------ */
/* out[t][h] = softmax(scale * q[t][h] . K^T) V over the visible positions of
 * t's sequence, query head h on kv head h / (n_heads / n_kv_heads).  A token
 * at position p sees the positions <= p; with window > 0 only those > p -
 * window, and the first `sinks` ones.  scale 0 stands for 1 / sqrt(head_dim);
 * else it is positive.  A row that sees nothing, or whose scores are all
 * -infinity, is 0.  What a token does not see has no influence on its row,
 * infinities and NaN included (a row that sees one is not finite where the
 * formula is not), and pages that no token of the call sees any part of may be
 * free: the kernel reads nothing of theirs that enters a result.
 * q [n_tokens][n_heads][head_dim] with q_stride elements between tokens (a
 * multiple of 8), out contiguous, not overlapping q, both of type q_type: the
 * cache's type, or F32 with an F16 cache.  Scores, softmax and sums are fp32.
 * 16-bit rows of a sequence with up to 32 of them a kv head (new tokens times
 * n_heads / n_kv_heads; 16 where the batch may hold more than 256 MiB of keys
 * and values) are rounded once, at the output; with more rows the
 * probabilities are rounded to the cache's type too.  F32 takes q and the
 * probabilities as pairs of halves (~22 bits, relative to a row's largest
 * element), so its rows are exact to about 1e-6.
 * workspace: tbq_attn_paged_workspace_size() bytes, 16-byte aligned, no
 * zero-fill needed; calls that share one must not overlap. */
size_t tbq_attn_paged_workspace_size(const tbq_kv_cache *c, const tbq_kv_batch *b, int n_heads, int q_type);
int tbq_attn_paged(const tbq_kv_cache *c, int layer, const tbq_kv_batch *b, int n_heads, int q_type, const void *q,
                   long long q_stride, void *out, int window, int sinks, float scale, void *workspace,
                   size_t workspace_bytes, void *stream);

/* ---- pages and rows moved ---------------------------------------------------- */
/* Page src[i] of every layer, K and V, is copied to page dst[i], for n pairs
 * of host ints (read before the call returns).  No page may be the destination
 * of two pairs, nor the source of one and the destination of another: such a
 * list is refused. */
int tbq_kv_copy_pages(const tbq_kv_cache *c, const int *src, const int *dst, int n, void *stream);

/* Row j of sequence s, in every layer, becomes its row keep[keep_start[s] +
 * j], for j below keep_start[s + 1] - keep_start[s] (device ints;
 * keep ascending within a sequence).  In place; rows from there on
 * keep their values.  Keys are not rotated again: they stay those of the
 * positions they were written at.  No page may be in two of the sequences'
 * kept or read rows, nor in a sequence outside the call that still reads it: a
 * page with a second holder (tbq_kv_pool_holders) is changed under that one, so
 * it is copied first.  keep has keep_start[n_seqs] entries, all of which may be
 * read. */
int tbq_kv_compact(const tbq_kv_cache *c, int n_seqs, const int *page_table, int max_pages, const int *keep_start,
                   const int *keep, void *stream);

/* ---- page pool (host) -------------------------------------------------------- */
/* Which pages of a cache are in use, by how many holders.  Not thread-safe. */
typedef struct tbq_kv_pool tbq_kv_pool;
tbq_kv_pool *tbq_kv_pool_create(int n_pages);
void tbq_kv_pool_destroy(tbq_kv_pool *p);
int tbq_kv_pool_free_pages(const tbq_kv_pool *p);
/* Holders of a page: 0 free, -1 for a page that is not there. */
int tbq_kv_pool_holders(const tbq_kv_pool *p, int page);
/* The n lowest free pages, each with one holder; 0 and no change where fewer
 * are free. */
int tbq_kv_pool_alloc(tbq_kv_pool *p, int n, int *pages);
/* One holder more, or fewer (the last one frees the page), for each page named
 * (as often as it is named).  0 and no change if any is not there or has too
 * few holders. */
int tbq_kv_pool_share(tbq_kv_pool *p, int n, const int *pages);
int tbq_kv_pool_release(tbq_kv_pool *p, int n, const int *pages);
/* A sequence of `positions` positions in ceil(positions / page_size) pages
 * gets a second holder: child[] = its pages, shared, but a last one that is
 * partly filled is replaced by a new page, and copy[0] -> copy[1] names the
 * tbq_kv_copy_pages that fills it (-1, -1: none).  0 and no change if no page
 * is free for it. */
int tbq_kv_pool_fork(tbq_kv_pool *p, int positions, int page_size, const int *pages, int *child, int copy[2]);
/* Moves that bring the used pages to the lowest numbers: at most `max` pairs
 * src[i] -> dst[i] for tbq_kv_copy_pages, done in the pool's books; the
 * caller replaces src[i] by dst[i] in every page table.  Returns their
 * number (-1: error). */
int tbq_kv_pool_defrag(tbq_kv_pool *p, int max, int *src, int *dst);

/* ---- dense model over a paged cache ------------------------------------------- */
/* The forward of tbq_dense_decode / tbq_dense_prefill (same model struct; its
 * max_ctx, k_cache and v_cache are not used) for n_seqs sequences at once:
 * sequence s's n_new[s] >= 1 tokens follow each other in tokens, kv_len[s]
 * counts its positions with them, and page_table is [n_seqs][max_pages].
 * n_new, kv_len, page_table and tokens are host arrays, read before
 * the call returns.  Writes every
 * layer's K and V rows and logits[s][vocab] of each sequence's last token.  A
 * row of a page that two new tokens would write is refused.
 * The cache is F16 and has the model's layers, kv heads and head_dim.  rope
 * NULL: the model's theta on the whole head in halves.  window, sinks: as
 * tbq_attn_paged, in every layer.  One token of one sequence runs on the
 * decode step's matvecs (logits as exact as the fp16 cache lets them be),
 * more on the batched prefill's fp16 products, for models whose rows those hold
 * (tbq_dense_prefill_batched); others run one token after the other, logits of
 * each included.  Those products leave the logits within 1e-2 relative L2 (1.5e-3
 * at most in 300 prompts of one to three tokens) unless the weights' sums nearly
 * cancel: weights whose rows have a mean took 1 prompt in 100 to 1e-2 .. 8e-2.
 * The lm_head (weights within fp16's 65504) is as exact as the decode step's for
 * any number of sequences.  Two single tokens take longer in one step than in two
 * (Qwen3-4B's shape at 4096: 3.9 ms and 1.65 each), three less.
 * A captured call repeats its tokens, lengths and pages at every replay, so a
 * step is not for capture.
 * The workspace size covers every call with at most that many sequences, tokens
 * and pages; a larger one changes nothing.  n_tokens at most 65536, n_seqs at
 * most 1024. */
size_t tbq_dense_step_workspace_size(const tbq_dense_model *m, const tbq_kv_cache *c, int n_seqs, int n_tokens,
                                     int max_pages);
int tbq_dense_step(const tbq_dense_model *m, const tbq_kv_cache *c, int n_seqs, const int *n_new, const int *kv_len,
                   const int *page_table, int max_pages, const int *tokens, const tbq_rope *rope, int window,
                   int sinks, float *logits, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
