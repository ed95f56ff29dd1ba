// tbq_paged.hpp -- what the kernels over the paged key/value cache share
// (include/tbq_kv.h): the arguments that describe cache and batch, and the
// lookups of a token's sequence and of a position's row.
#pragma once

#include <math.h>

#include "tbq_device.hpp"
#include "../../include/tbq_kv.h"

namespace tbq {

// One layer of a cache, and a batch.
struct PgArgs {
    void *k, *v;           // the layer's [n_pages][NKV][1 << shift][D]
    int n_pages, NKV, shift;
    int n_seqs, n_tokens, max_pages, max_q, max_kv;
    const int *q_start, *kv_len, *table;
};

struct PgRope {
    int rot, interleaved;
    float mscale;
    double turns[64];      // freq[j] / 2 pi
};

inline void pg_rope(const tbq_rope &r, PgRope &o) {
    o.rot = r.rot_dim;
    o.interleaved = r.layout == TBQ_ROPE_INTERLEAVED;
    o.mscale = (float)r.mscale;
    for (int j = 0; j < r.rot_dim / 2; j++) o.turns[j] = r.freq[j] * 0.15915494309189533577;
}

struct PgAppend {
    PgArgs pg;
    const void *q, *k, *v;             // heads of row t side by side at base + t * stride
    long long qs, ks, vs;
    void *qo;                          // [n_tokens][NQ][D]
    const float *qn, *kn;              // norm weights, or null
    const int *positions;              // rotation positions, or null
    float eps;
    int NQ;                            // 0: k and v only
    // the dense prefill's products: row t is scaled by 1 / rs[t], and the rows
    // are nsl split-K slices (slice z at base + z * slstride)
    const float *rs;
    int nsl;
    long long slstride;
    PgRope rope;
};

struct PgAttn {
    PgArgs pg;
    const void *q;         // heads of row t side by side at base + t * stride
    long long qs;
    void *out;             // [n_tokens][NQ][D], of q's type or (f32_out) fp32
    int NQ, window, sinks, f32_out;
    int few;               // rows up to which a sequence is one of few rows (launch_pg_attn sets it)
    float scale;           // of q . k, times log2(e): the softmax is in powers of two
};

// The scale of q . k times log2(e); 0 stands for 1 / sqrt(D).
inline float pg_scale(float scale, int D) { return (scale > 0 ? scale : 1.0f / sqrtf((float)D)) * 1.4426950408889634f; }

// Differences of positions and windows stay in 32 bits.
inline int pg_window(int n) { return n < (1 << 30) ? n : 1 << 30; }

inline int pg_log2(int n) {
    int s = 0;
    while ((1 << s) < n) s++;
    return s;
}

// Layer `layer` of a cache.
inline PgArgs pg_layer(const tbq_kv_cache *c, int layer) {
    PgArgs a{};
    const long long off = (long long)layer * c->n_pages * c->n_kv_heads * c->page_size * c->head_dim;
    a.k = (uint16_t *)c->k + off;
    a.v = (uint16_t *)c->v + off;
    a.n_pages = c->n_pages;
    a.NKV = c->n_kv_heads;
    a.shift = pg_log2(c->page_size);
    return a;
}

constexpr int PG_PAIRS = 128;   // page copies per launch, 1 KiB of kernel arguments
struct PgPairs {
    int src[PG_PAIRS], dst[PG_PAIRS];
};

// The sequence of token row t: the number of sequences that end at or before
// it (n_seqs: none).  The whole wave calls it; uniform.  Each round asks for every
// step-th end, a lane each (4096 single tokens appended: 64 us with 64 rounds of
// 64 ends side by side, 27 with two).
__device__ __forceinline__ int pg_seq_of(const int *__restrict__ q_start, int n_seqs, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n_seqs;
    while (lo < hi) {
        const int step = (hi - lo + 63) >> 6, i = lo + (lane + 1) * step - 1;
        const bool ends = i < hi && q_start[i + 1] <= t;
        lo += __builtin_popcountll(__builtin_amdgcn_ballot_w64(ends)) * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// The page of position p (>= 0) of sequence s, -1 where it has none.
__device__ __forceinline__ int pg_page(const PgArgs &a, int s, int p) {
    const int e = p >> a.shift;
    if (e >= a.max_pages) return -1;
    const int page = a.table[(long long)s * a.max_pages + e];
    return (unsigned)page < (unsigned)a.n_pages ? page : -1;
}

// Elements before row (p mod page size) of kv head h in a page.
template <int D>
__device__ __forceinline__ long long pg_row(const PgArgs &a, int page, int h, int p) {
    return ((((long long)page * a.NKV + h) << a.shift) + (p & ((1 << a.shift) - 1))) * D;
}

typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));   // 16 bytes moved as they are
typedef __bf16 pg_bf16;
typedef _Float16 pg_f16;

// Four elements as floats, and back (one rounding, to nearest even).
template <typename T>
__device__ __forceinline__ float4 pg_ld4(const T *p) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    const v4 v = *reinterpret_cast<const v4 *>(p);
    return make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
}
template <typename T>
__device__ __forceinline__ void pg_st4(T *p, float4 f) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4 *>(p) = v4{(T)f.x, (T)f.y, (T)f.z, (T)f.w};
}

// Launchers (tbq_paged.hip, tbq_paged_attn.hip).
hipError_t launch_pg_append(const PgAppend &a, int D, int in_type, int q_type, int c_type, hipStream_t st);
hipError_t launch_pg_copy(void *k, void *v, int n_layers, long long pbytes, long long lbytes, const PgPairs &pairs, int n,
                          hipStream_t st);
hipError_t launch_pg_compact(void *k, void *v, int n_layers, long long lelems, int D, const PgArgs &a, const int *keep_start,
                             const int *keep, hipStream_t st);
size_t pg_attn_workspace_bytes(const PgArgs &a, int D, int NQ, bool f32);
// at least that of every batch of up to n_seqs sequences, n_tokens tokens and max_kv positions
size_t pg_attn_workspace_upto(int n_seqs, int n_tokens, int max_kv, int NKV, int D, int NQ, bool f32);
// One token of one sequence (tbq_dense.hip), a batch of sequences (tbq_dense_prefill.hip).
hipError_t launch_dense_decode_paged(const tbq_dense_model *m, int token, const PgArgs &pg, size_t layer_bytes,
                                     const PgRope &rope, int window, int sinks, float *logits, void *ws, void *attn_ws,
                                     hipStream_t st);
size_t dense_step_workspace_bytes(const tbq_dense_model *m, const tbq_kv_cache *c, int n_seqs, int T, int max_pages);
bool dense_step_attn_fits(const tbq_dense_model *m, const tbq_kv_cache *c, int n_seqs, const int *n_new, const int *kv_len,
                          int max_pages);
hipError_t launch_dense_step(const tbq_dense_model *m, const tbq_kv_cache *c, int n_seqs, const int *n_new,
                             const int *kv_len, const int *page_table, int max_pages, const int *tokens,
                             const tbq_rope &rope, int window, int sinks, float *logits, void *ws, size_t ws_bytes,
                             hipStream_t st);
// *dst = n host ints, through kernel arguments (the host array is free at once)
hipError_t launch_put_ints(int *dst, const int *src, long long n, hipStream_t st);
hipError_t launch_pg_attn(const PgAttn &a, int D, int q_type, int c_type, void *ws, hipStream_t st);

}  // namespace tbq
