// tbq_paged_attn.hip -- causal attention of new tokens over the paged
// key/value cache (include/tbq_kv.h) on gfx950.
#include "tbq_kernels.h"
#include "tbq_paged.hpp"

namespace tbq {

// One wave per token and query head, a position at a time with the running
// maximum and sum of the softmax: lane l holds elements l and l + 64 of the
// head.
template <typename TA, typename TC, int D>
__global__ __launch_bounds__(64) void k_pg_attn_row(const PgAttn a) {
    const int h = blockIdx.x, t = blockIdx.y, lane = threadIdx.x;
    const int s = pg_seq_of(a.pg.q_start, a.pg.n_seqs, t);
    if (s >= a.pg.n_seqs || t < a.pg.q_start[s]) return;
    const int pos = a.pg.kv_len[s] - a.pg.q_start[s + 1] + t;
    const int kvh = h / (a.NQ / a.pg.NKV);
    const TA *q = (const TA *)a.q + t * a.qs + h * D;
    float qv[D / 64], o[D / 64] = {}, m = -3.402823466e38f, l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; i++) qv[i] = (float)q[lane + 64 * i];
    const int lo = a.window > 0 ? pos - a.window + 1 : 0;
    for (int p = 0; p <= pos; p++) {
        if (p < lo && p >= a.sinks) p = lo;
        const int page = pg_page(a.pg, s, p);
        if (page < 0) continue;
        const long long row = pg_row<D>(a.pg, page, kvh, p);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < D / 64; i++) dot += qv[i] * (float)((const TC *)a.pg.k)[row + lane + 64 * i];
        dot = group_sum<64>(dot) * a.scale;
        const float mn = fmaxf(m, dot), corr = __builtin_amdgcn_exp2f(m - mn), w = __builtin_amdgcn_exp2f(dot - mn);
        m = mn;
        l = l * corr + w;
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] = o[i] * corr + w * (float)((const TC *)a.pg.v)[row + lane + 64 * i];
    }
    TA *out = (TA *)a.out + ((long long)t * a.NQ + h) * D;
#pragma unroll
    for (int i = 0; i < D / 64; i++) out[lane + 64 * i] = (TA)(l > 0.f ? o[i] / l : l);
}

size_t pg_attn_workspace_bytes(const PgArgs &a, int D, int NQ, bool f32) {
    (void)a; (void)D; (void)NQ; (void)f32;
    return 0;
}

hipError_t launch_pg_attn(const PgAttn &a, int D, int q_type, int c_type, void *ws, size_t ws_bytes, hipStream_t st) {
    (void)ws; (void)ws_bytes;
    const dim3 grid(a.NQ, a.pg.n_tokens);
#define TBQ_AT(TA, TC)                                                                              \
    do {                                                                                            \
        if (D == 128) hipLaunchKernelGGL((k_pg_attn_row<TA, TC, 128>), grid, dim3(64), 0, st, a);   \
        else hipLaunchKernelGGL((k_pg_attn_row<TA, TC, 64>), grid, dim3(64), 0, st, a);             \
        return hipGetLastError();                                                                   \
    } while (0)
    if (q_type == TBQ_KV_F32) TBQ_AT(float, pg_f16);
    if (c_type == TBQ_KV_F16) TBQ_AT(pg_f16, pg_f16);
    TBQ_AT(pg_bf16, pg_bf16);
#undef TBQ_AT
}

}  // namespace tbq
