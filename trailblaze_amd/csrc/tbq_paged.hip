// tbq_paged.hip -- operators that move data of the paged key/value cache
// (include/tbq_kv.h) on gfx950: rotary positions with the append of new rows,
// page copies, and compaction of a sequence's kept rows.  Attention over the
// pages is in tbq_paged_attn.hip.
#include <string.h>

#include <algorithm>

#include "tbq_kernels.h"
#include "tbq_paged.hpp"

namespace tbq {

// ---------------------------------------------------------------------------
// Append.  x' = x * (1 / sqrt(mean(x^2) + eps)) * w per head, then every pair
// (u, w) of the first rot elements becomes m (u cos a - w sin a, u sin a + w
// cos a), a = position * freq[j]; q to q_out, k and v to the token's rows.
// The angle is formed in turns and reduced in fp64, so its error does not grow
// with the position.
//
// Bound by HBM (every element is read and written once).  D / 8 lanes hold a
// head, eight elements each as two groups of four (both elements of a pair in
// one lane): half layout 4j.. and rot / 2 + 4j.., interleaved 8j.. and 8j + 4..,
// and eight elements side by side behind rot.  A workgroup has one token and
// HPT times 16 (32) of its NQ + 2 NKV heads; a lane turns HPT heads by the
// four angles that it computed once.  8192 tokens of 32 + 8 + 8 heads of 128, fp32
// to fp16, 302 MB: 56 to 61 us (5.0 to 5.4 TB/s); one token 3.1 us.
// ---------------------------------------------------------------------------
constexpr int AP_THREADS = 256;
template <typename TI, typename TQ, typename TC, int D, int HPT, int TH>
__global__ __launch_bounds__(TH) void k_pg_append(const PgAppend a) {
    constexpr int LPH = D / 8, SL = TH / LPH;
    const int t = blockIdx.x, l = threadIdx.x % LPH, rot = a.rope.rot;
    const int nslots = a.NQ + 2 * a.pg.NKV;
    const int s = pg_seq_of(a.pg.q_start, a.pg.n_seqs, t);
    if (s >= a.pg.n_seqs) return;
    const int first = a.pg.q_start[s], last = a.pg.q_start[s + 1];
    const int pos = a.pg.kv_len[s] - last + t;
    if (t < first || pos < 0) return;
    const bool turn = 8 * l < rot;
    int oa = 8 * l, ob = 8 * l + 4;
    if (turn && !a.rope.interleaved) {
        oa = 4 * l;
        ob = rot / 2 + 4 * l;
    }
    // every head's elements are loaded before any is used
    float4 xa[HPT], xb[HPT];
    const float rs = a.rs ? a.rs[t] : 1.f;
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int hh = min((int)(blockIdx.y * HPT + i) * SL + (int)threadIdx.x / LPH, nslots - 1);
        const TI *x = hh < a.NQ              ? (const TI *)a.q + t * a.qs + hh * D
                      : hh < a.NQ + a.pg.NKV ? (const TI *)a.k + t * a.ks + (hh - a.NQ) * D
                                             : (const TI *)a.v + t * a.vs + (hh - a.NQ - a.pg.NKV) * D;
        xa[i] = pg_ld4(x + oa);
        xb[i] = pg_ld4(x + ob);
        if constexpr (sizeof(TI) == 4) {   // slices are added in slice order
            for (int z = 1; z < a.nsl; z++) {
                const float4 ya = pg_ld4(x + z * a.slstride + oa), yb = pg_ld4(x + z * a.slstride + ob);
                xa[i] = make_float4(xa[i].x + ya.x, xa[i].y + ya.y, xa[i].z + ya.z, xa[i].w + ya.w);
                xb[i] = make_float4(xb[i].x + yb.x, xb[i].y + yb.y, xb[i].z + yb.z, xb[i].w + yb.w);
            }
            xa[i] = make_float4(xa[i].x * rs, xa[i].y * rs, xa[i].z * rs, xa[i].w * rs);
            xb[i] = make_float4(xb[i].x * rs, xb[i].y * rs, xb[i].z * rs, xb[i].w * rs);
        }
    }
    const int page = pg_page(a.pg, s, pos);
    float cs[4], sn[4];
    if (turn) {
        const double p = a.positions ? a.positions[t] : pos;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const double turns = p * a.rope.turns[4 * l + j];
            float sj, cj;
            sincospif(2.f * (float)(turns - __builtin_rint(turns)), &sj, &cj);
            cs[j] = cj * a.rope.mscale;
            sn[j] = sj * a.rope.mscale;
        }
    }
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int hh = (int)(blockIdx.y * HPT + i) * SL + (int)threadIdx.x / LPH;
        const bool isv = hh >= a.NQ + a.pg.NKV;
        const float *w = hh < a.NQ ? a.qn : a.kn;
        float4 u = xa[i], v = xb[i];
        const float ss = group_sum<LPH>(u.x * u.x + u.y * u.y + u.z * u.z + u.w * u.w + v.x * v.x + v.y * v.y +
                                        v.z * v.z + v.w * v.w);
        if (hh >= nslots) continue;
        if (!isv && w) {
            const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
            const float4 wa = pg_ld4(w + oa), wb = pg_ld4(w + ob);
            u = make_float4(u.x * r * wa.x, u.y * r * wa.y, u.z * r * wa.z, u.w * r * wa.w);
            v = make_float4(v.x * r * wb.x, v.y * r * wb.y, v.z * r * wb.z, v.w * r * wb.w);
        }
        if (!isv && turn) {
            if (a.rope.interleaved) {
                u = make_float4(u.x * cs[0] - u.y * sn[0], u.x * sn[0] + u.y * cs[0], u.z * cs[1] - u.w * sn[1],
                                u.z * sn[1] + u.w * cs[1]);
                v = make_float4(v.x * cs[2] - v.y * sn[2], v.x * sn[2] + v.y * cs[2], v.z * cs[3] - v.w * sn[3],
                                v.z * sn[3] + v.w * cs[3]);
            } else {
                const float4 x = u, y = v;
                u = make_float4(x.x * cs[0] - y.x * sn[0], x.y * cs[1] - y.y * sn[1], x.z * cs[2] - y.z * sn[2],
                                x.w * cs[3] - y.w * sn[3]);
                v = make_float4(x.x * sn[0] + y.x * cs[0], x.y * sn[1] + y.y * cs[1], x.z * sn[2] + y.z * cs[2],
                                x.w * sn[3] + y.w * cs[3]);
            }
        }
        if (hh < a.NQ) {
            TQ *o = (TQ *)a.qo + ((long long)t * a.NQ + hh) * D;
            pg_st4(o + oa, u);
            pg_st4(o + ob, v);
        } else if (page >= 0) {
            const int kvh = isv ? hh - a.NQ - a.pg.NKV : hh - a.NQ;
            TC *o = (TC *)(isv ? a.pg.v : a.pg.k) + pg_row<D>(a.pg, page, kvh, pos);
            pg_st4(o + oa, u);
            pg_st4(o + ob, v);
        }
    }
}

template <typename TI, typename TQ, typename TC, int D>
static hipError_t append_d(const PgAppend &a, hipStream_t st) {
    constexpr int SL = AP_THREADS / (D / 8);
    const int nb = (a.NQ + 2 * a.pg.NKV + SL - 1) / SL;
    // Long prompts share the angles between up to three heads a lane: 8192 tokens, 48 heads of 128,
    // fp32 71 -> 61 us, bf16 67 -> 49; below about eight workgroups a CU one head a lane is as fast
    // (512 tokens) or faster (64 tokens 3.8 us, 4.8 with three).
    const int hpt = (long long)a.pg.n_tokens * nb >= 2048 ? std::min(nb, 3) : 1;
    const dim3 grid(a.pg.n_tokens, (nb + hpt - 1) / hpt);
    // Few heads (a shard of a model) leave most of a workgroup idle: one of 64 or 128 threads then.  12
    // prompts of 410 tokens, 4 + 1 + 1 heads of 64: 10.7 -> 6 us.
    const int th = nb > 1 ? AP_THREADS : (a.NQ + 2 * a.pg.NKV) * (D / 8);
    if (hpt == 3) hipLaunchKernelGGL((k_pg_append<TI, TQ, TC, D, 3, AP_THREADS>), grid, dim3(AP_THREADS), 0, st, a);
    else if (hpt == 2) hipLaunchKernelGGL((k_pg_append<TI, TQ, TC, D, 2, AP_THREADS>), grid, dim3(AP_THREADS), 0, st, a);
    else if (th <= 64) hipLaunchKernelGGL((k_pg_append<TI, TQ, TC, D, 1, 64>), grid, dim3(64), 0, st, a);
    else if (th <= 128) hipLaunchKernelGGL((k_pg_append<TI, TQ, TC, D, 1, 128>), grid, dim3(128), 0, st, a);
    else hipLaunchKernelGGL((k_pg_append<TI, TQ, TC, D, 1, AP_THREADS>), grid, dim3(AP_THREADS), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_pg_append(const PgAppend &a, int D, int in_type, int q_type, int c_type, hipStream_t st) {
#define TBQ_AP(TI, TQ, TC) return D == 128 ? append_d<TI, TQ, TC, 128>(a, st) : append_d<TI, TQ, TC, 64>(a, st)
    if (c_type == TBQ_KV_MXFP4) return launch_mx_append(a, D, in_type, q_type, st);
    const bool fi = in_type == TBQ_KV_F32, fq = q_type == TBQ_KV_F32;
    if (c_type == TBQ_KV_F16) {
        if (fi && fq) TBQ_AP(float, float, pg_f16);
        if (fi) TBQ_AP(float, pg_f16, pg_f16);
        TBQ_AP(pg_f16, pg_f16, pg_f16);
    }
    if (fi && fq) TBQ_AP(float, float, pg_bf16);
    if (fi) TBQ_AP(float, pg_bf16, pg_bf16);
    TBQ_AP(pg_bf16, pg_bf16, pg_bf16);
#undef TBQ_AP
}

// ---------------------------------------------------------------------------
// Page copies.  The pairs travel in the kernel's arguments, so the caller's
// lists are free when the call returns and nothing has to be staged.  A page
// of one layer of K or V is `pbytes` side by side; a workgroup copies CP_BYTES
// of it, past the caches (100 pages of 36 layers, 1.89 GB: 360 -> 295 to 343 us,
// 5.5 to 6.4 TB/s; 4 pages, 75 MB, 18.4 -> 15.5).  Bound by HBM.
// ---------------------------------------------------------------------------
constexpr int CP_THREADS = 256, CP_V = 8, CP_BYTES = CP_THREADS * CP_V * 16;
__global__ __launch_bounds__(CP_THREADS) void k_pg_copy(uint8_t *k, uint8_t *v, long long pbytes, long long lbytes,
                                                        const PgPairs pairs) {
    uint8_t *base = (blockIdx.y & 1 ? v : k) + (blockIdx.y >> 1) * lbytes;
    const uint8_t *src = base + pairs.src[blockIdx.z] * pbytes;
    uint8_t *dst = base + pairs.dst[blockIdx.z] * pbytes;
    const long long at = (long long)blockIdx.x * CP_BYTES + threadIdx.x * 16;
    pg_u4 r[CP_V];
#pragma unroll
    for (int i = 0; i < CP_V; i++)   // clamped: loads stay unconditional
        r[i] = __builtin_nontemporal_load(reinterpret_cast<const pg_u4 *>(src + min(at + i * CP_THREADS * 16, pbytes - 16)));
#pragma unroll
    for (int i = 0; i < CP_V; i++)
        if (at + i * CP_THREADS * 16 < pbytes) __builtin_nontemporal_store(r[i], reinterpret_cast<pg_u4 *>(dst + at + i * CP_THREADS * 16));
}

hipError_t launch_pg_copy(void *k, void *v, int n_layers, long long pbytes, long long lbytes, const PgPairs &pairs, int n,
                          hipStream_t st) {
    const dim3 grid((unsigned)((pbytes + CP_BYTES - 1) / CP_BYTES), 2 * n_layers, n);
    hipLaunchKernelGGL(k_pg_copy, grid, dim3(CP_THREADS), 0, st, (uint8_t *)k, (uint8_t *)v, pbytes, lbytes, pairs);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Compaction, in place: row j of a sequence becomes its row keep[j] >= j, keep
// ascending.  Rows are moved as columns of 128 bytes.  A workgroup has one
// sequence, layer, K or V, and hpw of the NKV * D / 64 columns (no other
// workgroup touches them) and goes through the kept rows a step of CO_UNITS / hpw
// at a time: all of a step's rows have arrived in every wave before any is
// stored, and a step's stores reach no row that a later step loads (keep[j'] >=
// j' > j), so the next step's rows are loaded before this one's are stored.
// Pages are looked up for CO_LIST rows at a time, into LDS: memory operations
// complete in order, so a lookup per step would have waited for all of the
// step's rows first.  16000 rows to 9001 in 36 layers, 4 heads of 128, 1.33 GB:
// 261 to 313 us (4.2 to 5.1 TB/s; 803 with a step's lookups, loads and stores in
// turn); 24 rows of 16 sequences to 9: 9.4 to 11 us, one step of each workgroup.
// ---------------------------------------------------------------------------
constexpr int CO_THREADS = 256, CO_V = 4, CO_UNITS = CO_THREADS / 8 * CO_V, CO_LIST = 1024;
template <int D>
__global__ __launch_bounds__(CO_THREADS) void k_pg_compact(uint16_t *k, uint16_t *v, long long lelems, const PgArgs a,
                                                           const int *__restrict__ keep_start,
                                                           const int *__restrict__ keep, int hpw) {
    constexpr int SL = D / 64;   // columns of a row
    __shared__ int src[2][CO_LIST], dst[2][CO_LIST];   // rows of head 0, dst -1: nothing to store
    const int s = blockIdx.z, l = threadIdx.x % 8, u0 = threadIdx.x / 8, c0 = blockIdx.x * hpw;
    const int jr = CO_UNITS / hpw, lr = CO_LIST / jr * jr;   // rows of a step, of a list
    uint16_t *base = (blockIdx.y & 1 ? v : k) + (blockIdx.y >> 1) * lelems + 8 * l;
    const int at = keep_start[s], n = keep_start[s + 1] - at;
    if (n <= 0) return;
    auto look_up = [&](int j0) {
        const int b = j0 / lr & 1;
#pragma unroll
        for (int i = 0; i < CO_LIST / CO_THREADS; i++) {
            if (CO_THREADS * i >= n - j0 + jr) break;   // past the last step (uniform)
            const int e = threadIdx.x + CO_THREADS * i, j = j0 + e, jc = min(j, n - 1);
            const int from = keep[at + jc], p = max(from, 0), ps = pg_page(a, s, p), pd = pg_page(a, s, jc);
            const bool moves = j < n && from >= 0 && p != j && ps >= 0 && pd >= 0;
            // a row that does not move is loaded from where it is (or page 0) and not stored
            src[b][e] = (int)(pg_row<1>(a, max(ps, 0), 0, p));
            dst[b][e] = moves ? (int)(pg_row<1>(a, pd, 0, jc)) : -1;
        }
    };
    // unit u of a step: row u % jr, column c0 + u / jr
    int uj[CO_V];
    long long uc[CO_V];   // elements between row 0 of head 0 and of the column; -1: no unit
#pragma unroll
    for (int i = 0; i < CO_V; i++) {
        const int u = i * (CO_THREADS / 8) + u0, c = u / jr, cc = c0 + min(c, hpw - 1);
        uj[i] = u % jr;
        uc[i] = (((long long)(cc / SL) << a.shift) * D + 64 * (cc % SL)) | (c < hpw ? 0 : 1);
    }
    pg_u4 r[2][CO_V];
    auto load = [&](int b, int j0) {
#pragma unroll
        for (int i = 0; i < CO_V; i++)
            r[b][i] = *reinterpret_cast<const pg_u4 *>(base + (uc[i] & ~1ll) + (long long)src[j0 / lr & 1][j0 % lr + uj[i]] * D);
    };
    auto store = [&](int b, int j0) {
#pragma unroll
        for (int i = 0; i < CO_V; i++) {
            const int to = uc[i] & 1 ? -1 : dst[j0 / lr & 1][j0 % lr + uj[i]];
            if (to >= 0) *reinterpret_cast<pg_u4 *>(base + uc[i] + (long long)to * D) = r[b][i];
        }
    };
    auto step = [&](int b, int j0) {
        // every wave's rows have arrived, and it is done with the list before this one
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (j0 + jr < n) load(b ^ 1, j0 + jr);
        store(b, j0);
        if (j0 % lr == 0 && j0 + lr < n) look_up(j0 + lr);   // a list (of two steps or more) ahead
    };
    look_up(0);
    __syncthreads();
    load(0, 0);
    for (int j0 = 0; j0 < n; j0 += 2 * jr) {   // uniform
        step(0, j0);
        if (j0 + jr < n) step(1, j0 + jr);
    }
}

// Columns of a workgroup: all, or as many as leave about four workgroups a CU
// (many short sequences: one step does it all, and the lookups are shared).
hipError_t launch_pg_compact(void *k, void *v, int n_layers, long long lelems, int D, const PgArgs &a, const int *keep_start,
                             const int *keep, hipStream_t st) {
    const int cols = a.NKV * (D / 64);
    int hpw = 1;
    for (int h = 2; h <= cols && h <= 64; h++)
        if (cols % h == 0 && (long long)a.n_seqs * 2 * n_layers * (cols / h) >= 1024) hpw = h;
    const dim3 grid(cols / hpw, 2 * n_layers, a.n_seqs);
    if (D == 128)
        hipLaunchKernelGGL(k_pg_compact<128>, grid, dim3(CO_THREADS), 0, st, (uint16_t *)k, (uint16_t *)v, lelems, a,
                           keep_start, keep, hpw);
    else
        hipLaunchKernelGGL(k_pg_compact<64>, grid, dim3(CO_THREADS), 0, st, (uint16_t *)k, (uint16_t *)v, lelems, a,
                           keep_start, keep, hpw);
    return hipGetLastError();
}

// Host ints to the device in the kernel's arguments.
constexpr int PUT_INTS = 960;
struct PgInts {
    int v[PUT_INTS];
};
__global__ __launch_bounds__(PUT_INTS) void k_pg_put(int *dst, const PgInts src, int n) {
    if ((int)threadIdx.x < n) dst[threadIdx.x] = src.v[threadIdx.x];
}

hipError_t launch_put_ints(int *dst, const int *src, long long n, hipStream_t st) {
    for (long long i = 0; i < n; i += PUT_INTS) {
        PgInts v;
        const int m = (int)(n - i < PUT_INTS ? n - i : PUT_INTS);
        memcpy(v.v, src + i, m * sizeof(int));
        hipLaunchKernelGGL(k_pg_put, dim3(1), dim3(PUT_INTS), 0, st, dst + i, v, m);
    }
    return hipGetLastError();
}

}  // namespace tbq
