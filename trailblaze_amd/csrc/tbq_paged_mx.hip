// tbq_paged_mx.hip -- operators that move data of a paged key/value cache held
// in MXFP4 (tbq_mx.hpp): append with rotary positions, pages back to values, and
// compaction of a sequence's kept rows.  Attention over such pages is in
// tbq_paged_mx_attn.hip; page copies are bytes (tbq_paged.hip).
#include <algorithm>
#include <type_traits>

#include "tbq_kernels.h"
#include "tbq_mx.hpp"

namespace tbq {

// 1 / sqrt(x): from fp32's by Newton's iteration, twice (1e-7, 1e-14, then fp64's own).
__device__ __forceinline__ double mx_rsqrt(double x) {
    if (!(x > 1e-30 && x < 1e30)) return 1. / sqrt(x);
    double r = (double)(1.0f / sqrtf((float)x));
    r = r * fma(-0.5 * x * r, r, 1.5);
    return r * fma(-0.5 * x * r, r, 1.5);
}

// Eight values side by side, of the four lanes that share a block of 32: the codes,
// and the block's scale byte.  A value that is not finite makes the block NaN.
__device__ __forceinline__ uint32_t mx_block(const float (&x)[8], uint32_t *scale) {
    float a = 0.f, odd = 0.f;   // odd: NaN where a value is not finite
#pragma unroll
    for (int i = 0; i < 8; i++) {
        a = fmaxf(a, fabsf(x[i]));
        odd += x[i] - x[i];
    }
    a = fmaxf(a, dpp_f32<DPP_QXOR1>(a));
    a = fmaxf(a, dpp_f32<DPP_QXOR2>(a));
    odd += dpp_f32<DPP_QXOR1>(odd);
    odd += dpp_f32<DPP_QXOR2>(odd);
    const bool fine = odd == 0.f;
    const int E = mx_exponent(a);
    *scale = fine ? E + 127 : MX_NAN;
    return fine ? mx_codes(x, mx_scale(E + 127)) : 0u;
}

// ---------------------------------------------------------------------------
// Append: k_pg_append's norms and rotation, then the blocks' scales and codes.
// Keys are formed in fp64, from the norm's sum and the angles on: which of two codes
// a value becomes is decided at borders, where an fp32 error of 1e-7 would make
// the cache's bytes depend on the order of a sum.  q is fp32, as over 16-bit pages.
//
// A workgroup has one token and HPT times 16 (32) of its NQ + 2 NKV heads; D / 8
// lanes hold a head, eight elements each.  One lane a pair forms an angle; rotated
// keys go through LDS to lanes of eight elements side by side.
//
// 8191 tokens, 32 / 8 heads of 128, fp32 -> fp16: 57 us, 4.8 TB/s of rows in and out, a
// large copy's rate.  1 / sqrt in fp64 by two Newton steps from fp32's (the compiler's
// division and root: 62 us).  One token: 4.1-4.4 us, a chain of q_start, the rows, the
// angles' sine and cosine in fp64 and the stores.
// ---------------------------------------------------------------------------
constexpr int MA_THREADS = 256;
template <typename TI, typename TQ, int D, int HPT>
__global__ __launch_bounds__(MA_THREADS) void k_mx_append(const PgAppend a) {
    constexpr int LPH = D / 8, SL = MA_THREADS / LPH;
    __shared__ double cs[D / 2], sn[D / 2];
    __shared__ __attribute__((aligned(16))) float kx[SL][D];
    // Sixteen tokens side by side go to one XCD's workgroups, one after the other: they write into the same lines
    // (four positions of V share each), which one L2 then holds (8191 tokens: 62.7 -> 61.2 us).
    constexpr int XCDS = 8, RUN = 16;
    const int run0 = blockIdx.x / (XCDS * RUN) * (XCDS * RUN), in_run = blockIdx.x - run0;
    const int t = run0 + XCDS * RUN <= (int)gridDim.x ? run0 + in_run % XCDS * RUN + in_run / XCDS : (int)blockIdx.x;
    const int l = threadIdx.x % LPH, rot = a.rope.rot, slot = threadIdx.x / LPH;
    const int nslots = a.NQ + 2 * a.pg.NKV;
    const int s = pg_seq_of(a.pg.q_start, a.pg.n_seqs, t);
    if (s >= a.pg.n_seqs) return;
    const int first = a.pg.q_start[s], last = a.pg.q_start[s + 1];
    const int pos = a.pg.kv_len[s] - last + t;
    if (t < first || pos < 0) return;
    const bool turn = 8 * l < rot;
    int oa = 8 * l, ob = 8 * l + 4;   // of q and k; v's are side by side
    if (turn && !a.rope.interleaved) {
        oa = 4 * l;
        ob = rot / 2 + 4 * l;
    }
    float4 xa[HPT], xb[HPT];
    const float rs = a.rs ? a.rs[t] : 1.f;
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int hh = min((int)(blockIdx.y * HPT + i) * SL + slot, nslots - 1);
        const bool isv = hh >= a.NQ + a.pg.NKV;
        const int pa = isv ? 8 * l : oa, pb = isv ? 8 * l + 4 : ob;
        const TI *x = hh < a.NQ ? (const TI *)a.q + t * a.qs + hh * D
                      : !isv    ? (const TI *)a.k + t * a.ks + (hh - a.NQ) * D
                                : (const TI *)a.v + t * a.vs + (hh - a.NQ - a.pg.NKV) * D;
        xa[i] = pg_ld4(x + pa);
        xb[i] = pg_ld4(x + pb);
        if constexpr (sizeof(TI) == 4) {   // slices are added in slice order
            for (int z = 1; z < a.nsl; z++) {
                const float4 ya = pg_ld4(x + z * a.slstride + pa), yb = pg_ld4(x + z * a.slstride + pb);
                xa[i] = make_float4(xa[i].x + ya.x, xa[i].y + ya.y, xa[i].z + ya.z, xa[i].w + ya.w);
                xb[i] = make_float4(xb[i].x + yb.x, xb[i].y + yb.y, xb[i].z + yb.z, xb[i].w + yb.w);
            }
            xa[i] = make_float4(xa[i].x * rs, xa[i].y * rs, xa[i].z * rs, xa[i].w * rs);
            xb[i] = make_float4(xb[i].x * rs, xb[i].y * rs, xb[i].z * rs, xb[i].w * rs);
        }
    }
    const int page = pg_page(a.pg, s, pos), in = pos & ((1 << a.pg.shift) - 1);
    if ((int)threadIdx.x < rot / 2) {
        const double turns = (a.positions ? a.positions[t] : pos) * a.rope.turns[threadIdx.x];
        double sj, cj;
        sincospi(2. * (turns - __builtin_rint(turns)), &sj, &cj);
        cs[threadIdx.x] = cj * a.rope.mscale64;
        sn[threadIdx.x] = sj * a.rope.mscale64;
    }
    __syncthreads();
    // the lane's four pairs: elements j and j + 4, or (interleaved) 2 j and 2 j + 1
    auto rotate = [&](auto (&y)[8]) {
        typedef std::remove_reference_t<decltype(y[0])> F;
        auto turn_pair = [&](F &u, F &w, int j) {
            const F c = (F)cs[4 * l + j], n = (F)sn[4 * l + j], x = u;
            u = x * c - w * n;
            w = x * n + w * c;
        };
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (a.rope.interleaved) turn_pair(y[2 * j], y[2 * j + 1], j);
            else turn_pair(y[j], y[j + 4], j);
        }
    };
#pragma unroll
    for (int i = 0; i < HPT; i++) {
        const int hh = (int)(blockIdx.y * HPT + i) * SL + slot;
        const bool isq = hh < a.NQ, isv = hh >= a.NQ + a.pg.NKV;
        float x[8] = {xa[i].x, xa[i].y, xa[i].z, xa[i].w, xb[i].x, xb[i].y, xb[i].z, xb[i].w};
        if (hh >= nslots) continue;
        if (isq) {
            float y[8], ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = x[e];
                ss += x[e] * x[e];
            }
            if (a.qn) {
                ss = group_sum<LPH>(ss);
                const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
                const float4 wa = pg_ld4(a.qn + oa), wb = pg_ld4(a.qn + ob);
                const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = y[e] * r * w[e];
            }
            if (turn) rotate(y);
            TQ *o = (TQ *)a.qo + ((long long)t * a.NQ + hh) * D;
            pg_st4(o + oa, make_float4(y[0], y[1], y[2], y[3]));
            pg_st4(o + ob, make_float4(y[4], y[5], y[6], y[7]));
            continue;
        }
        const int kvh = isv ? hh - a.NQ - a.pg.NKV : hh - a.NQ;
        float v[8];
        if (isv) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = x[e];
        } else {
            double y[8], ss = 0.;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = x[e];
                ss = fma(y[e], y[e], ss);
            }
            if (a.kn) {
                const double r = mx_rsqrt(group_sum<LPH>(ss) / D + (double)a.eps);
                const float4 wa = pg_ld4(a.kn + oa), wb = pg_ld4(a.kn + ob);
                const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = y[e] * r * w[e];
            }
            if (turn) rotate(y);
            // to eight elements side by side (the head's lanes are of one wave)
            float *row = kx[slot];
            *reinterpret_cast<float4 *>(row + oa) = make_float4(mx_odd(y[0]), mx_odd(y[1]), mx_odd(y[2]), mx_odd(y[3]));
            *reinterpret_cast<float4 *>(row + ob) = make_float4(mx_odd(y[4]), mx_odd(y[5]), mx_odd(y[6]), mx_odd(y[7]));
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const float4 va = *reinterpret_cast<const float4 *>(row + 8 * l), vb = *reinterpret_cast<const float4 *>(row + 8 * l + 4);
            __builtin_amdgcn_wave_barrier();
            v[0] = va.x, v[1] = va.y, v[2] = va.z, v[3] = va.w, v[4] = vb.x, v[5] = vb.y, v[6] = vb.z, v[7] = vb.w;
        }
        uint32_t scale;
        const uint32_t codes = mx_block(v, &scale);
        if (page < 0) continue;
        uint8_t *o = (uint8_t *)(isv ? a.pg.v : a.pg.k) + mx_head<D>(a.pg, page, kvh), *sc = o + ((D / 2) << a.pg.shift);
        *reinterpret_cast<uint32_t *>(o + (isv ? mx_v_code<D>(in, l) : mx_k_code<D>(in, l))) = codes;
        if (l % 4 == 0) sc[isv ? mx_v_scale<D>(in, l / 4) : mx_k_scale<D>(in, l / 4)] = (uint8_t)scale;
    }
}

template <typename TI, typename TQ, int D>
static hipError_t mx_append_d(const PgAppend &a, hipStream_t st) {
    constexpr int SL = MA_THREADS / (D / 8);
    const int nb = (a.NQ + 2 * a.pg.NKV + SL - 1) / SL;
    const int hpt = (long long)a.pg.n_tokens * nb >= 2048 ? std::min(nb, 3) : 1;
    const dim3 grid(a.pg.n_tokens, (nb + hpt - 1) / hpt);
    if (hpt == 3) hipLaunchKernelGGL((k_mx_append<TI, TQ, D, 3>), grid, dim3(MA_THREADS), 0, st, a);
    else if (hpt == 2) hipLaunchKernelGGL((k_mx_append<TI, TQ, D, 2>), grid, dim3(MA_THREADS), 0, st, a);
    else hipLaunchKernelGGL((k_mx_append<TI, TQ, D, 1>), grid, dim3(MA_THREADS), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_mx_append(const PgAppend &a, int D, int in_type, int q_type, hipStream_t st) {
#define TBQ_AP(TI, TQ) return D == 128 ? mx_append_d<TI, TQ, 128>(a, st) : mx_append_d<TI, TQ, 64>(a, st)
    if (in_type == TBQ_KV_F16) TBQ_AP(pg_f16, pg_f16);
    if (in_type == TBQ_KV_BF16) TBQ_AP(pg_bf16, pg_bf16);
    if (q_type == TBQ_KV_F16) TBQ_AP(float, pg_f16);
    if (q_type == TBQ_KV_BF16) TBQ_AP(float, pg_bf16);
    TBQ_AP(float, float);
#undef TBQ_AP
}

// ---------------------------------------------------------------------------
// Pages back to values: out [pages][NKV][page size][D].  A lane has eight dims of a
// position, 64 lanes four positions in V's order of the codes, so its dwords are
// read side by side and whole lines are written.  Bound by HBM (the values' bytes).
// ---------------------------------------------------------------------------
constexpr int MD_THREADS = 256;
template <typename TO, int D, int ROUNDS>
__global__ __launch_bounds__(MD_THREADS) void k_mx_dequant(const PgArgs a, const int *__restrict__ pages, TO *k, TO *v) {
    constexpr int LPR = D / 8, RPW = MD_THREADS / LPR;   // rows of a workgroup's round
    const int g = threadIdx.x / 4 % LPR, r = threadIdx.x / (4 * LPR) * 4 + threadIdx.x % 4;
    const int rows = 1 << a.shift, chunks = (rows + RPW * ROUNDS - 1) / (RPW * ROUNDS);
    const int n = blockIdx.x / chunks, h = blockIdx.y, page = pages ? pages[n] : n;
    const bool there = (unsigned)page < (unsigned)a.n_pages;
    const long long from = mx_head<D>(a, there ? page : 0, h), to = ((long long)n * a.NKV + h) << a.shift;
    const int codes = (D / 2) << a.shift, r0 = blockIdx.x % chunks * RPW * ROUNDS + r;
    const uint8_t *kp = (const uint8_t *)a.k + from, *vp = (const uint8_t *)a.v + from;
    uint32_t kc[ROUNDS], vc[ROUNDS], ks[ROUNDS], vs[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int in = min(r0 + RPW * i, rows - 1);
        kc[i] = *reinterpret_cast<const uint32_t *>(kp + mx_k_code<D>(in, g));
        vc[i] = *reinterpret_cast<const uint32_t *>(vp + mx_v_code<D>(in, g));
        ks[i] = kp[codes + mx_k_scale<D>(in, g / 4)];
        vs[i] = vp[codes + mx_v_scale<D>(in, g / 4)];
    }
    typedef TO out8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int in = r0 + RPW * i;
        if (in >= rows) break;
        const mx_h8 x = mx_eight(there ? kc[i] : 0u, mx_scale(there ? ks[i] : 0u));
        const mx_h8 y = mx_eight(there ? vc[i] : 0u, mx_scale(there ? vs[i] : 0u));
        out8 xo, yo;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            xo[e] = (TO)(float)x[e];
            yo[e] = (TO)(float)y[e];
        }
        *reinterpret_cast<out8 *>(k + (to + in) * D + 8 * g) = xo;
        *reinterpret_cast<out8 *>(v + (to + in) * D + 8 * g) = yo;
    }
}

template <typename TO, int D, int ROUNDS>
static void mx_dequant(const PgArgs &a, const int *pages, int n, void *k, void *v, hipStream_t st) {
    constexpr int rows = MD_THREADS / (D / 8) * ROUNDS;
    const dim3 grid((unsigned)n * (((1 << a.shift) + rows - 1) / rows), a.NKV);
    hipLaunchKernelGGL((k_mx_dequant<TO, D, ROUNDS>), grid, dim3(MD_THREADS), 0, st, a, pages, (TO *)k, (TO *)v);
}

hipError_t launch_mx_dequant(const PgArgs &a, int D, const int *pages, int n, int out_type, void *k, void *v,
                             hipStream_t st) {
    // Up to four rounds a workgroup, their loads in flight together, where there are many rows and a page has as many: fp16,
    // 8192 positions of 8 heads of 128 in one / two / four: pages of 64 9.2 / 8.0 / 8.2 us (8.9 MB in, 33.6 out: 5.2 TB/s), of
    // 32 9.05 / 8.1 / 8.7, of 16 9.0 / 9.4 / 10.4; heads of 64, pages of 64 5.8 / 5.7 / 6.0, of 16 6.05 / 6.3 / 6.9, 40000
    // positions in pages of 256 17.9 in one, 15.5 in four.  One round where there are few: 64 positions 2.6-2.9 us, a chain of
    // a page's number, codes and stores.
    const int of_page = (1 << a.shift) / (MD_THREADS / (D / 8));
    const int rounds = (long long)n * a.NKV << a.shift >= 1 << 15 ? std::min(of_page, 4) : 1;
#define TBQ_MD_D(TO, D)                                                   \
    if (rounds == 4) mx_dequant<TO, D, 4>(a, pages, n, k, v, st);         \
    else if (rounds == 2) mx_dequant<TO, D, 2>(a, pages, n, k, v, st);    \
    else mx_dequant<TO, D, 1>(a, pages, n, k, v, st)
#define TBQ_MD(TO)              \
    if (D == 128) {             \
        TBQ_MD_D(TO, 128);      \
    } else {                    \
        TBQ_MD_D(TO, 64);       \
    }
    if (out_type == TBQ_KV_F32) {
        TBQ_MD(float)
    } else if (out_type == TBQ_KV_F16) {
        TBQ_MD(pg_f16)
    } else {
        TBQ_MD(pg_bf16)
    }
#undef TBQ_MD
#undef TBQ_MD_D
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Compaction, in place: row j of a sequence becomes its row keep[j] >= j, keep
// ascending.  A workgroup has one sequence, layer, kv head and K or V (no other
// touches its rows) and moves MC_ROWS rows a step: all of them have arrived in every
// wave before any is stored, and no later step loads a row that this one stores.
// Bound by a step's chain of lookups, loads and stores: in 36 layers, 16000 rows of one sequence to 9001,
// 4 heads of 128, 321 us (fp16 pages, four times the bytes: 315; the bytes alone 75), 16 x 24 to 9, 8 heads,
// 17 (14); HBM where sequences are many: 64 x 1000 to 600, 8 heads of 128 903 us (2182), heads of 64 in
// pages of 16 569 (1169).
// ---------------------------------------------------------------------------
constexpr int MC_THREADS = 256, MC_ROWS = 64;
template <int D>
__global__ __launch_bounds__(MC_THREADS) void k_mx_compact(uint8_t *k, uint8_t *v, long long lbytes, const PgArgs a,
                                                           const int *__restrict__ keep_start,
                                                           const int *__restrict__ keep) {
    constexpr int GR = D / 8, N = MC_ROWS * GR / MC_THREADS;   // dwords of a row, of a thread
    __shared__ int src[MC_ROWS], dst[MC_ROWS];   // page and row in it, as page << shift | row; dst -1: stays
    const int h = blockIdx.x, s = blockIdx.z, isv = blockIdx.y & 1;
    uint8_t *base = (isv ? v : k) + (blockIdx.y >> 1) * lbytes;
    const int at = keep_start[s], n = keep_start[s + 1] - at, mask = (1 << a.shift) - 1, codes = (D / 2) << a.shift;
    auto head = [&](int row) { return base + mx_head<D>(a, row >> a.shift, h); };
    auto code = [&](int in, int g) { return isv ? mx_v_code<D>(in, g) : mx_k_code<D>(in, g); };
    auto scale = [&](int in, int b) { return codes + (isv ? mx_v_scale<D>(in, b) : mx_k_scale<D>(in, b)); };
    for (int j0 = 0; j0 < n; j0 += MC_ROWS) {   // uniform
        if (threadIdx.x < MC_ROWS) {
            const int j = j0 + threadIdx.x, jc = min(j, n - 1), from = keep[at + jc], p = max(from, 0);
            const int ps = pg_page(a, s, p), pd = pg_page(a, s, jc);
            const bool moves = j < n && from >= 0 && p != j && ps >= 0 && pd >= 0;
            src[threadIdx.x] = max(ps, 0) << a.shift | (p & mask);
            dst[threadIdx.x] = moves ? pd << a.shift | (jc & mask) : -1;
        }
        __syncthreads();
        uint32_t x[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int u = threadIdx.x + MC_THREADS * i, row = src[u / GR];
            x[i] = *reinterpret_cast<const uint32_t *>(head(row) + code(row & mask, u % GR));
        }
        const int br = threadIdx.x / (D / 32), b = threadIdx.x % (D / 32);   // (D = 64: the upper half has none)
        const int brow = br < MC_ROWS ? src[br] : -1;
        const uint8_t sc = brow >= 0 ? head(brow)[scale(brow & mask, b)] : 0;
        asm volatile("s_waitcnt vmcnt(0)" ::"v"(x[0]), "v"((uint32_t)sc) : "memory");
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int u = threadIdx.x + MC_THREADS * i, row = dst[u / GR];
            if (row >= 0) *reinterpret_cast<uint32_t *>(head(row) + code(row & mask, u % GR)) = x[i];
        }
        if (br < MC_ROWS && dst[br] >= 0) head(dst[br])[scale(dst[br] & mask, b)] = sc;
        __syncthreads();   // the lists are rewritten
    }
}

hipError_t launch_mx_compact(void *k, void *v, int n_layers, long long lbytes, int D, const PgArgs &a,
                             const int *keep_start, const int *keep, hipStream_t st) {
    const dim3 grid(a.NKV, 2 * n_layers, a.n_seqs);
    if (D == 128)
        hipLaunchKernelGGL(k_mx_compact<128>, grid, dim3(MC_THREADS), 0, st, (uint8_t *)k, (uint8_t *)v, lbytes, a,
                           keep_start, keep);
    else
        hipLaunchKernelGGL(k_mx_compact<64>, grid, dim3(MC_THREADS), 0, st, (uint8_t *)k, (uint8_t *)v, lbytes, a,
                           keep_start, keep);
    return hipGetLastError();
}

}  // namespace tbq
