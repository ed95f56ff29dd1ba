// tbq_paged_mx.hip -- operators that move data of a paged key/value cache held
// in MXFP4 (tbq_mx.hpp): append with rotary positions, pages back to values, and
// compaction of a sequence's kept rows.  Attention over such pages is in
// tbq_paged_mx_attn.hip; page copies are bytes (tbq_paged.hip).
#include <algorithm>
#include <type_traits>

#include "tbq_kernels.h"
#include "tbq_mx.hpp"

namespace tbq {

template <typename F, int WIDTH>
__device__ __forceinline__ F mx_group_max(F v) {
#pragma unroll
    for (int d = 1; d < WIDTH; d *= 2) {
        const F o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}
template <int WIDTH>
__device__ __forceinline__ double mx_group_sum(double v) {
#pragma unroll
    for (int d = 1; d < WIDTH; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// Eight values side by side, of the four lanes that share a block of 32: the codes,
// and the block's scale byte.  A value that is not finite makes the block NaN.
template <typename F>
__device__ __forceinline__ uint32_t mx_block(const F (&x)[8], uint32_t *scale) {
    F a = 0;
    int odd = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const F m = x[i] < 0 ? -x[i] : x[i];
        odd |= !(m < F(__builtin_huge_val()));
        a = m > a ? m : a;
    }
    a = mx_group_max<F, 4>(a);
    odd |= __shfl_xor(odd, 1);
    odd |= __shfl_xor(odd, 2);
    if (odd) a = 0;
    const int E = mx_exponent(a);
    *scale = odd ? MX_NAN : E + 127;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) codes |= mx_code(ldexp(x[i], -E)) << (4 * i);
    return odd ? 0u : codes;
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
// ---------------------------------------------------------------------------
constexpr int MA_THREADS = 256;
template <typename TI, typename TQ, int D, int HPT>
__global__ __launch_bounds__(MA_THREADS) void k_mx_append(const PgAppend a) {
    constexpr int LPH = D / 8, SL = MA_THREADS / LPH;
    __shared__ double cs[D / 2], sn[D / 2];
    __shared__ __attribute__((aligned(16))) double kx[SL][D];
    const int t = blockIdx.x, l = threadIdx.x % LPH, rot = a.rope.rot, slot = threadIdx.x / LPH;
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
        const float x[8] = {xa[i].x, xa[i].y, xa[i].z, xa[i].w, xb[i].x, xb[i].y, xb[i].z, xb[i].w};
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
        uint32_t codes, scale;
        if (isv) codes = mx_block(x, &scale);
        else {
            double y[8], ss = 0.;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = x[e];
                ss = fma(y[e], y[e], ss);
            }
            if (a.kn) {
                ss = mx_group_sum<LPH>(ss);
                const double r = 1. / sqrt(ss / D + (double)a.eps);
                const float4 wa = pg_ld4(a.kn + oa), wb = pg_ld4(a.kn + ob);
                const float w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = y[e] * r * w[e];
            }
            if (turn) rotate(y);
            // to eight elements side by side (the head's lanes are of one wave)
            double *row = kx[slot];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                row[oa + e] = y[e];
                row[ob + e] = y[e + 4];
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = row[8 * l + e];
            __builtin_amdgcn_wave_barrier();
            codes = mx_block(y, &scale);
        }
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
template <typename TO, int D>
__global__ __launch_bounds__(MD_THREADS) void k_mx_dequant(const PgArgs a, const int *__restrict__ pages, TO *k, TO *v) {
    constexpr int LPR = D / 8, RPW = MD_THREADS / LPR;   // rows of a workgroup's round
    const int g = threadIdx.x / 4 % LPR, r = threadIdx.x / (4 * LPR) * 4 + threadIdx.x % 4;
    const int chunks = max(1, (1 << a.shift) / RPW), n = blockIdx.x / chunks, h = blockIdx.y;
    const int page = pages ? pages[n] : n, in = blockIdx.x % chunks * RPW + r;
    if (in >= 1 << a.shift) return;
    const bool there = (unsigned)page < (unsigned)a.n_pages;
    const long long from = mx_head<D>(a, there ? page : 0, h);
    const long long to = ((long long)n * a.NKV + h) << a.shift;
    const int codes = (D / 2) << a.shift;
    const uint8_t *kp = (const uint8_t *)a.k + from, *vp = (const uint8_t *)a.v + from;
    const uint32_t kc = *reinterpret_cast<const uint32_t *>(kp + mx_k_code<D>(in, g));
    const uint32_t vc = *reinterpret_cast<const uint32_t *>(vp + mx_v_code<D>(in, g));
    const uint32_t ks = kp[codes + mx_k_scale<D>(in, g / 4)], vs = vp[codes + mx_v_scale<D>(in, g / 4)];
    mx_h8 x = mx_eight(kc, mx_scale(ks)), y = mx_eight(vc, mx_scale(vs));
    if (!there) x = y = mx_h8{};
    TO *ko = k + (to + in) * D + 8 * g, *vo = v + (to + in) * D + 8 * g;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        pg_st4(ko + e, make_float4((float)x[e], (float)x[e + 1], (float)x[e + 2], (float)x[e + 3]));
        pg_st4(vo + e, make_float4((float)y[e], (float)y[e + 1], (float)y[e + 2], (float)y[e + 3]));
    }
}

hipError_t launch_mx_dequant(const PgArgs &a, int D, const int *pages, int n, int out_type, void *k, void *v,
                             hipStream_t st) {
    const int rows = MD_THREADS / (D / 8);
    const dim3 grid((unsigned)n * std::max(1, (1 << a.shift) / rows), a.NKV);
#define TBQ_MD(TO)                                                                                                       \
    if (D == 128) hipLaunchKernelGGL((k_mx_dequant<TO, 128>), grid, dim3(MD_THREADS), 0, st, a, pages, (TO *)k, (TO *)v); \
    else hipLaunchKernelGGL((k_mx_dequant<TO, 64>), grid, dim3(MD_THREADS), 0, st, a, pages, (TO *)k, (TO *)v)
    if (out_type == TBQ_KV_F32) {
        TBQ_MD(float);
    } else if (out_type == TBQ_KV_F16) {
        TBQ_MD(pg_f16);
    } else {
        TBQ_MD(pg_bf16);
    }
#undef TBQ_MD
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Compaction, in place: row j of a sequence becomes its row keep[j] >= j, keep
// ascending.  A workgroup has one sequence, layer, kv head and K or V (no other
// touches its rows) and moves MC_ROWS rows a step: all of them have arrived in every
// wave before any is stored, and no later step loads a row that this one stores.
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
