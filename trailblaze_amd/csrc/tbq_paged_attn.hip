// tbq_paged_attn.hip -- causal attention of new tokens over the paged
// key/value cache (include/tbq_kv.h) on gfx950.
//
// The query heads that share a kv head are rows of one product: row r of a
// sequence's kv head is token r / G, head r % G of its G.  Sequences with few
// rows (single tokens) go to k_pg_attn_rows, bound by the cache's bytes; the
// others to k_pg_attn_chunk, bound by MFMA and the softmax.  Both are one pass
// over the visible positions with the softmax's running maximum and sum (in
// powers of two), and both form S^T = K Q^T, so that a lane holds scores of one
// row only and the probabilities are, without any exchange, the operand of
// O^T += V^T P^T when the products' positions are taken in the order that the
// accumulators have.
//
// F32 rows (HL): q, scaled by the power of two that puts its largest element in
// [2^13, 2^14), and the probabilities are each taken as two halves, x = hi + lo,
// which keeps ~22 bits; the keys and values are halves already.  16-bit rows: few
// take the probabilities as two of the cache's type as well, in a second product
// (0 to 3% of the time, bound by the bytes: 64 sequences of up to 8192 213.4 -> 214.1
// us); many round them once, which adds a third to the output's own rounding (errors
// against 64 bits 2.7e-4 with fp16, 2.1e-4 without): two would take 462 us instead of
// 344 for 2048 tokens after 8192, 44 instead of 35 for 9 mixed sequences.  Half
// probabilities are scaled by 2^14, so those that a half cannot hold are below 2^-38
// of the largest; bf16's by 2^-32, so that sums of values near their type's end stay
// within fp32.
//
// What a row does not see must not reach it, NaN and infinities included.
// Scores are replaced before the maximum.  In the product with V an unseen
// position's weight is 0, but 0 times a NaN is a NaN: values of positions that
// no row of the block sees are made zero in the tiles on the edges, and a row
// whose outputs are not all finite at the end is formed again in a way that
// multiplies only what the row sees.
#include <algorithm>
#include <type_traits>

#include "tbq_dma.hpp"
#include "tbq_kernels.h"
#include "tbq_paged_attn.hpp"

namespace tbq {

// One row by one wave, 64 positions at a time, from what the row sees only: lane
// i scores position i of the tile, then the wave adds p V for the seen positions
// in turn, lane l the dims l and l + 64.  *m, *l: maximum and sum; probabilities,
// sum and output are scaled by 2^shift, as the other splits of the row have them.
template <typename TA, typename TC, int D>
__device__ __forceinline__ void pg_slow_row(const PgArgs &pg, const TA *q, float cs, int s, int kvh, int pos, int back,
                                         int sinks, PgTiles tiles, int it0, int it1, float shift,
                                         float (&o)[D / 64], float *m, float *l) {
    const int lane = threadIdx.x & 63, last = min(pos, pg.max_kv - 1);
#pragma unroll
    for (int i = 0; i < D / 64; i++) o[i] = 0.f;
    *m = PG_LOW;
    *l = 0.f;
    for (int it = it0; it < it1; it++) {
        const int k0 = tiles.at(it) * 64, key = k0 + lane;
        const int page = pg_block_page(pg, s, key, last);
        const long long at = pg_row<D>(pg, max(page, 0), kvh, key);
        const bool sees = page >= 0 && ((pg_seen(k0, pos - back, last, sinks) >> lane) & 1);
        float dot = 0.f;
        for (int d = 0; d < D; d += 4) {
            const float4 x = pg_ld4(q + d), y = pg_ld4((const TC *)pg.k + at + d);
            dot = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, dot))));
        }
        dot = sees ? dot * cs : -__builtin_huge_valf();
        const float mn = fmaxf(*m, wave_max(dot)), corr = __builtin_amdgcn_exp2f(*m - mn);
        const float p = __builtin_amdgcn_exp2f(dot - mn + shift);
        *m = mn;
        *l = *l * corr + group_sum<64>(p);
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] *= corr;
        for (unsigned long long left = __builtin_amdgcn_ballot_w64(sees); left; left &= left - 1) {
            const int k = __builtin_ctzll(left);
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), k));
            const long long row = pg_row<D>(pg, __builtin_amdgcn_readlane(page, k), kvh, k0 + k);
#pragma unroll
            for (int i = 0; i < D / 64; i++) o[i] = fmaf(w, (float)((const TC *)pg.v)[row + lane + 64 * i], o[i]);
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows.  A workgroup has one sequence, one kv head, RB = 16 rows (8 as F32:
// their hi halves are the MFMA's columns 0-7, their lo halves 8-15) and a range
// of tiles of 32 positions, dealt to its four waves, which keep maxima, sums
// and outputs of their own until the end.  K and V go from memory to registers
// only: lane l holds row l % 16 of each 16 keys as the MFMA's A operand wants
// them; of V it loads 8 (4) dims, D / 16 * (l % 16) on, of the 8 positions
// whose probabilities it computed, and the 8 x 8 halves, transposed in
// registers, are the A operands of D / 16 products, product j giving the dims
// congruent to j.  A tile's loads are issued a tile ahead.
//
// Bound by HBM: 64 ragged sequences of up to 8192 positions, 32 / 8 heads of 128,
// read their 1.19 GB of keys and values once in 191 to 203 us (5.9 to 6.2 TB/s);
// one token over 131072 positions, 268 MB, 45 to 48 us; one over 4096, 16.8 MB,
// 7 us: 3.6 of the bytes, and a launch with the chain of lengths, page, rows and
// merge (the page looked up beside the lengths instead of after them: 0.2 less).
// ---------------------------------------------------------------------------
// x: kv head + NKV * row block; z: split; s: sequence.  ONCE: one row block reads the values,
// whole lines at a time, which then need not stay in the caches (64 sequences of up to 8192:
// 242 -> 228 us; keys, whose lines take two loads, are slower so).
template <typename TC, int D, bool HL, bool ONCE>
__device__ __forceinline__ void pg_rows(const PgAttn &a, int nrb, int tps, int nsplit, float *__restrict__ part, int x, int z,
                                        int s, PrLds<D> *lds) {
    typedef typename PgVec<TC>::h8 h8;
    typedef TC hv __attribute__((ext_vector_type(D / 16)));
    constexpr int RB = HL ? 8 : 16, NS = D / 32, ND = D / 16;
    constexpr float SH = PgVec<TC>::SHIFT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, h = lane >> 4;
    const int kvh = x % a.pg.NKV, r0 = x / a.pg.NKV * RB, G = a.NQ / a.pg.NKV;
    const int q0 = a.pg.q_start[s], qn = a.pg.q_start[s + 1] - q0;
    if (qn <= 0 || q0 < 0 || qn > a.pg.n_tokens - q0 || qn > PR_MAX) return;
    const int rows = qn * G;
    if (rows > a.few || r0 >= rows) return;
    const int base = a.pg.kv_len[s] - qn;   // position of the first token
    const int t0 = r0 / G, t1 = (min(r0 + RB, rows) - 1) / G;   // the block's tokens
    const int plo = base + t0, phi = base + t1, last = min(phi, a.pg.max_kv - 1);
    const int back = a.window > 0 ? a.window : 0x40000000;   // a token at p sees the positions > p - back
    const PgTiles tiles = pg_tiles<PR_TS>(plo, phi, a.window, a.sinks, a.pg.max_kv);
    const int nz = (tiles.n + tps - 1) / tps, it0 = z * tps, it1 = min(it0 + tps, tiles.n);
    if (z > 0 && it0 >= it1) return;
    const int row = r0 + (HL ? li & 7 : li), rc = min(row, rows - 1), tok = rc / G, pos = base + tok;
    // Q^T's columns
    h8 qf[NS];
    float cs = fmaxf(a.scale, PG_TINY);
    {
        const long long off = (long long)(q0 + tok) * a.qs + (long long)(kvh * G + rc % G) * D + 8 * h;
        if constexpr (HL) {
            const float *q = (const float *)a.q + off;
            float4 x[NS][2];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float4 v = x[i][j] = pg_ld4(q + 32 * i + 4 * j);
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                }
            mx = swap32_max(swap16_max(mx));
            const int sh = pg_row_shift(mx);
            const float f = ldexpf(1.f, sh);
            cs = fmaxf(cs * ldexpf(1.f, -sh), PG_TINY);
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float v[4] = {x[i][j].x * f, x[i][j].y * f, x[i][j].z * f, x[i][j].w * f};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const TC hi = (TC)v[e];
                        qf[i][4 * j + e] = li < 8 ? hi : (TC)(v[e] - (float)hi);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < NS; i++) qf[i] = *reinterpret_cast<const h8 *>((const TC *)a.q + off + 32 * i);
        }
    }
    const long long hstride = (long long)D << a.pg.shift;   // elements of a kv head in a page
    const uint32_t koff = (uint32_t)(li * D + 8 * h), voff = (uint32_t)(4 * h * D + ND * li);
    int pages = -1;   // lane i: the page of block i % 2 of the wave's tile i / 2 (of 32 tiles)
    auto tile_at = [&](int n) { return tiles.at(it0 + wave + PR_WAVES * n) * PR_TS; };
    auto page_of = [&](int n, int b) { return __builtin_amdgcn_readlane(pages, 2 * (n & 31) + b); };
    const int nt = (it1 - it0 - wave + PR_WAVES - 1) / PR_WAVES;   // this wave's tiles
    auto look_up = [&](int n) {
        const int k = n + (lane >> 1);
        pages = k < nt ? pg_block_page(a.pg, s, tile_at(k) + 16 * (lane & 1), last) : -1;
    };
    h8 kf[2][2][NS];
    hv vf[2][8];
    auto load = [&](int buf, int n) {
        if ((n & 31) == 0) look_up(n);
        const int k0 = tile_at(n);
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int in = (k0 + 16 * b) & ((1 << a.pg.shift) - 1);
            const long long off = ((long long)max(page_of(n, b), 0) * a.pg.NKV + kvh) * hstride + (long long)in * D;
            const TC *kp = (const TC *)a.pg.k + off, *vp = (const TC *)a.pg.v + off;
#pragma unroll
            for (int i = 0; i < NS; i++) kf[buf][b][i] = *reinterpret_cast<const h8 *>(kp + koff + 32 * i);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const hv *v = reinterpret_cast<const hv *>(vp + voff + i * D);
                if constexpr (ONCE) vf[buf][4 * b + i] = __builtin_nontemporal_load(v);
                else vf[buf][4 * b + i] = *v;
            }
        }
    };
    pg_f4 o[ND];
    float m, l;
    // b: whether the block has a page
    auto compute = [&](int buf, int n, bool safe) {
        const int k0 = tile_at(n);
        const bool pg0 = page_of(n, 0) >= 0, pg1 = page_of(n, 1) >= 0;
        const bool whole = pg0 && pg1 && k0 + PR_TS - 1 <= min(plo, a.pg.max_kv - 1) &&
                           (k0 > phi - back || k0 + PR_TS <= a.sinks);
        const uint32_t has = (pg0 ? 0xFFFFu : 0u) | (pg1 ? 0xFFFF0000u : 0u);
        // the lane's positions that tokens at lo .. hi see: element e is bit 16 (e / 4) + e % 4
        auto seen = [&](int lo, int hi) {
            return ((uint32_t)pg_seen(k0, lo - back, min(hi, last), a.sinks) & has) >> (4 * h);
        };
        pg_f4 sc[2] = {pg_f4{}, pg_f4{}};
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int b = 0; b < 2; b++) sc[b] = pg_mfma16(kf[buf][b][i], qf[i], sc[b]);
        if constexpr (HL) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = sc[b][r], y = dpp_f32<0x128>(x), hi = li < 8 ? x : y;   // row_ror:8
                    // (q's lo half times an infinite key may be the other infinity, or 0 times it)
                    sc[b][r] = safe && !(fabsf(hi) < __builtin_huge_valf()) ? hi : x + y;
                }
        }
        auto bit = [](int e) { return 16 * (e / 4) + e % 4; };
        if (!whole) {
            const uint32_t mine = seen(pos, pos);
#pragma unroll
            for (int e = 0; e < 8; e++) sc[e / 4][e % 4] = pg_hide(sc[e / 4][e % 4], pg_ones(mine, bit(e)));
        }
        float mx = sc[0][0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = fmaxf(mx, sc[e / 4][e % 4]);
        mx = swap32_max(swap16_max(mx)) * cs;
        if (__builtin_amdgcn_ballot_w64(mx > m)) {
            const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int j = 0; j < ND; j++) o[j] *= corr;
        }
        h8 pf, pl;   // (F32 rows' lo halves are columns of their own)
        const float mb = SH - m;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / 4][e % 4], cs, mb));
            l += p;
            const TC hi = (TC)p;
            const TC lo = (TC)(p - (float)hi);
            if constexpr (HL) pf[e] = li < 8 ? hi : lo;
            else {
                pf[e] = hi;
                pl[e] = lo;
            }
        }
        if (!whole) {   // values that no row of the block sees
            const uint32_t any = seen(plo, phi);
#pragma unroll
            for (int e = 0; e < 8; e++) vf[buf][e] = pg_keep(vf[buf][e], pg_ones(any, bit(e)));
        }
        if (whole || !safe) {
#pragma unroll
            for (int j = 0; j < ND; j++) {
                h8 v;
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = vf[buf][e][j];
                o[j] = pg_mfma16(v, pf, o[j]);
                if constexpr (!HL) o[j] = pg_mfma16(v, pl, o[j]);
            }
        } else {
            for (int t = t0; t <= t1; t++) {
                const uint32_t its = seen(base + t, base + t);
                hv w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = pg_keep(vf[buf][e], pg_ones(its, bit(e)));
#pragma unroll
                for (int j = 0; j < ND; j++) {
                    h8 v;
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = w[e][j];
                    pg_f4 u = pg_mfma16(v, pf, o[j]);
                    if constexpr (!HL) u = pg_mfma16(v, pl, u);
                    if (tok == t) o[j] = u;
                }
            }
        }
    };
    for (int safe = 0;; safe = 1) {
        m = PG_LOW;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < ND; j++) o[j] = pg_f4{};
        if (nt > 0) load(0, 0);
        for (int n = 0; n < nt; n += 2) {
            if (n + 1 < nt) load(1, n + 1);
            compute(0, n, safe);
            if (n + 1 >= nt) break;
            if (n + 2 < nt && ((n + 2) & 31) != 0) load(0, n + 2);
            compute(1, n + 1, safe);
            if (n + 2 < nt && ((n + 2) & 31) == 0) load(0, n + 2);   // the pages of 32 tiles are used up first
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < ND; j++) sum += (o[j][0] - o[j][0]) + (o[j][1] - o[j][1]) + (o[j][2] - o[j][2]) + (o[j][3] - o[j][3]);
        if (safe || !__builtin_amdgcn_ballot_w64(row < rows && sum != 0.f)) break;   // no NaN or infinity
    }
    pg_rows_out<TC, D, HL>(a, o, m, l, r0, rows, G, kvh, q0, s, z, nz, nrb, nsplit, part, lds);
}

template <typename TC, int D, bool HL, bool ONCE>
__global__ __launch_bounds__(64 * PR_WAVES) __attribute__((amdgpu_waves_per_eu(2, 2))) void k_pg_attn_rows(
    const PgAttn a, int nrb, int tps, int nsplit, float *__restrict__ part) {
    __shared__ __attribute__((aligned(16))) PrLds<D> lds;
    pg_rows<TC, D, HL, ONCE>(a, nrb, tps, nsplit, part, blockIdx.x, blockIdx.y, blockIdx.z, &lds);
}

// Joins the nz splits of a row: out = sum_z 2^(m_z - M) o_z / sum_z 2^(m_z - M) l_z.
// One workgroup a row.  GROUPS groups of D / 4 lanes each add every GROUPS-th
// split, then the groups are added in order: a row's records (hundreds for one
// token over a long context) are read by as many lanes as there are, 8 in flight
// each.
constexpr int PJ_THREADS = 256, PJ_MAX = 1024;   // most splits (pg_plan)
template <typename TO, int D>
__device__ __forceinline__ void pg_join_row(const float *__restrict__ rec, int nz, TO *out) {
    constexpr int GROUPS = PJ_THREADS / (D / 4), REC = pg_rec(D);
    __shared__ float fs[PJ_MAX];
    __shared__ float red[2][PJ_THREADS / 64];
    __shared__ __attribute__((aligned(16))) float os[GROUPS][D];
    const int tid = threadIdx.x;
    float mz[PJ_MAX / PJ_THREADS], lz[PJ_MAX / PJ_THREADS], M = PG_LOW;
#pragma unroll
    for (int i = 0; i < PJ_MAX / PJ_THREADS; i++) {
        const int z = tid + PJ_THREADS * i;
        const float2 ml = *reinterpret_cast<const float2 *>(rec + (long long)min(z, nz - 1) * REC + D);
        mz[i] = z < nz ? ml.x : PG_LOW;
        lz[i] = z < nz ? ml.y : 0.f;
        M = fmaxf(M, mz[i]);
    }
    M = wave_max(M);
    if ((tid & 63) == 0) red[0][tid >> 6] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PJ_THREADS / 64; i++) M = fmaxf(M, red[0][i]);
    float den = 0.f;
#pragma unroll
    for (int i = 0; i < PJ_MAX / PJ_THREADS; i++) {
        const float f = __builtin_amdgcn_exp2f(mz[i] - M);
        fs[tid + PJ_THREADS * i] = f;
        den = fmaf(f, lz[i], den);
    }
    den = group_sum<64>(den);
    if ((tid & 63) == 0) red[1][tid >> 6] = den;
    __syncthreads();
    const int g = tid / (D / 4), d = tid % (D / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int z = g; z < nz; z += 8 * GROUPS) {
        float4 y[8];
#pragma unroll
        for (int i = 0; i < 8; i++)   // past the last: the last again, weighed 0
            y[i] = *reinterpret_cast<const float4 *>(rec + (long long)min(z + i * GROUPS, nz - 1) * REC + d);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (z + i * GROUPS >= nz) continue;
            const float f = fs[z + i * GROUPS];
            x = make_float4(fmaf(f, y[i].x, x.x), fmaf(f, y[i].y, x.y), fmaf(f, y[i].z, x.z), fmaf(f, y[i].w, x.w));
        }
    }
    *reinterpret_cast<float4 *>(&os[g][d]) = x;
    __syncthreads();
    if (tid >= D) return;
    den = 0.f;
#pragma unroll
    for (int i = 0; i < PJ_THREADS / 64; i++) den += red[1][i];
    float num = os[0][tid];
#pragma unroll
    for (int i = 1; i < GROUPS; i++) num += os[i][tid];
    out[tid] = (TO)(den == 0.f ? 0.f : num / den);
}

// Joins nz records by D / 4 lanes, dims d .. d + 3 each, eight records at once.
template <typename TO, int D>
__device__ __forceinline__ void pg_join_few(const float *__restrict__ rec, int nz, int d, TO *out) {
    constexpr int REC = pg_rec(D);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f, M = PG_LOW;
    for (int z0 = 0; z0 < nz; z0 += 8) {
        float2 ml[8];
        float4 y[8];
        float mn = M;
#pragma unroll
        for (int z = 0; z < 8; z++) {   // past the last: the last again, not added
            ml[z] = *reinterpret_cast<const float2 *>(rec + min(z0 + z, nz - 1) * REC + D);
            y[z] = *reinterpret_cast<const float4 *>(rec + min(z0 + z, nz - 1) * REC + d);
            mn = fmaxf(mn, ml[z].x);
        }
        const float c = __builtin_amdgcn_exp2f(M - mn);
        M = mn;
        x = make_float4(x.x * c, x.y * c, x.z * c, x.w * c);
        den *= c;
#pragma unroll
        for (int z = 0; z < 8; z++) {
            if (z0 + z >= nz) continue;
            const float f = __builtin_amdgcn_exp2f(ml[z].x - M);
            x = make_float4(fmaf(f, y[z].x, x.x), fmaf(f, y[z].y, x.y), fmaf(f, y[z].z, x.z), fmaf(f, y[z].w, x.w));
            den = fmaf(f, ml[z].y, den);
        }
    }
    const float inv = den == 0.f ? 0.f : 1.0f / den;
    pg_st4(out + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
}

// A row of a sequence of few rows.  x: kv head + NKV * row; s: sequence; d: of FEW lanes'
// dims the first.
template <typename TO, int D, bool HL, bool FEW>
__device__ __forceinline__ void pg_join_rows(const PgAttn &a, int nrb, int tps, int nsplit, const float *__restrict__ part,
                                             int x, int s, int d) {
    constexpr int RB = HL ? 8 : 16;
    const int kvh = x % a.pg.NKV, r = x / a.pg.NKV, G = a.NQ / a.pg.NKV;
    const int q0 = a.pg.q_start[s], qn = a.pg.q_start[s + 1] - q0;
    if (qn <= 0 || q0 < 0 || qn > a.pg.n_tokens - q0 || qn > PR_MOST) return;
    const int rows = qn * G;
    if (rows > a.few || r >= rows) return;
    const int base = a.pg.kv_len[s] - qn, r0 = r / RB * RB;
    const int nz = (pg_tiles<PR_TS>(base + r0 / G, base + (min(r0 + RB, rows) - 1) / G, a.window, a.sinks, a.pg.max_kv).n +
                    tps - 1) / tps;
    const float *rec = part + (((long long)s * a.pg.NKV + kvh) * nrb * RB + r) * nsplit * pg_rec(D);
    TO *out = (TO *)a.out + ((long long)(q0 + r / G) * a.NQ + kvh * G + r % G) * D;
    if (nz <= 1) return;
    if constexpr (FEW) pg_join_few<TO, D>(rec, nz, d, out);
    else pg_join_row<TO, D>(rec, nz, out);
}

// ---------------------------------------------------------------------------
// Many rows.  A workgroup has one kv head and 128 of a sequence's rows, 32 a
// wave, and goes through K and V 64 positions at a time in LDS, copied there
// directly a tile ahead, each 16 positions from their page.  A wave forms S^T
// (64 positions x its 32 rows) with v_mfma_f32_32x32x16: lane l holds of row l %
// 32 the positions 32 b + 8 (r / 4) + 4 (l / 32) + r % 4.  V stays as the cache
// has it, [position][dim]: ds_read_b64_tr_b16 gives 16 lanes 4 positions of 16
// dims transposed, which are the A operand's positions in the order of the
// probabilities.  The 16-byte segments of LDS rows are XOR-swizzled by the
// copies' source addresses: K's by row, V's so that the four positions of a
// transposing read lie in different banks.
//
// Blocks are numbered over the batch (a sequence's last one first, its rows see
// most); several workgroups share a block's tiles where there are few
// blocks.
//
// Bound by power where it fills the chip: 2048 tokens after 8192 positions, 32 / 8
// heads of 128, fp16, 341 to 371 us (0.83 to 0.91 PFLOP/s), MFMAs and VALU each half of
// a SIMD's cycles at 1.65 GHz.  With a quarter more cycles a tile (added by counting
// them) the clock rose to 2.0 GHz and a tile took as long; so fewer waits gain
// nothing there: keys read ahead of their products -1 to 3%, copies between the products
// -10%, the next tile's scores under this one's softmax -9%, three tiles in LDS 0 to
// -4%.  Half the LDS reads would gain 15% (two row tiles a wave, for which 256
// registers are too few), no copies at all 14%; eight waves on one tile gain 4% for 4096
// tokens and lose 4 to 40% for fewer.  Smaller batches are bound by a tile's chain of
// products, maximum and powers, 0.95 us with heads of 64.
// ---------------------------------------------------------------------------
template <int D>
struct PcLds {
    unsigned char k[2][PC_TS * D * 2], v[2][PC_TS * D * 2];
};

// x: kv head + NKV * block; z: split.
template <typename TC, int D, bool HL>
__device__ __forceinline__ void pg_chunk(const PgAttn &a, int nsplit, float *__restrict__ part, int x, int z,
                                         PcLds<D> *st) {
    typedef typename PgVec<TC>::h8 h8;
    constexpr int NT = D / 32, NS = D / 16, SEG = D / 8, NP = HL ? 2 : 1, RPC = 64 / SEG;   // rows per copy
    constexpr int CPW = PC_TS / RPC / PC_WAVES;                                                 // copies per wave
    // (m is the exact maximum: the position that holds it then has a power of two for its weight and no
    // rounding.  One that may lag 2^8 behind spares most rescalings of o, 350 -> 340 us for 2048 tokens
    // after 8192, but the errors of 16-bit rows grow by 8 to 15%)
    constexpr float SH = PgVec<TC>::SHIFT;
    const int kvh = x % a.pg.NKV, G = a.NQ / a.pg.NKV;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 31, h = lane >> 5;
    const PcBlock blk = pg_chunk_block(a.pg, a.few, G, x / a.pg.NKV);
    const int s = blk.s, q0 = blk.q0, qn = blk.qn;
    if (s < 0 || q0 < 0 || qn > a.pg.n_tokens - q0) return;
    const int rows = qn * G, base = blk.len - qn;
    const int r0 = blk.yb * PC_ROWS, r1 = min(r0 + PC_ROWS, rows) - 1;
    const int plo = base + r0 / G, phi = base + r1 / G, last = min(phi, a.pg.max_kv - 1);
    const int back = a.window > 0 ? a.window : 0x40000000;   // a token at p sees the positions > p - back
    const PgTiles tiles = pg_tiles<PC_TS>(plo, phi, a.window, a.sinks, a.pg.max_kv);
    const int tps = max((tiles.n + nsplit - 1) / nsplit, 1), it0 = z * tps, it1 = min(it0 + tps, tiles.n);
    const int nz = (tiles.n + tps - 1) / tps;
    if (z > 0 && it0 >= it1) return;
    const int row = r0 + wave * 32 + li, rc = min(row, rows - 1), tok = rc / G, pos = base + tok;
    // the wave's tokens
    const int w0 = min(r0 + wave * 32, rows - 1) / G, w1 = min(r0 + wave * 32 + 31, rows - 1) / G;
    // Q^T's columns: dim step i, lane half h has dims 16 i + 8 h .. + 8
    h8 qf[NP][NS];
    float cs = fmaxf(a.scale, PG_TINY);
    {
        const long long off = (long long)(q0 + tok) * a.qs + (long long)(kvh * G + rc % G) * D + 8 * h;
        if constexpr (HL) {
            const float *q = (const float *)a.q + off;
            float4 qx[NS][2];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float4 v = qx[i][j] = pg_ld4(q + 16 * i + 4 * j);
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                }
            const int sh = pg_row_shift(swap32_max(mx));
            const float f = ldexpf(1.f, sh);
            cs = fmaxf(cs * ldexpf(1.f, -sh), PG_TINY);
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float v[4] = {qx[i][j].x * f, qx[i][j].y * f, qx[i][j].z * f, qx[i][j].w * f};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        qf[0][i][4 * j + e] = (TC)v[e];
                        qf[NP - 1][i][4 * j + e] = (TC)(v[e] - (float)qf[0][i][4 * j + e]);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < NS; i++) qf[0][i] = *reinterpret_cast<const h8 *>((const TC *)a.q + off + 16 * i);
        }
    }
    // copies: copy c = wave + 4 i takes rows RPC c .. + RPC of the tile, which lie in one
    // 16-position block of it
    auto kswz = [](int r) { return SEG == 16 ? r & 15 : (r & 7) ^ ((r >> 3) & 1); };
    auto vswz = [](int r) { return SEG == 16 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; };
    uint32_t ko[CPW], vo[CPW];
#pragma unroll
    for (int i = 0; i < CPW; i++) {
        const int r = (wave + PC_WAVES * i) * RPC + lane / SEG;
        ko[i] = (uint32_t)((r & 15) * D * 2 + 16 * ((lane % SEG) ^ kswz(r)));
        vo[i] = (uint32_t)((r & 15) * D * 2 + 16 * ((lane % SEG) ^ vswz(r)));
    }
    const uint32_t lk = lds_addr(st->k[0]), lv = lds_addr(st->v[0]);
    uint32_t off_lo = 0, off_hi = 0;   // lane i: bytes before block i % 4 of tile i / 4 (of 16 tiles)
    uint64_t nopage = 0;               // bit i: lane i's has no page
    const int pmask = (1 << a.pg.shift) - 1;
    const long long hbytes = (long long)(2 * D) << a.pg.shift;   // bytes of a kv head in a page
    auto look_up = [&](int n) {
        const int it = it0 + n + (lane >> 2), pos = tiles.at(it) * PC_TS + 16 * (lane & 3);
        const int page = it < it1 ? pg_block_page(a.pg, s, pos, last) : -1;
        nopage = __builtin_amdgcn_ballot_w64(page < 0);
        const long long off = ((long long)max(page, 0) * a.pg.NKV + kvh) * hbytes + (long long)(pos & pmask) * (2 * D);
        off_lo = (uint32_t)off;
        off_hi = (uint32_t)(off >> 32);
    };
    auto copy = [&](int buf, int n) {
#pragma unroll
        for (int i = 0; i < CPW; i++) {
            const int c = wave + PC_WAVES * i, at = 4 * (n & 15) + c * RPC / 16;
            const long long off = (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)off_hi, at) << 32 |
                                              (uint32_t)__builtin_amdgcn_readlane((int)off_lo, at));
            const uint32_t to = buf * (PC_TS * D * 2) + c * 1024;
            dma16(lk + to, ko[i], dma_rsrc((const uint8_t *)a.pg.k + off, 32 * D), 0);
            dma16(lv + to, vo[i], dma_rsrc((const uint8_t *)a.pg.v + off, 32 * D), 0);
        }
    };
    // V's transposing reads: lane l of 16 addresses position kk = l / 4 of 4, dims 4 (l % 4) .. + 4
    // of 16; of dim block j the address is voff[j] + the step's rows
    uint32_t voff[NT];
    {
        const int kk = (lane & 15) >> 2;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int seg = 4 * j + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            voff[j] = (uint32_t)((4 * h + kk) * D * 2 + 16 * (seg ^ vswz(kk)) + 8 * (lane & 1));
        }
    }
    pg_f16x o[NT];
    float m, l;
    const int ksw = kswz(li);
    {
        m = PG_LOW;
        l = 0.f;
#pragma unroll
        for (int j = 0; j < NT; j++) o[j] = pg_f16x{};
        const int nt = it1 - it0;
        if (nt > 0) {
            look_up(0);
            copy(0, 0);
        }
        dma_wait_barrier();
        for (int n = 0, buf = 0; n < nt; n++, buf ^= 1) {
            const int k0 = tiles.at(it0 + n) * PC_TS;
            const int none = (int)(nopage >> (4 * (n & 15))) & 15;   // its blocks without a page
            if (n + 1 < nt) {
                if (((n + 1) & 15) == 0) look_up(n + 1);
                copy(buf ^ 1, n + 1);
            }
            // every row of the block sees all of the tile
            const bool inner = none == 0 && k0 + PC_TS - 1 <= min(plo, last) && (k0 > phi - back || k0 + PC_TS <= a.sinks);
            uint64_t has = ~0ull;   // positions of the tile that have a page
            if (!inner) {
#pragma unroll
                for (int b = 0; b < 4; b++) has &= (none >> b) & 1 ? ~(0xFFFFull << (16 * b)) : ~0ull;
                // values that no row of the block sees are made zero
                const uint64_t dead = ~(pg_seen(k0, plo - back, last, a.sinks) & has);
                if (dead) {   // uniform
#pragma unroll
                    for (int i = 0; i < PC_TS * SEG / (64 * PC_WAVES); i++) {
                        const int f = threadIdx.x + 64 * PC_WAVES * i;
                        if ((dead >> (f / SEG)) & 1) *reinterpret_cast<pg_u4 *>(st->v[buf] + 16 * f) = pg_u4{};
                    }
                    __syncthreads();
                }
            }
            const int wlo = base + w0, whi = base + w1;
            if (inner || (k0 <= whi && (k0 + PC_TS > wlo - back || k0 < a.sinks))) {   // the wave's rows see some of it
                const bool whole = inner || (has == ~0ull && k0 + PC_TS - 1 <= min(wlo, last) &&
                                             (k0 > whi - back || k0 + PC_TS <= a.sinks));
                // the positions that tokens at lo .. hi see, from the lane's 4 h on
                auto seen = [&](int lo, int hi) {
                    return (pg_seen(k0, lo - back, min(hi, last), a.sinks) & has) >> (4 * h);
                };
                const unsigned char *Kb = st->k[buf] + li * (D * 2);
                pg_f16x sc[2] = {pg_f16x{}, pg_f16x{}};
#pragma unroll
                for (int i = 0; i < NS; i++)
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        const h8 x = *reinterpret_cast<const h8 *>(Kb + b * (32 * D * 2) + 16 * ((2 * i + h) ^ ksw));
#pragma unroll
                        for (int p = 0; p < NP; p++) sc[b] = pg_mfma32(x, qf[p][i], sc[b]);
                    }
                if (!whole) {
                    const uint64_t mine = seen(pos, pos);
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        sc[e / 16][e % 16] = pg_hide(sc[e / 16][e % 16], pg_ones((uint32_t)(mine >> (e / 16 * 32)),
                                                                                 8 * (e % 16 / 4) + e % 4));
                }
                float mx = sc[0][0];
#pragma unroll
                for (int e = 1; e < 32; e++) mx = fmaxf(mx, sc[e / 16][e % 16]);
                mx = swap32_max(mx) * cs;
                if (__builtin_amdgcn_ballot_w64(mx > m)) {
                    const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - mn);
                    m = mn;
                    l *= corr;
#pragma unroll
                    for (int j = 0; j < NT; j++) o[j] *= corr;
                }
                h8 pf[NP][4];
                const float mb = SH - m;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16], cs, mb));
                    sum += p;
                    pf[0][e / 8][e % 8] = (TC)p;
                    if constexpr (HL) pf[NP - 1][e / 8][e % 8] = (TC)(p - (float)pf[0][e / 8][e % 8]);
                }
                l += sum;
                const uint32_t vb = lv + buf * (PC_TS * D * 2);
                auto vfrag = [&](int u, int j) {
                    const pg_s4 x = pg_read_tr(vb + voff[j] + 16 * u * (D * 2)), y = pg_read_tr(vb + voff[j] + (16 * u + 8) * (D * 2));
                    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                };
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const h8 x = __builtin_bit_cast(h8, vfrag(u, j));
#pragma unroll
                        for (int p = 0; p < NP; p++) o[j] = pg_mfma32(x, pf[p][u], o[j]);
                    }
            }
            dma_wait_barrier();
        }
    }
    l = swap32_sum(l);
    // rows with an output that is not finite are formed again, one at a time
    float odd = 0.f;   // NaN where an output is NaN or infinite
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) odd += o[j][r] - o[j][r];
    odd += __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * (lane ^ 32), __builtin_bit_cast(int, odd)));
    const bool again = row < rows && !(odd == 0.f);
    for (unsigned long long left = __builtin_amdgcn_ballot_w64(again && h == 0); left; left &= left - 1) {
        typedef typename std::conditional<HL, float, TC>::type TA;
        const int c = __builtin_ctzll(left), r = r0 + wave * 32 + c, t = r / G;
        float so[D / 64], sm, sl;
        pg_slow_row<TA, TC, D>(a.pg, (const TA *)a.q + (long long)(q0 + t) * a.qs + (long long)(kvh * G + r % G) * D, a.scale,
                               s, kvh, base + t, back, a.sinks, tiles, it0, it1, SH, so, &sm, &sl);
        const long long to = (long long)(q0 + t) * a.NQ + kvh * G + r % G;
        float *rec = part + (to * nsplit + z) * pg_rec(D);
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            const float x = nz > 1 ? so[i] : sl == 0.f ? 0.f : so[i] / sl;
            if (nz > 1) rec[lane + 64 * i] = x;
            else if (HL || a.f32_out) ((float *)a.out)[to * D + lane + 64 * i] = x;
            else ((TC *)a.out)[to * D + lane + 64 * i] = (TC)x;
        }
        if (nz > 1 && lane == 0) {
            rec[D] = sm;
            rec[D + 1] = sl;
        }
    }
    if (again) return;
    if (row >= rows) return;
    const long long at = ((long long)(q0 + tok) * a.NQ + kvh * G + row % G);
    if (nz <= 1) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;   // a row that sees nothing is 0
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4 x = make_float4(o[j][4 * r] * inv, o[j][4 * r + 1] * inv, o[j][4 * r + 2] * inv, o[j][4 * r + 3] * inv);
                const long long d = at * D + 32 * j + 8 * r + 4 * h;
                if (HL || a.f32_out) pg_st4((float *)a.out + d, x);
                else pg_st4((TC *)a.out + d, x);
            }
        return;
    }
    float *rec = part + (at * nsplit + z) * pg_rec(D);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *reinterpret_cast<float4 *>(rec + 32 * j + 8 * r + 4 * h) =
                make_float4(o[j][4 * r], o[j][4 * r + 1], o[j][4 * r + 2], o[j][4 * r + 3]);
    if (h == 0) {
        rec[D] = m;
        rec[D + 1] = l;
    }
}

// Sequences of many rows and, in the last workgroups, of few.  One launch: the few
// rows' reads run beside the last of the many rows' products (9 mixed sequences
// 39.8 us, 45.5 as two launches, 41.7 with the few rows first; 35 to 36 since).
template <typename TC, int D, bool HL>
__global__ __launch_bounds__(64 * PC_WAVES)
    __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2))) void k_pg_attn_chunk(
        const PgAttn a, int nrb, int tps, int row_splits, float *__restrict__ row_part, int nsplit,
        float *__restrict__ part) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char pc_lds[];
    const int nrows = a.pg.NKV * nrb, chunks = (int)gridDim.x - nrows * row_splits * a.pg.n_seqs, x = blockIdx.x;
    if (x >= chunks) {
        const int y = (x - chunks) / nrows;
        pg_rows<TC, D, HL, false>(a, nrb, tps, row_splits, row_part, (x - chunks) % nrows, y % row_splits, y / row_splits,
                                  reinterpret_cast<PrLds<D> *>(pc_lds));
    } else {
        const int y = x / a.pg.NKV;
        pg_chunk<TC, D, HL>(a, nsplit, part, x % a.pg.NKV + a.pg.NKV * (y / nsplit), y % nsplit,
                            reinterpret_cast<PcLds<D> *>(pc_lds));
    }
}

// The splits of head hd's row of token t in a sequence of many rows (0 or 1: no records).
__device__ __forceinline__ int pg_chunk_splits(const PgAttn &a, int q0, int rows, int base, int t, int hd, int nsplit) {
    const int G = a.NQ / a.pg.NKV, r0 = ((t - q0) * G + hd % G) / PC_ROWS * PC_ROWS;
    const int n = pg_tiles<PC_TS>(base + r0 / G, base + (min(r0 + PC_ROWS, rows) - 1) / G, a.window, a.sinks, a.pg.max_kv).n;
    const int tps = max((n + nsplit - 1) / nsplit, 1);
    return (n + tps - 1) / tps;
}

// Joins the rows of token t (heads hd0 .. hd1 - 1) in a sequence of many rows: up to
// PC_FEW splits D / 4 lanes have a head and load eight of its records at once, else
// a workgroup has a head (384 tokens of 16 heads of 64 in 10 splits 24.8 and 37.4 us;
// 64 tokens of 32 heads of 128 in 64 splits 74 and 66).
constexpr int PC_FEW = 32, PC_SPLITS = 256, PC_LEAST = 4, PC_LONG = 16;   // ..., most splits, tiles of one at least
constexpr long long PC_SHORT = 8;
__host__ __device__ constexpr int pj_heads(int D) { return PJ_THREADS / (D / 4); }   // of a workgroup
template <typename TO, int D>
__device__ __forceinline__ void pg_join_chunk(const PgAttn &a, int nsplit, const float *__restrict__ part, int t, int hd0,
                                              int hd1) {
    constexpr int REC = pg_rec(D);
    const int s = pg_seq_of(a.pg.q_start, a.pg.n_seqs, t);
    if (s >= a.pg.n_seqs || t < a.pg.q_start[s]) return;
    const int q0 = a.pg.q_start[s], qn = a.pg.q_start[s + 1] - q0;
    if (q0 < 0 || qn > a.pg.n_tokens - q0 || (long long)qn * (a.NQ / a.pg.NKV) <= a.few) return;
    const int rows = qn * (a.NQ / a.pg.NKV), base = a.pg.kv_len[s] - qn;
    if (nsplit > PC_FEW) {
        const long long at = (long long)t * a.NQ + hd0;
        const int nz = pg_chunk_splits(a, q0, rows, base, t, hd0, nsplit);
        if (nz > 1) pg_join_row<TO, D>(part + at * nsplit * REC, nz, (TO *)a.out + at * D);
        return;
    }
    const int hd = hd0 + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
    if (hd >= hd1) return;
    const int nz = pg_chunk_splits(a, q0, rows, base, t, hd, nsplit);
    if (nz <= 1) return;
    const long long at = (long long)t * a.NQ + hd;
    pg_join_few<TO, D>(part + at * nsplit * REC, nz, d, (TO *)a.out + at * D);
}

// grid: row_wgs = NKV * (most rows of a few-row sequence) * n_seqs workgroups for
// few rows (0: they were not split; FEW: one for pj_heads of them), then one for
// pj_heads of a token's heads, or for one of them (none if the many rows were not split).
template <typename TO, int D, bool HL, bool FEW>
__global__ __launch_bounds__(PJ_THREADS) void k_pg_join(const PgAttn a, int nrb, int tps, int row_splits,
                                                        const float *__restrict__ row_part, int row_wgs, int most,
                                                        int nsplit, const float *__restrict__ part) {
    const int x = blockIdx.x, n = a.pg.NKV * most, y = x - row_wgs;
    if (FEW && x < row_wgs) {
        const int i = x * pj_heads(D) + threadIdx.x / (D / 4), s = i / n;
        if (s < a.pg.n_seqs)
            pg_join_rows<TO, D, HL, true>(a, nrb, tps, row_splits, row_part, i % n, s, threadIdx.x % (D / 4) * 4);
    } else if (x < row_wgs) pg_join_rows<TO, D, HL, false>(a, nrb, tps, row_splits, row_part, x % n, x / n, 0);
    else if (nsplit > PC_FEW) pg_join_chunk<TO, D>(a, nsplit, part, y / a.NQ, y % a.NQ, y % a.NQ + 1);
    else {
        const int hpw = pj_heads(D), g = (a.NQ + hpw - 1) / hpw;
        pg_join_chunk<TO, D>(a, nsplit, part, y / g, y % g * hpw, min(y % g * hpw + hpw, a.NQ));
    }
}

// ---------------------------------------------------------------------------
// Host side: the splits, by what the host knows (max_q, max_kv, n_tokens).
// ---------------------------------------------------------------------------
static int pg_few(const PgArgs &a, int D, int G, bool f32, int c_type) {
    const double positions = (double)a.n_seqs * a.max_kv * a.NKV;   // of kv heads
    const bool mx = c_type == TBQ_KV_MXFP4;
    if (mx) {
        const long long rows = (long long)a.max_q * G;
        if (rows <= PR_MAX) return PR_MOST;
        if (rows <= PR_MOST && (!f32 || (positions <= PR_SHORT32 && (long long)a.n_seqs * a.NKV < 256))) return PR_MOST;
        if (rows > PR_MOST && positions <= (f32 ? PR_SHORT32 : PR_SHORT)) return PR_MOST;
    }
    if (positions * 2 * pg_row_bytes(c_type, D) > 256 << 20) return PR_MAX / 2;
    return mx && !f32 ? PR_MAX + PR_MAX / 2 : PR_MAX;
}

PgPlan pg_plan(const PgArgs &a, int D, int NQ, int window, int sinks, bool f32, int c_type) {
    PgPlan p{};
    const int G = NQ / a.NKV, RB = f32 ? 8 : 16, cu = 256;
    p.few = pg_few(a, D, G, f32, c_type);
    p.most = (int)std::min((long long)a.max_q * G, (long long)p.few);
    p.nrb = (p.most + RB - 1) / RB;
    // positions that one block can see
    long long seen = a.max_kv;
    if (window > 0) seen = std::min(seen, (long long)window + sinks + 2 * PC_TS + std::min(a.max_q, PC_ROWS));
    p.chunks = (long long)a.max_q * G > p.few;
    p.chunk_splits = 1;
    if (p.chunks) {
        // a last block that is not full for each sequence that has many rows; half of them
        // counted as there
        const long long full = ((long long)a.n_tokens * G + PC_ROWS - 1) / PC_ROWS;
        p.blocks = (int)(full + std::min((long long)a.n_seqs, (long long)a.n_tokens * G / (p.few + 1)));
        const long long w = a.NKV * ((full + p.blocks) / 2);
        // two workgroups a CU, each with PC_LEAST tiles: 16 tokens of 32 / 8 heads after 100000 positions
        // 351 us in 8 splits, 97 in 64; 40 tokens after 2500 27.2 us with 8 tiles at least, 21.7 with 4,
        // 4 prompts of 100 after 1000 32.8 and 33.4
        const long long t = (seen + PC_TS - 1) / PC_TS;
        long long n = std::min(2 * cu / w, t / PC_LEAST);
        // or half so many tiles, up to PC_SHORT splits that all run at once: 72 tokens after 393 14.9 -> 12.9,
        // 835 tokens 21.4 -> 17.9, 15 sequences of 65 after 633 17.2 -> 18.5 (more splits, or of fewer than 8
        // tiles, are slower)
        if (t >= 2 * PC_LEAST) n = std::max(n, std::min(2 * cu / ((long long)a.NKV * p.blocks), std::min(2 * t / PC_LEAST, PC_SHORT)));
        // Heads of 64 leave room for three, which pays where a split keeps PC_LONG tiles: 16 ragged prompts
        // of up to 300 after 3000 positions 66.8 us in one split, 49.5 in two; but 600 after 3000 with a
        // window of 1024 34.3 in one, 35.7 in two.
        if (D == 64) n = std::max(n, std::min(3 * cu / w, t / PC_LONG));
        p.chunk_splits = (int)std::max(1ll, std::min((long long)PC_SPLITS, n));
    }
    const long long tiles = (seen + PR_TS - 1) / PR_TS + 1;
    // Two workgroups a CU run at once, so at least as many splits as fill them.  Longer ranges than
    // PR_LONG make the last workgroups of a ragged batch late (64 sequences of up to 8192 in ranges of
    // 512 / 2048 / 4096 / 8192 positions: 212 / 210 / 218 / 295 us), shorter ones add to the join
    // (one token over 131072: 58 us with 128 ranges, 66 with 256).
    const long long wgs = (long long)a.NKV * p.nrb * a.n_seqs, want = (2 * cu + wgs - 1) / wgs;
    // (a batch of thousands of workgroups evens out by itself, so its ranges, and records, stay few)
    const long long longest = PR_LONG * std::max(1ll, wgs / PR_MANY);
    long long tps = (tiles + want - 1) / want;
    // Beside many rows, ranges that take about as long as a split of theirs (a wave of few rows takes
    // half as long a position) fill the chip no worse, and rows that are not split need no join: 9
    // mixed sequences with a window of 1024 41.3 -> 37.1 us.
    if (p.chunks) tps = std::max(tps, (seen + PC_TS - 1) / PC_TS * 4 / p.chunk_splits);
    tps = std::max((long long)PR_MIN, std::min(longest, (tps + 3) / 4 * 4));
    // Over 4-bit pages a wave's tile takes 0.7 us (heads of 64: 0.55), so a short range in one split is done before a join (and
    // its launch) would be: single tokens in one split / in several, in a graph, 32 / 8 heads of 128, fp16: 1 sequence after 350
    // positions 6.8 / 8.5 us, after 750 8.8 / 8.5, after 1000 10.1 / 8.5; 8 after 500 8.1 / 9.8, after 1000 10.7 / 11.1, after
    // 1500 13.3 / 11.3; 32 after 500 8.1 / 12.7, after 2000 16.9 / 18.9.  fp32: 1 after 500 8.2 / 9.3, after 750 9.8 / 9.3; 8 after
    // 750 10.0 / 11.2, after 1500 14.0 / 12.1.  16 / 8 heads of 64, fp16: 1 after 500 6.5 / 8.1, after 1000 8.7 / 8.2; 8 after 750
    // 8.0 / 9.3, after 1500 11.2 / 10.3.
    if (c_type == TBQ_KV_MXFP4 && !p.chunks && tiles <= std::min((long long)PR_LONG, 22 + wgs / 6)) tps = (tiles + 3) / 4 * 4;
    if ((tiles + tps - 1) / tps > PJ_MAX) tps = (tiles + PJ_MAX - 1) / PJ_MAX;
    p.row_tps = (int)tps;
    p.row_splits = (int)((tiles + tps - 1) / tps);
    // room for the most splits that any window can lead to
    const long long all = ((long long)a.max_kv + PR_TS - 1) / PR_TS + 1;
    const long long room = std::min((long long)PJ_MAX, std::max(std::min(want, (all + PR_MIN - 1) / PR_MIN),
                                                                (all + longest - 1) / longest));
    if (room > 1) p.rows_bytes = (size_t)a.n_seqs * a.NKV * p.nrb * RB * room * pg_rec(D) * 4;
    p.bytes = p.rows_bytes;
    if (p.chunk_splits > 1) p.bytes += (size_t)a.n_tokens * NQ * p.chunk_splits * pg_rec(D) * 4;
    return p;
}

// What a call with any window needs: the rows' room does not depend on it, and
// the chunks' splits only fall with it.
size_t pg_attn_workspace_bytes(const PgArgs &a, int D, int NQ, bool f32, int c_type) {
    if (a.n_seqs == 0 || a.n_tokens == 0) return 0;
    return pg_plan(a, D, NQ, 0, 0, f32, c_type).bytes;
}

// Rows: a batch of w workgroups a split has at most 512 / w + 1 splits to fill the
// chip, or one for each `longest` tiles, where w / longest <= 2 PR_MANY / PR_LONG;
// chunks: more than one split only while all of them fill three workgroups a CU.
size_t pg_attn_workspace_upto(int n_seqs, int n_tokens, int max_kv, int NKV, int D, int NQ, bool f32,
                              int c_type) {
    const long long RB = f32 ? 8 : 16, w = (long long)NKV * ((c_type == TBQ_KV_MXFP4 ? PR_MOST : PR_MAX) / RB) * n_seqs;
    const long long all = ((long long)max_kv + PR_TS - 1) / PR_TS + 1;
    const long long rows = std::max(512 + w, std::max(std::min(w, 2ll * PR_MANY) * ((all + PR_LONG - 1) / PR_LONG),
                                                      2ll * PR_MANY * all / PR_LONG + w));
    const long long chunk = std::min((long long)n_tokens * NQ * PC_SPLITS, 768ll * PC_ROWS);
    return (size_t)(rows * RB + chunk) * pg_rec(D) * 4;
}

// Adds the split ranges of a launch, where there are any.
template <typename TO, int D, bool HL, bool FEW>
static hipError_t pg_join(const PgAttn &a, const PgPlan &p, const float *ws, hipStream_t st) {
    const float *part = ws + p.rows_bytes / 4;
    long long row_wgs = p.row_splits > 1 ? (long long)a.pg.NKV * p.most * a.pg.n_seqs : 0;
    if (FEW) row_wgs = (row_wgs + pj_heads(D) - 1) / pj_heads(D);
    const long long wgs = row_wgs + (p.chunk_splits > PC_FEW ? (long long)a.pg.n_tokens * a.NQ
                                     : p.chunk_splits > 1   ? (long long)a.pg.n_tokens * ((a.NQ + pj_heads(D) - 1) / pj_heads(D))
                                                            : 0);
    if (wgs > PG_WGS) return hipErrorInvalidConfiguration;
    if (wgs > 0)
        hipLaunchKernelGGL((k_pg_join<TO, D, HL, FEW>), dim3((unsigned)wgs), dim3(PJ_THREADS), 0, st, a, p.nrb, p.row_tps,
                           p.row_splits, ws, (int)row_wgs, p.most, p.chunk_splits, part);
    return hipGetLastError();
}

// Over 4-bit pages.  A batch's few splits of many rows: D / 4 lanes a row (2048 rows of up to 5 splits 7.2 -> 4.6 us);
// else a workgroup (256 rows of 17 2.9 against 4.2, of 33 2.9 against 6.2).
template <typename TO, int D, bool HL>
static hipError_t mx_join(const PgAttn &a, const PgPlan &p, const float *ws, hipStream_t st) {
    const bool few = p.row_splits <= 8 && (long long)a.pg.NKV * p.most * a.pg.n_seqs > 512;
    return few ? pg_join<TO, D, HL, true>(a, p, ws, st) : pg_join<TO, D, HL, false>(a, p, ws, st);
}
hipError_t launch_mx_join(const PgAttn &a, int D, const PgPlan &p, bool f32, int out_type, const float *ws, hipStream_t st) {
    if (f32) return D == 128 ? mx_join<float, 128, true>(a, p, ws, st) : mx_join<float, 64, true>(a, p, ws, st);
    if (out_type == TBQ_KV_F32) return D == 128 ? mx_join<float, 128, false>(a, p, ws, st) : mx_join<float, 64, false>(a, p, ws, st);
    if (out_type == TBQ_KV_F16) return D == 128 ? mx_join<pg_f16, 128, false>(a, p, ws, st) : mx_join<pg_f16, 64, false>(a, p, ws, st);
    return D == 128 ? mx_join<pg_bf16, 128, false>(a, p, ws, st) : mx_join<pg_bf16, 64, false>(a, p, ws, st);
}

template <typename TC, int D, bool HL>
static hipError_t pg_attn(PgAttn a, float *ws, hipStream_t st) {
    const PgPlan p = pg_plan(a.pg, D, a.NQ, a.window, a.sinks, HL, TBQ_KV_F16);
    a.few = p.few;
    float *part = ws + p.rows_bytes / 4;
    if (!p.chunks) {
        const dim3 grid(a.pg.NKV * p.nrb, p.row_splits, a.pg.n_seqs);
        if (p.nrb == 1)
            hipLaunchKernelGGL((k_pg_attn_rows<TC, D, HL, true>), grid, dim3(64 * PR_WAVES), 0, st, a, p.nrb, p.row_tps,
                               p.row_splits, ws);
        else
            hipLaunchKernelGGL((k_pg_attn_rows<TC, D, HL, false>), grid, dim3(64 * PR_WAVES), 0, st, a, p.nrb, p.row_tps,
                               p.row_splits, ws);
    } else {
        constexpr int lds = std::max(sizeof(PcLds<D>), sizeof(PrLds<D>));
        static_assert(lds <= 65536, "what a launch may ask for without an attribute of the kernel");
        const long long wgs = (long long)a.pg.NKV * ((long long)p.nrb * p.row_splits * a.pg.n_seqs +
                                                     (long long)p.blocks * p.chunk_splits);
        if (wgs > PG_WGS) return hipErrorInvalidConfiguration;
        hipLaunchKernelGGL((k_pg_attn_chunk<TC, D, HL>), dim3((unsigned)wgs), dim3(64 * PC_WAVES), lds, st, a, p.nrb,
                           p.row_tps, p.row_splits, ws, p.chunk_splits, part);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return HL || a.f32_out ? pg_join<float, D, HL, false>(a, p, ws, st) : pg_join<TC, D, HL, false>(a, p, ws, st);
}

hipError_t launch_pg_attn(const PgAttn &a, int D, int q_type, int c_type, void *ws, hipStream_t st) {
    if (c_type == TBQ_KV_MXFP4) return launch_mx_attn(a, D, q_type, ws, st);
    float *w = (float *)ws;
    if (q_type == TBQ_KV_F32) return D == 128 ? pg_attn<pg_f16, 128, true>(a, w, st) : pg_attn<pg_f16, 64, true>(a, w, st);
    if (c_type == TBQ_KV_F16) return D == 128 ? pg_attn<pg_f16, 128, false>(a, w, st) : pg_attn<pg_f16, 64, false>(a, w, st);
    return D == 128 ? pg_attn<pg_bf16, 128, false>(a, w, st) : pg_attn<pg_bf16, 64, false>(a, w, st);
}

}  // namespace tbq
