// tbq_paged_mx_attn.hip -- causal attention of new tokens over a paged key/value
// cache held in MXFP4 (tbq_mx.hpp) on gfx950.
//
// The division of the work, the one pass with the softmax's running maximum and
// sum, and what hidden positions must not do are tbq_paged_attn.hip's.  Here the
// products take halves that the codes and scales become in registers (few rows) or
// on their way to LDS (many rows); the values are halves exactly, so this rounds
// nothing.  16-bit rows of q: fp16 as they are, bf16 scaled by a power of two into
// fp16's range (a row with elements that a half then cannot hold, below 2^-31 of its
// largest one, is formed alone, from q as it is); fp32 rows as two halves each.
// Probabilities are two halves each for every type (2^-22 of one, or 2^-39 of the
// largest, is lost), so a 16-bit row is rounded once, at the output.  As one half they
// would add 17% (few rows, fp16, 64 sequences of up to 8192) and 29% (2048 tokens after
// 8192) to the output's own rounding, 2.1e-4 against 64 bits.
#include <algorithm>
#include <type_traits>

#include "tbq_kernels.h"
#include "tbq_mx.hpp"

namespace tbq {

constexpr float MX_SH = PgVec<pg_f16>::SHIFT;   // probabilities are scaled by 2^14

// One row by one wave, 64 positions at a time, from what the row sees only, as
// pg_slow_row; key(i): the lane's position of the i-th 64 (-1: none).  *m, *l:
// maximum and sum; probabilities, sum and output are scaled by 2^14.
template <typename TA, int D, typename Key>
__device__ __forceinline__ void mx_slow_row(const PgArgs &pg, const TA *q, float cs, int s, int kvh, int pos, int back,
                                            int sinks, int n, Key key, float (&o)[D / 64], float *m, float *l) {
    const int lane = threadIdx.x & 63, last = min(pos, pg.max_kv - 1), mask = (1 << pg.shift) - 1;
    const int codes = (D / 2) << pg.shift;
#pragma unroll
    for (int i = 0; i < D / 64; i++) o[i] = 0.f;
    *m = PG_LOW;
    *l = 0.f;
    for (int it = 0; it < n; it++) {
        const int k = key(it), in = k & mask;
        const int page = k >= 0 ? pg_block_page(pg, s, k, last) : -1;
        const uint8_t *kp = (const uint8_t *)pg.k + mx_head<D>(pg, max(page, 0), kvh);
        const bool sees = page >= 0 && k <= last && (k > pos - back || k < sinks);
        float dot = 0.f;
        for (int g = 0; g < D / 8; g++) {
            const mx_h8 y = mx_eight(*reinterpret_cast<const uint32_t *>(kp + mx_k_code<D>(in, g)),
                                     mx_scale(kp[codes + mx_k_scale<D>(in, g / 4)]));
            const float4 a = pg_ld4(q + 8 * g), b = pg_ld4(q + 8 * g + 4);
            const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; e++) dot = fmaf(x[e], (float)y[e], dot);
        }
        dot = sees ? dot * cs : -__builtin_huge_valf();
        const float mn = fmaxf(*m, wave_max(dot)), corr = __builtin_amdgcn_exp2f(*m - mn);
        const float p = __builtin_amdgcn_exp2f(dot - mn + MX_SH);
        *m = mn;
        *l = *l * corr + group_sum<64>(p);
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] *= corr;
        for (unsigned long long left = __builtin_amdgcn_ballot_w64(sees); left; left &= left - 1) {
            const int c = __builtin_ctzll(left), kin = __builtin_amdgcn_readlane(in, c);
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), c));
            const uint8_t *vp = (const uint8_t *)pg.v + mx_head<D>(pg, __builtin_amdgcn_readlane(page, c), kvh);
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                const int d = lane + 64 * i;
                const uint32_t x = *reinterpret_cast<const uint32_t *>(vp + mx_v_code<D>(kin, d / 8)) >> (4 * (d % 8));
                o[i] = fmaf(w, (float)mx_pair<0>(x, mx_scale(vp[codes + mx_v_scale<D>(kin, d / 32)]))[0], o[i]);
            }
        }
    }
}

// N dims of row tok's head (from element `at` of q) at `step` elements apart, as halves:
// fp16 as it is, bf16 and fp32 scaled by 2^sh so that the row's largest element (over the
// lanes that share it: spread) lies in [2^13, 2^14); fp32 as hi and lo.  Returns whether a
// bf16 row has an element that is no half then.
template <typename TA, int NS, typename Spread>
__device__ __forceinline__ bool mx_load_q(const TA *q, Spread spread, mx_h8 (&hi)[NS], mx_h8 (&lo)[NS], float *cs) {
    if constexpr (std::is_same<TA, pg_f16>::value) {
#pragma unroll
        for (int i = 0; i < NS; i++) hi[i] = *reinterpret_cast<const mx_h8 *>(q + 8 * i);
        return false;
    } else {
        float x[NS][8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const float4 v = pg_ld4(q + 8 * i + j);
                x[i][j] = v.x;
                x[i][j + 1] = v.y;
                x[i][j + 2] = v.z;
                x[i][j + 3] = v.w;
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
        const int sh = pg_row_shift(spread(mx));
        const float f = ldexpf(1.f, sh), back = ldexpf(1.f, -sh);
        *cs = fmaxf(*cs * back, PG_TINY);
        bool lost = false;
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = x[i][e] * f;
                hi[i][e] = (pg_f16)v;
                if constexpr (std::is_same<TA, float>::value) lo[i][e] = (pg_f16)(v - (float)hi[i][e]);
                else lost |= (float)hi[i][e] * back != x[i][e];
            }
        return spread(lost ? 1.f : 0.f) > 0.f;
    }
}

// ---------------------------------------------------------------------------
// Few rows.  A workgroup has one sequence, one kv head, 16 rows (8 as fp32: their hi
// halves are the MFMA's columns 0-7, their lo halves 8-15) and a range of tiles of 32
// positions, dealt to its four waves.  Lane (li = l % 16, h = l / 16) loads of each 16
// keys a quarter of row li (D / 4 dims, of one block), which are its part of the A
// operands when the product's dims are taken in that order, and of V D / 16 dims of the
// positions 4 h .. 4 h + 3, whose probabilities it computed; the codes become halves in
// registers.
//
// Bound by HBM where there are many positions: 64 ragged sequences to 8192, 32 / 8 heads
// of 128, fp16 rows 62-64 us, 5.0 TB/s.  What that took (a first form: 81):
//   codes of one row block loaded past the caches: 73 -> 67.5;
//   loads without a condition, so that a whole tile stays in flight, and three waves a SIMD.
// The lo halves' product (fp32 rows': columns of the same one) takes 2 to 5%, up to 11% with
// heads of 64: 64 sequences of 4096 62-65 -> 64-68, of 8192 107 -> 111, of 4096 with 16 / 8 heads of
// 64 44 -> 49 us.
// One sequence of 131072: 18 us (4.0 TB/s), of 4096: 6, a chain of page, codes, products and
// the workgroup's own join.
// ---------------------------------------------------------------------------
template <int D>
struct MxRaw {
    uint32_t kc[2][D / 32], vc[2][4], ks[2], vs[2];
    int k0;          // first position of the tile
    uint32_t has;    // bit b: block b has a page
};

// ONCE: one row block reads the pages, so they need not stay in the caches.
template <typename TA, int D, bool ONCE>
__device__ __forceinline__ void mx_rows(const PgAttn &a, int nrb, int tps, int nsplit, float *__restrict__ part, int x, int z,
                                        int s, PrLds<D> *lds) {
    constexpr bool HL = std::is_same<TA, float>::value;
    constexpr int RB = HL ? 8 : 16, NS = D / 32, ND = D / 16;
    typedef uint32_t kvec __attribute__((ext_vector_type(NS)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, h = lane >> 4;
    const int kvh = x % a.pg.NKV, r0 = x / a.pg.NKV * RB, G = a.NQ / a.pg.NKV;
    const int q0 = a.pg.q_start[s], qn = a.pg.q_start[s + 1] - q0;
    if (qn <= 0 || q0 < 0 || qn > a.pg.n_tokens - q0 || qn > PR_MOST) return;
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
    mx_h8 qf[NS];
    float cs = fmaxf(a.scale, PG_TINY);
    uint64_t lost;   // of the lanes' rows
    {
        mx_h8 lo[NS];
        const TA *q = (const TA *)a.q + (long long)(q0 + tok) * a.qs + (long long)(kvh * G + rc % G) * D + D / 4 * h;
        lost = __builtin_amdgcn_ballot_w64(
            mx_load_q(q, [](float v) { return swap32_max(swap16_max(v)); }, qf, lo, &cs));
        if constexpr (HL) {
#pragma unroll
            for (int i = 0; i < NS; i++)
                if (li >= 8) qf[i] = lo[i];
        }
    }
    const int nt = (it1 - it0 - wave + PR_WAVES - 1) / PR_WAVES;   // this wave's tiles
    auto tile_at = [&](int n) { return tiles.at(it0 + wave + PR_WAVES * n) * PR_TS; };
    const uint32_t koff = li * (D / 2) + D / 8 * h, ksoff = li * (D / 32) + h * (D / 32) / 4;
    const uint32_t voff = 2 * D * h + 16 * (li * ND / 8), vsoff = D / 8 * h + 4 * (li * ND / 32);
    // lane i, of block i % 2 of the wave's tile i / 2 (of 32 tiles): bytes before its codes, from them to
    // its scales; bit i of pages: whether it has a page
    uint32_t off_lo = 0, off_hi = 0, to_scales = 0;
    uint64_t pages = 0;
    auto get = [](const auto *p) {
        if constexpr (ONCE) return __builtin_nontemporal_load(p);
        else return *p;
    };
    auto load = [&](MxRaw<D> &w, int n) {
        if ((n & 31) == 0) {
            const int k = n + (lane >> 1), p = tile_at(k) + 16 * (lane & 1), in = p & ((1 << a.pg.shift) - 1);
            const int page = k < nt ? pg_block_page(a.pg, s, p, last) : -1;
            const long long off = mx_head<D>(a.pg, max(page, 0), kvh) + in * (D / 2);
            pages = __builtin_amdgcn_ballot_w64(page >= 0);
            off_lo = (uint32_t)off;
            off_hi = (uint32_t)(off >> 32);
            to_scales = ((D / 2) << a.pg.shift) - in * (D / 2 - D / 32);
        }
        w.k0 = tile_at(n);
        w.has = (uint32_t)(pages >> (2 * (n & 31))) & 3;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int at = 2 * (n & 31) + b;
            const long long off = (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)off_hi, at) << 32 |
                                              (uint32_t)__builtin_amdgcn_readlane((int)off_lo, at));
            const uint32_t sc = __builtin_amdgcn_readlane((int)to_scales, at);
            const uint8_t *kp = (const uint8_t *)a.pg.k + off, *vp = (const uint8_t *)a.pg.v + off;
            const kvec kc = get(reinterpret_cast<const kvec *>(kp + koff));
#pragma unroll
            for (int i = 0; i < NS; i++) w.kc[b][i] = kc[i];
            const pg_u4 vc = get(reinterpret_cast<const pg_u4 *>(vp + voff));
#pragma unroll
            for (int i = 0; i < 4; i++) w.vc[b][i] = vc[i];
            w.ks[b] = (kp + sc)[ksoff];
            w.vs[b] = *reinterpret_cast<const uint32_t *>(vp + sc + vsoff);
        }
    };
    pg_f4 o[ND];
    float m = PG_LOW, l = 0.f;
#pragma unroll
    for (int j = 0; j < ND; j++) o[j] = pg_f4{};
    auto compute = [&](MxRaw<D> &w) {
        const int k0 = w.k0;
        const bool whole = w.has == 3 && k0 + PR_TS - 1 <= min(plo, a.pg.max_kv - 1) &&
                           (k0 > phi - back || k0 + PR_TS <= a.sinks);
        pg_f4 sc[2] = {pg_f4{}, pg_f4{}};
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < NS; i++) sc[b] = pg_mfma16(mx_eight(w.kc[b][i], mx_scale(w.ks[b])), qf[i], sc[b]);
        if constexpr (HL) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int r = 0; r < 4; r++) sc[b][r] += dpp_f32<0x128>(sc[b][r]);   // row_ror:8
        }
        if (!whole) {
            // the lane's positions that tokens at lo .. hi see: element e is bit 16 (e / 4) + e % 4
            const uint32_t has = (w.has & 1 ? 0xFFFFu : 0u) | (w.has & 2 ? 0xFFFF0000u : 0u);
            auto seen = [&](int lo, int hi) {
                return ((uint32_t)pg_seen(k0, lo - back, min(hi, last), a.sinks) & has) >> (4 * h);
            };
            const uint32_t mine = seen(pos, pos), any = seen(plo, phi);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int bit = 16 * (e / 4) + e % 4;
                sc[e / 4][e % 4] = pg_hide(sc[e / 4][e % 4], pg_ones(mine, bit));
                // values that no row of the block sees are 0 (under whatever scale but NaN)
                const uint32_t on = pg_ones(any, bit);
                w.vc[e / 4][e % 4] &= on;
                w.vs[e / 4] &= on | ~(0xFFu << (8 * (e % 4)));
            }
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
        mx_h8 pf, pl;   // (fp32 rows' lo halves are columns of their own)
        const float mb = MX_SH - m;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / 4][e % 4], cs, mb));
            l += p;
            const pg_f16 hi = (pg_f16)p, lo = (pg_f16)(p - (float)hi);
            if constexpr (HL) pf[e] = li < 8 ? hi : lo;
            else {
                pf[e] = hi;
                pl[e] = lo;
            }
        }
        auto two = [&](auto S) {   // dims 2 S and 2 S + 1 of the lane's ND
            constexpr int I = decltype(S)::value;
            mx_h8 va, vb;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t c = w.vc[e / 4][e % 4] >> (D == 64 ? 16 * (li & 1) : 0);
                const mx_h2 y = mx_pair<I>(c, mx_scale((w.vs[e / 4] >> (8 * (e % 4))) & 0xFFu));
                va[e] = y[0];
                vb[e] = y[1];
            }
            o[2 * I] = pg_mfma16(va, pf, o[2 * I]);
            o[2 * I + 1] = pg_mfma16(vb, pf, o[2 * I + 1]);
            if constexpr (!HL) {
                o[2 * I] = pg_mfma16(va, pl, o[2 * I]);
                o[2 * I + 1] = pg_mfma16(vb, pl, o[2 * I + 1]);
            }
        };
        two(std::integral_constant<int, 0>{});
        two(std::integral_constant<int, 1>{});
        if constexpr (ND == 8) {
            two(std::integral_constant<int, 2>{});
            two(std::integral_constant<int, 3>{});
        }
    };
    if (nt > 0) {
        // (a last load is of a tile that was there already: as many loads are in flight on every way to a
        // product, or the compiler would wait for all of them)
        MxRaw<D> w[2];
        load(w[0], 0);
        for (int n = 0;; n += 2) {
            load(w[1], min(n + 1, nt - 1));
            compute(w[0]);
            if (n + 1 >= nt) break;
            load(w[0], min(n + 2, nt - 1));
            compute(w[1]);
            if (n + 2 >= nt) break;
        }
    }
    // rows with an output that is not finite, and those whose q lost something, are formed again, one at a time
    float odd = 0.f;   // NaN where an output is NaN or infinite
#pragma unroll
    for (int j = 0; j < ND; j++) odd += (o[j][0] - o[j][0]) + (o[j][1] - o[j][1]) + (o[j][2] - o[j][2]) + (o[j][3] - o[j][3]);
    const bool again = row < rows && (!(odd == 0.f) || (lost >> lane & 1));
    pg_rows_out<TA, D, HL>(a, o, m, l, r0, rows, G, kvh, q0, s, z, nz, nrb, nsplit, part, lds, [&] {
        uint64_t left = __builtin_amdgcn_ballot_w64(again);   // lane bits: a row's are li (HL: and li + 8) of each 16
        left |= left >> 32;
        left |= left >> 16;
        left = (HL ? left | left >> 8 : left) & (HL ? 0xFF : 0xFFFF);
        for (; left; left &= left - 1) {
            const int c = __builtin_ctzll(left), r = r0 + c, t = r / G;
            float so[D / 64], sm, sl;
            mx_slow_row<TA, D>(a.pg, (const TA *)a.q + (long long)(q0 + t) * a.qs + (long long)(kvh * G + r % G) * D, a.scale,
                               s, kvh, base + t, back, a.sinks, (nt + 1) / 2,
                               [&](int i) {
                                   const int n = 2 * i + (lane >> 5);
                                   return n < nt ? tile_at(n) + (lane & 31) : -1;
                               },
                               so, &sm, &sl);
#pragma unroll
            for (int i = 0; i < D / 64; i++) {
                lds->o[wave][c * (D + 4) + lane + 64 * i] = so[i];
                if constexpr (HL) lds->o[wave][(c + 8) * (D + 4) + lane + 64 * i] = 0.f;
            }
            if (lane == 0) {
                lds->m[wave][c] = sm;
                lds->l[wave][c] = sl;
            }
        }
    });
}

template <typename TA, int D, bool ONCE>
__global__ __launch_bounds__(64 * PR_WAVES) __attribute__((amdgpu_waves_per_eu(3, 3))) void k_mx_attn_rows(
    const PgAttn a, int nrb, int tps, int nsplit, float *__restrict__ part) {
    __shared__ __attribute__((aligned(16))) PrLds<D> lds;
    mx_rows<TA, D, ONCE>(a, nrb, tps, nsplit, part, blockIdx.x, blockIdx.y, blockIdx.z, &lds);
}

// ---------------------------------------------------------------------------
// Many rows.  pg_chunk's products over LDS tiles of 64 positions as halves; a tile's codes
// come to registers two tiles ahead and to LDS as halves one tile ahead, each wave
// those of one 16-position block.
//
// 2048 tokens after 8192, 32 / 8 heads of 128: 16-bit rows 445-471 us over several cards (0.67 PFLOP/s
// of the attention's, 1.0 with the lo halves' product), fp32 ones, a product of q more, 573; over fp16
// pages 348 and 572.  Matrix units busy for 45% of the cycles, vector units (softmax, halves, the
// codes' conversions) for 53%, at 1.97 GHz: two waves a SIMD overlap little of the two.  With the
// probabilities as one half 348-391, 38% and 47% at 2.07 GHz; 512 after 4096 64 -> 76.  Nine mixed sequences under a
// window of 1024 + 4, heads of 64, bf16: 47-49 (one half: 39), about 19 tiles one after the other in 304
// workgroups on 256 CUs.  Not kept for it, measured with one half: three waves a SIMD, codes two tiles
// ahead in two sets of registers, all of a tile's LDS reads ahead of its products (no change each), the
// positions in two ranges (32, and 9.5 the join), two groups of four waves that share a block's tiles
// and add at the end (44, with registers spilled; heads of 128, where none are: 2048 tokens after none
// 66 -> 60, but 512 after 4096 64 -> 72).
// ---------------------------------------------------------------------------
template <int D>
struct McLds {
    unsigned char k[2][PC_TS * D * 2], v[2][PC_TS * D * 2];
};

// x: kv head + NKV * block; z: split.
template <typename TA, int D>
__device__ __forceinline__ void mx_chunk(const PgAttn &a, int nsplit, float *__restrict__ part, int x, int z,
                                         McLds<D> *st) {
    constexpr bool HL = std::is_same<TA, float>::value;
    constexpr int NT = D / 32, NS = D / 16, SEG = D / 8, NP = HL ? 2 : 1, NC = D / 32;   // dwords of codes a lane
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
    // Q^T's columns: dim step i, lane half h has dims 8 NS h + 8 i .. + 8 (the keys' in that order too)
    mx_h8 qf[NP][NS];
    float cs = fmaxf(a.scale, PG_TINY);
    uint64_t lost;   // of the lanes' rows
    {
        mx_h8 lo[NS];
        const TA *q = (const TA *)a.q + (long long)(q0 + tok) * a.qs + (long long)(kvh * G + rc % G) * D + 8 * NS * h;
        lost = __builtin_amdgcn_ballot_w64(mx_load_q(q, [](float v) { return swap32_max(v); }, qf[0], lo, &cs));
        if constexpr (HL) {
#pragma unroll
            for (int i = 0; i < NS; i++) qf[NP - 1][i] = lo[i];
        }
    }
    auto kswz = [](int r) { return SEG == 16 ? r & 15 : (r & 7) ^ ((r >> 3) & 1); };
    auto vswz = [](int r) { return SEG == 16 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; };
    uint32_t off_lo = 0, off_hi = 0;   // lane i: bytes before the head's page of block i % 4 of tile i / 4 (of 16 tiles)
    uint64_t nopage = 0;               // bit i: lane i's has no page
    const int pmask = (1 << a.pg.shift) - 1, codes = (D / 2) << a.pg.shift;
    auto look_up = [&](int n) {
        const int it = it0 + n + (lane >> 2), p = tiles.at(it) * PC_TS + 16 * (lane & 3);
        const int page = it < it1 ? pg_block_page(a.pg, s, p, last) : -1;
        nopage = __builtin_amdgcn_ballot_w64(page < 0);
        const long long off = mx_head<D>(a.pg, max(page, 0), kvh);
        off_lo = (uint32_t)off;
        off_hi = (uint32_t)(off >> 32);
    };
    // A wave's block of a tile: lane l has a quarter of key l / 4 and, of V, NC positions of 8 dims
    struct Raw {
        uint32_t kc[NC], vc[NC], ks, vs;
    };
    const int kr = lane >> 2, kq = lane & 3, vp4 = lane >> 4;            // of 16 positions; quarter; four positions
    const int vg = D == 128 ? lane & 15 : (lane & 15) >> 1, vi = D == 128 ? 0 : 2 * (lane & 1);   // 8 dims, first position
    typedef uint32_t cvec __attribute__((ext_vector_type(NC)));
    int none = 0, none1 = 0, none2 = 0;   // blocks without a page of the tile, the next and the one after
    auto load = [&](Raw &w, int n) {
        if ((n & 15) == 0) look_up(n);
        none2 = (int)(nopage >> (4 * (n & 15))) & 15;
        const int at = 4 * (n & 15) + wave, in = (tiles.at(it0 + n) * PC_TS + 16 * wave) & pmask;
        const long long off = (long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)off_hi, at) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)off_lo, at));
        const uint8_t *kp = (const uint8_t *)a.pg.k + off, *vp = (const uint8_t *)a.pg.v + off;
        const cvec kc = *reinterpret_cast<const cvec *>(kp + in * (D / 2) + kr * (D / 2) + kq * (D / 8));
        const cvec vc = *reinterpret_cast<const cvec *>(vp + in * (D / 2) + vp4 * 2 * D + 16 * vg + 4 * vi);
#pragma unroll
        for (int i = 0; i < NC; i++) {
            w.kc[i] = kc[i];
            w.vc[i] = vc[i];
        }
        w.ks = kp[codes + (in + kr) * (D / 32) + kq * (D / 32) / 4];
        w.vs = *reinterpret_cast<const uint32_t *>(vp + codes + in * (D / 32) + vp4 * (D / 8) + 4 * (vg / 4));
    };
    auto store = [&](const Raw &w, int buf) {
        const int r = 16 * wave + kr;
#pragma unroll
        for (int i = 0; i < NC; i++)   // dims D / 4 kq + 8 i: segment NC kq + i
            *reinterpret_cast<mx_h8 *>(st->k[buf] + r * (D * 2) + 16 * ((NC * kq + i) ^ kswz(r))) =
                mx_eight(w.kc[i], mx_scale(w.ks));
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const int rv = 16 * wave + 4 * vp4 + vi + i;
            *reinterpret_cast<mx_h8 *>(st->v[buf] + rv * (D * 2) + 16 * (vg ^ vswz(rv))) =
                mx_eight(w.vc[i], mx_scale((w.vs >> (8 * (vi + i))) & 0xFFu));
        }
    };
    auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // V's transposing reads: lane l of 16 addresses position kk = l / 4 of 4, dims 4 (l % 4) .. + 4
    // of 16; of dim block j the address is voff[j] + the step's rows
    const uint32_t lv = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)st->v[0];
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
    float m = PG_LOW, l = 0.f;
    const int ksw = kswz(li);
#pragma unroll
    for (int j = 0; j < NT; j++) o[j] = pg_f16x{};
    const int nt = it1 - it0;
    Raw raw;
    if (nt > 0) {
        load(raw, 0);
        none = none2;
        store(raw, 0);
        if (nt > 1) load(raw, 1);
        none1 = none2;
    }
    barrier();
    for (int n = 0, buf = 0; n < nt; n++, buf ^= 1) {
        const int k0 = tiles.at(it0 + n) * PC_TS;
        if (n + 1 < nt) {
            store(raw, buf ^ 1);
            if (n + 2 < nt) load(raw, n + 2);
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
                barrier();
            }
        }
        const int wlo = base + w0, whi = base + w1;
        if (inner || (k0 <= whi && (k0 + PC_TS > wlo - back || k0 < a.sinks))) {   // the wave's rows see some of it
            const bool whole = inner || (has == ~0ull && k0 + PC_TS - 1 <= min(wlo, last) &&
                                         (k0 > whi - back || k0 + PC_TS <= a.sinks));
            // the positions that tokens at lo .. hi see, from the lane's 4 h on
            auto seen = [&](int lo, int hi) { return (pg_seen(k0, lo - back, min(hi, last), a.sinks) & has) >> (4 * h); };
            const unsigned char *Kb = st->k[buf] + li * (D * 2);
            pg_f16x sc[2] = {pg_f16x{}, pg_f16x{}};
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const mx_h8 y = *reinterpret_cast<const mx_h8 *>(Kb + b * (32 * D * 2) + 16 * ((NS * h + i) ^ ksw));
#pragma unroll
                    for (int p = 0; p < NP; p++) sc[b] = pg_mfma32(y, qf[p][i], sc[b]);
                }
            if (!whole) {
                const uint64_t mine = seen(pos, pos);
#pragma unroll
                for (int e = 0; e < 32; e++)
                    sc[e / 16][e % 16] = pg_hide(sc[e / 16][e % 16],
                                                 pg_ones((uint32_t)(mine >> (e / 16 * 32)), 8 * (e % 16 / 4) + e % 4));
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
            mx_h8 pf[2][4];   // hi and lo halves
            const float mb = MX_SH - m;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 32; e++) {
                const float p = __builtin_amdgcn_exp2f(fmaf(sc[e / 16][e % 16], cs, mb));
                sum += p;
                pf[0][e / 8][e % 8] = (pg_f16)p;
                pf[1][e / 8][e % 8] = (pg_f16)(p - (float)pf[0][e / 8][e % 8]);
            }
            l += sum;
            const uint32_t vb = lv + buf * (PC_TS * D * 2);
            auto vfrag = [&](int u, int j) {
                const pg_s4 y = pg_read_tr(vb + voff[j] + 16 * u * (D * 2)), w = pg_read_tr(vb + voff[j] + (16 * u + 8) * (D * 2));
                return __builtin_shufflevector(y, w, 0, 1, 2, 3, 4, 5, 6, 7);
            };
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const mx_h8 y = __builtin_bit_cast(mx_h8, vfrag(u, j));
#pragma unroll
                    for (int p = 0; p < 2; p++) o[j] = pg_mfma32(y, pf[p][u], o[j]);
                }
        }
        none = none1;
        none1 = none2;
        barrier();
    }
    l = swap32_sum(l);
    // rows with an output that is not finite, and those whose q lost something, are formed again, one at a time
    float odd = 0.f;   // NaN where an output is NaN or infinite
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) odd += o[j][r] - o[j][r];
    odd += __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * (lane ^ 32), __builtin_bit_cast(int, odd)));
    const bool again = row < rows && (!(odd == 0.f) || (lost >> lane & 1));
    auto put = [&](long long at, float v) {
        if (HL || a.f32_out) ((float *)a.out)[at] = v;
        else ((TA *)a.out)[at] = (TA)v;
    };
    for (unsigned long long left = __builtin_amdgcn_ballot_w64(again && h == 0); left; left &= left - 1) {
        const int c = __builtin_ctzll(left), r = r0 + wave * 32 + c, t = r / G;
        float so[D / 64], sm, sl;
        mx_slow_row<TA, D>(a.pg, (const TA *)a.q + (long long)(q0 + t) * a.qs + (long long)(kvh * G + r % G) * D, a.scale, s,
                           kvh, base + t, back, a.sinks, it1 - it0,
                           [&](int i) { return tiles.at(it0 + i) * PC_TS + lane; }, so, &sm, &sl);
        const long long to = (long long)(q0 + t) * a.NQ + kvh * G + r % G;
        float *rec = part + (to * nsplit + z) * pg_rec(D);
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            if (nz > 1) rec[lane + 64 * i] = so[i];
            else put(to * D + lane + 64 * i, sl == 0.f ? 0.f : so[i] / sl);
        }
        if (nz > 1 && lane == 0) {
            rec[D] = sm;
            rec[D + 1] = sl;
        }
    }
    if (again || row >= rows) return;
    const long long at = (long long)(q0 + tok) * a.NQ + kvh * G + row % G;
    const float inv = nz > 1 ? 1.f : l == 0.f ? 0.f : 1.0f / l;   // a row that sees nothing is 0
    float *rec = part + (at * nsplit + z) * pg_rec(D);
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float4 y = make_float4(o[j][4 * r] * inv, o[j][4 * r + 1] * inv, o[j][4 * r + 2] * inv, o[j][4 * r + 3] * inv);
            const int d = 32 * j + 8 * r + 4 * h;
            if (nz > 1) *reinterpret_cast<float4 *>(rec + d) = y;
            else if (HL || a.f32_out) pg_st4((float *)a.out + at * D + d, y);
            else pg_st4((TA *)a.out + at * D + d, y);
        }
    if (nz > 1 && h == 0) {
        rec[D] = m;
        rec[D + 1] = l;
    }
}

// Sequences of many rows and, in the last workgroups, of few.
template <typename TA, int D>
__global__ __launch_bounds__(64 * PC_WAVES)
    __attribute__((amdgpu_waves_per_eu(2, 2))) void k_mx_attn_chunk(const PgAttn a, int nrb, int tps, int row_splits,
                                                                    float *__restrict__ row_part, int nsplit,
                                                                    float *__restrict__ part) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char mx_lds[];
    const int nrows = a.pg.NKV * nrb, chunks = (int)gridDim.x - nrows * row_splits * a.pg.n_seqs, x = blockIdx.x;
    if (x >= chunks) {
        const int y = (x - chunks) / nrows;
        mx_rows<TA, D, false>(a, nrb, tps, row_splits, row_part, (x - chunks) % nrows, y % row_splits, y / row_splits,
                       reinterpret_cast<PrLds<D> *>(mx_lds));
    } else {
        const int y = x / a.pg.NKV;
        mx_chunk<TA, D>(a, nsplit, part, x % a.pg.NKV + a.pg.NKV * (y / nsplit), y % nsplit,
                        reinterpret_cast<McLds<D> *>(mx_lds));
    }
}

template <typename TA, int D>
static hipError_t mx_attn(PgAttn a, int out_type, float *ws, hipStream_t st) {
    constexpr bool HL = std::is_same<TA, float>::value;
    const PgPlan p = pg_plan(a.pg, D, a.NQ, a.window, a.sinks, HL, TBQ_KV_MXFP4);
    a.few = p.few;
    float *part = ws + p.rows_bytes / 4;
    if (!p.chunks) {
        const dim3 grid(a.pg.NKV * p.nrb, p.row_splits, a.pg.n_seqs);
        if (p.nrb == 1)
            hipLaunchKernelGGL((k_mx_attn_rows<TA, D, true>), grid, dim3(64 * PR_WAVES), 0, st, a, p.nrb, p.row_tps,
                               p.row_splits, ws);
        else
            hipLaunchKernelGGL((k_mx_attn_rows<TA, D, false>), grid, dim3(64 * PR_WAVES), 0, st, a, p.nrb, p.row_tps,
                               p.row_splits, ws);
    } else {
        constexpr int lds = std::max(sizeof(McLds<D>), sizeof(PrLds<D>));
        static_assert(lds <= 65536, "what a launch may ask for without an attribute of the kernel");
        const long long wgs = (long long)a.pg.NKV * ((long long)p.nrb * p.row_splits * a.pg.n_seqs +
                                                     (long long)p.blocks * p.chunk_splits);
        if (wgs > PG_WGS) return hipErrorInvalidConfiguration;
        hipLaunchKernelGGL((k_mx_attn_chunk<TA, D>), dim3((unsigned)wgs), dim3(64 * PC_WAVES), lds, st, a, p.nrb, p.row_tps,
                           p.row_splits, ws, p.chunk_splits, part);
    }
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_mx_join(a, D, p, HL, a.f32_out ? TBQ_KV_F32 : out_type, ws, st);
}

hipError_t launch_mx_attn(const PgAttn &a, int D, int q_type, void *ws, hipStream_t st) {
    float *w = (float *)ws;
    if (q_type == TBQ_KV_F32) return D == 128 ? mx_attn<float, 128>(a, q_type, w, st) : mx_attn<float, 64>(a, q_type, w, st);
    if (q_type == TBQ_KV_F16) return D == 128 ? mx_attn<pg_f16, 128>(a, q_type, w, st) : mx_attn<pg_f16, 64>(a, q_type, w, st);
    return D == 128 ? mx_attn<pg_bf16, 128>(a, q_type, w, st) : mx_attn<pg_bf16, 64>(a, q_type, w, st);
}

}  // namespace tbq
