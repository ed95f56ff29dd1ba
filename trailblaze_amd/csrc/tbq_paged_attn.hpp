// tbq_paged_attn.hpp -- what the attention kernels over the paged key/value
// cache share: tbq_paged_attn.hip (16-bit pages) and tbq_paged_mx_attn.hip (4-bit
// pages).  Tiles and masks, the rows' and chunks' division into workgroups, and
// the host's plan of their splits.
#pragma once

#include "tbq_paged.hpp"

namespace tbq {

constexpr float PG_LOW = -3.402823466e38f;   // the running maximum before any score
constexpr float PG_TINY = 1.17549435e-38f;   // least scale: a hidden score, -infinity, times it stays one

template <typename T>
struct PgVec;
template <>
struct PgVec<pg_f16> {
    typedef pg_f16 h8 __attribute__((ext_vector_type(8)));
    static constexpr float SHIFT = 14.f;
};
template <>
struct PgVec<pg_bf16> {
    typedef pg_bf16 h8 __attribute__((ext_vector_type(8)));
    static constexpr float SHIFT = -32.f;
};
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef float pg_f16x __attribute__((ext_vector_type(16)));

__device__ __forceinline__ pg_f4 pg_mfma16(PgVec<pg_f16>::h8 a, PgVec<pg_f16>::h8 b, pg_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ pg_f4 pg_mfma16(PgVec<pg_bf16>::h8 a, PgVec<pg_bf16>::h8 b, pg_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ pg_f16x pg_mfma32(PgVec<pg_f16>::h8 a, PgVec<pg_f16>::h8 b, pg_f16x c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ pg_f16x pg_mfma32(PgVec<pg_bf16>::h8 a, PgVec<pg_bf16>::h8 b, pg_f16x c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The tiles of TS positions that tokens at plo .. phi see any part of: first
// the sinks' tiles in front of the window, then the window's.
struct PgTiles {
    int sinks, first, n;
    __device__ __forceinline__ int at(int it) const { return it < sinks ? it : first + it - sinks; }
};
template <int TS>
__device__ __forceinline__ PgTiles pg_tiles(int plo, int phi, int window, int sinks, int max_kv) {
    phi = min(phi, max_kv - 1);
    if (phi < 0) return {0, 0, 0};
    const int lo = window > 0 ? max(0, plo - window + 1) : 0;
    if (lo > phi) return {0, 0, 0};
    const int first = lo / TS, ns = min((min(sinks, phi + 1) + TS - 1) / TS, first);
    return {ns, first, ns + phi / TS - first + 1};
}

// Bit k: whether position k0 + k of 64 is in (lo, hi] or, up to hi, below sinks.
__device__ __forceinline__ uint64_t pg_upto(int k) { return k < 0 ? 0ull : k >= 63 ? ~0ull : (2ull << k) - 1ull; }
__device__ __forceinline__ uint64_t pg_seen(int k0, int lo, int hi, int sinks) {
    return pg_upto(hi - k0) & (~pg_upto(lo - k0) | pg_upto(sinks - 1 - k0));
}
// All ones where bit c of m is set.
__device__ __forceinline__ uint32_t pg_ones(uint32_t m, int c) { return (uint32_t)__builtin_amdgcn_sbfe((int)m, c, 1); }
// s where its mask is ones, -infinity where it is 0.
__device__ __forceinline__ float pg_hide(float s, uint32_t ones) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, s) & ones) | (0xFF800000u & ~ones));
}

// The page of a 16-position block, -1 where there is none to read: blocks past
// the last visible position are not looked up.
__device__ __forceinline__ int pg_block_page(const PgArgs &a, int s, int pos, int last) {
    return pos <= last ? pg_page(a, s, pos) : -1;
}

// Power of two that puts a row's largest element in [2^13, 2^14).
__device__ __forceinline__ int pg_row_shift(float amax) {
    int e = 0;
    frexpf(amax, &e);
    const int sh = amax > 0.f ? 14 - e : 0;
    return min(max(sh, -126), 126);
}

// The halves of v, or zeros, by a mask of ones or 0.
template <typename V>
__device__ __forceinline__ V pg_keep(V v, uint32_t ones) {
    typedef uint32_t w __attribute__((ext_vector_type(sizeof(V) / 4)));
    w x = __builtin_bit_cast(w, v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); i++) x[i] &= ones;
    return __builtin_bit_cast(V, x);
}

constexpr int pg_rec(int D) { return D + 4; }   // floats of a split's record: D outputs, max, sum, padding

constexpr int PR_WAVES = 4, PR_TS = 32;
// Rows up to which a sequence is one of few rows (PgAttn::few): PR_MAX, or half as
// many where the batch's keys and values are more than the 256 MiB that the last
// cache holds, so that each row block reads them from HBM again.  8 tokens of 4
// heads a kv head, fp16, as two row blocks / as many rows: 1 sequence after 4096
// positions 13.7 / 19.4 us, 32 after 1000 34.4 / 43.4, 32 after 4096 155 / 119, 64
// after 4096 294 / 212; 16 tokens of 8 sequences after 2000 40.0 as four, 33.4 as
// many.  fp32 as four blocks / as many: 24 after 1000 41.8 / 50.2, 64 after 4096
// 417 / 284; 4 tokens as two / as many: 64 after 4096 267 / 275.  One token of 17 to 32
// heads a kv head, fp16, as two / as many: 32 heads of 64 sequences over 4096 260 / 211, of
// 5 over 65536 202 / 172, of 9 over 16384 142 / 156; 17 heads of 64 over 2000 114 / 120;
// fp32 (four blocks) 32 heads of 64 over 4096 362 / 280, of 9 over 16384 207 / 182.
constexpr int PR_MAX = 32;
// Over 4-bit pages a row block's codes become halves in registers, where many rows wait for them in LDS.  So where no
// sequence has more than PR_MOST rows, 16-bit ones are few whatever the batch, and fp32 ones up to PR_MAX, or up to PR_MOST in
// batches of up to PR_SHORT32 positions of kv heads that, as many rows, would be less than a block a CU.  As row blocks / as
// many rows, fp16, 32 / 8 heads of 128: 20 rows a kv head, 1 sequence after 300 positions 7.4 / 15.2 us, 64 after 4096 100 /
// 191, after 32768 708 / 1494, 1000 after 300 163 / 351; 48 rows, 64 after 4096 150 / 198; 64 rows, 32 after 4096 101 / 109,
// 64 after 300 24.2 / 23.1, after 32768 1274 / 1553; 16 / 8 heads of 64, 64 rows, 64 after 300 18.7 / 19.9, 32 after 4096 75 / 83.
// fp32, 32 / 8 heads of 128: 20 rows, 64 after 4096 143 / 233; 32 rows, 64 after 4096 188 / 236; 64 rows, 1 after 16384 and 4
// after 4096 32 / 37, 32 after 300 26.8 / 20.4, 64 after 1000 90 / 67; 16 / 8 heads of 64: 32 rows, 64 after 300 20.9 / 19.1,
// after 4096 144 / 150, 64 rows, 16 after 1000 22.6 / 26.6, 4 after 16384 73 / 51.
// Beside longer prompts the blocks that a short sequence does not have are workgroups all the same, so there it is PR_MOST in
// batches of PR_SHORT positions only (fp32: PR_SHORT32), else half as many again as over 16-bit pages for 16-bit rows: 64
// single tokens to 8192 beside a prompt of 1000, fp16, up to 16 rows as few 126 us, up to 64 215; 32 x 5 tokens beside one of
// 500 up to 48 80, up to 64 102.
constexpr int PR_MOST = 64, PR_SHORT = 1 << 19, PR_SHORT32 = 1 << 17;
constexpr int PR_MIN = 4, PR_LONG = 64;   // tiles of a split: one a wave at least, 2048 positions at most
constexpr int PR_MANY = 1024;              // (in batches of up to twice so many workgroups)

template <int D>
struct PrLds {
    float o[PR_WAVES][16 * (D + 4)], m[PR_WAVES][16], l[PR_WAVES][16];
};

// The end of a workgroup of few rows: its waves' maxima, sums and outputs are added
// and written (nz <= 1), or kept as split z's record of each row in part.  o[j],
// register r of lane (li, h): row li, dims ND (4 h + r) + j; HL: rows 8 .. 15 are the lo
// halves' shares.
// fix: called by every wave between its stores and the workgroup's sum (rows formed again).
struct PgNoFix {
    __device__ __forceinline__ void operator()() const {}
};
template <typename TO, int D, bool HL, typename Fix = PgNoFix>
__device__ __forceinline__ void pg_rows_out(const PgAttn &a, pg_f4 (&o)[D / 16], float m, float l, int r0, int rows, int G,
                                            int kvh, int q0, int s, int z, int nz, int nrb, int nsplit, float *__restrict__ part,
                                            PrLds<D> *lds, Fix fix = Fix{}) {
    constexpr int RB = HL ? 8 : 16, ND = D / 16, OST = D + 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, h = lane >> 4;
    l = swap32_sum(swap16_sum(l));
    // accumulator register r of lane (li, h): row li, dims ND (4 h + r) + j
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int j = 0; j < ND; j += 4)
            *reinterpret_cast<float4 *>(&lds->o[wave][li * OST + ND * (4 * h + r) + j]) =
                make_float4(o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]);
    if (h == 0) {
        lds->m[wave][li] = m;
        lds->l[wave][li] = l;
    }
    fix();
    __syncthreads();
    for (int i = threadIdx.x; i < RB * D / 4; i += 64 * PR_WAVES) {
        const int c = i / (D / 4), d = i % (D / 4) * 4, r = r0 + c;
        if (r >= rows) break;
        float M = lds->m[0][c];
#pragma unroll
        for (int w = 1; w < PR_WAVES; w++) M = fmaxf(M, lds->m[w][c]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < PR_WAVES; w++) {
            const float f = __builtin_amdgcn_exp2f(lds->m[w][c] - M);
            float4 y = *reinterpret_cast<const float4 *>(&lds->o[w][c * OST + d]);
            if constexpr (HL) {
                const float4 y2 = *reinterpret_cast<const float4 *>(&lds->o[w][(c + 8) * OST + d]);
                y = make_float4(y.x + y2.x, y.y + y2.y, y.z + y2.z, y.w + y2.w);
            }
            sum = make_float4(fmaf(f, y.x, sum.x), fmaf(f, y.y, sum.y), fmaf(f, y.z, sum.z), fmaf(f, y.w, sum.w));
            den = fmaf(f, lds->l[w][c], den);
        }
        if (nz <= 1) {
            const float inv = den == 0.f ? 0.f : 1.0f / den;   // a row that sees nothing is 0
            const long long at = ((long long)(q0 + r / G) * a.NQ + kvh * G + r % G) * D + d;
            sum = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
            if (HL || a.f32_out) pg_st4((float *)a.out + at, sum);
            else pg_st4((TO *)a.out + at, sum);
        } else {
            float *rec = part + ((((long long)s * a.pg.NKV + kvh) * nrb * RB + r) * nsplit + z) * pg_rec(D);
            *reinterpret_cast<float4 *>(rec + d) = sum;
            if (d == 0) {
                rec[D] = M;
                rec[D + 1] = den;
            }
        }
    }
}

constexpr int PC_WAVES = 4, PC_TS = 64, PC_ROWS = 32 * PC_WAVES;


typedef short pg_s4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ pg_s4 pg_read_tr(uint32_t addr) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pg_s4 *)(uintptr_t)addr);
}

// Block y of the batch: its sequence s (-1: there is none) with its first token row,
// its tokens and positions, and the block's number in it.  One round of loads.
struct PcBlock {
    int s, q0, qn, len, yb;
};
__device__ __forceinline__ PcBlock pg_chunk_block(const PgArgs &a, int few, int G, int y) {
    const int lane = threadIdx.x & 63;
    for (int i = 0; i < a.n_seqs; i += 64) {
        const int s = min(i + lane, a.n_seqs - 1), q0 = a.q_start[s], qn = a.q_start[s + 1] - q0, len = a.kv_len[s];
        const long long rows = i + lane < a.n_seqs ? (long long)qn * G : 0;
        const int nb = rows > few ? (int)((rows + PC_ROWS - 1) / PC_ROWS) : 0;
        int sum = nb;   // inclusive over the lanes
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const unsigned long long past = __builtin_amdgcn_ballot_w64(sum > y);
        if (past) {
            const int f = __builtin_ctzll(past);
            return {i + f, __builtin_amdgcn_readlane(q0, f), __builtin_amdgcn_readlane(qn, f),
                    __builtin_amdgcn_readlane(len, f), __builtin_amdgcn_readlane(sum, f) - 1 - y};   // the last block first
        }
        y -= __builtin_amdgcn_readlane(sum, 63);
    }
    return {-1, 0, 0, 0, 0};
}

// The splits of a call, by what the host knows (max_q, max_kv, n_tokens).
struct PgPlan {
    int few, most, nrb, row_tps, row_splits;   // few rows: up to, most there can be, row blocks, tiles of a split, splits
    bool chunks;                          // whether a sequence can have many rows
    int blocks, chunk_splits;
    size_t rows_bytes, bytes;             // workspace: the few rows' records, then the others'
};

PgPlan pg_plan(const PgArgs &a, int D, int NQ, int window, int sinks, bool f32, int c_type);

constexpr long long PG_WGS = (1ll << 32) / 256 - 1;   // a launch's threads along x stay below 2^32

// Adds the split ranges of a launch over 4-bit pages (nothing to do where there are none): the few rows'
// records in ws, the others' behind them.  out_type: TBQ_KV_*.
hipError_t launch_mx_join(const PgAttn &a, int D, const PgPlan &p, bool f32, int out_type, const float *ws, hipStream_t st);

}  // namespace tbq
