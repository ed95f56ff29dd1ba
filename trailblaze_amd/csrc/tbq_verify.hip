// tbq_verify.hip -- drafted tokens against the target's logits from given random
// numbers (include/tbq_kv.h, tbq_draft_verify) on gfx950.
//
// p = softmax(l / T).  A draft x stays where u q(x) < p(x); behind the first that
// does not, the next token is drawn from max(p - q, 0), behind the last draft from
// p: the first token whose cumulative weight, in the order of the vocabulary, is above u times the
// whole.  Which token that is changes at as many borders as there are tokens, so
// weights and sums are fp64: with fp32's 1e-7 one draw in thirty over 150000 tokens
// would depend on the order of a sum, with fp64 one in 10^10.
//
// Three launches: a chunk's largest logit and sum of exponentials, for all rows;
// with a draft model, the sums of max(p - q, 0) a chunk for the one row of a
// sequence that is drawn from; and the draw, which looks for its token in one chunk.
#include "tbq_kernels.h"
#include "tbq_serve.hpp"

namespace tbq {

constexpr int DV_THREADS = 256, DV_PICK = 1024;

struct DvRec {      // of a chunk of a row: the largest logit, where first, and the sum of the weights 2^(k (l - m))
    float m;
    int at;         // (of rows without a temperature only)
    double sum;
};
typedef DvRec DvRow;   // of a row: the same

// 2^t for t <= 0: t = k + r, |r| <= 1/2, and the series of 2^r up to the term in which the next
// one, (ln 2 / 2)^12 / 12!, is below 2^-47 of the whole; a NaN gives 0.  (The library's exp takes twice as
// long: 218 + 154 rows of 151936 113 us, 5x with this one.)
__device__ __forceinline__ double dv_exp2(double t) {
    t = fmax(t, -1100.);
    const double k = __builtin_rint(t), r = t - k;
    double p = 4.4455382718708116e-10;   // (ln 2)^11 / 11!
    p = fma(p, r, 7.0549116208011234e-9);
    p = fma(p, r, 1.0178086009239699e-7);
    p = fma(p, r, 1.3215486790144309e-6);
    p = fma(p, r, 1.5252733804059841e-5);
    p = fma(p, r, 1.5403530393381609e-4);
    p = fma(p, r, 1.3333558146428443e-3);
    p = fma(p, r, 9.6181291076284772e-3);
    p = fma(p, r, 5.5504108664821580e-2);
    p = fma(p, r, 2.4022650695910071e-1);
    p = fma(p, r, 6.9314718055994531e-1);
    return ldexp(fma(p, r, 1.), (int)k);
}
// The weight exp((l - m) / T) for l <= m, k = log2(e) / T: 1 for the largest itself (also where it is infinite), 0 for
// -infinity and NaN.
__device__ __forceinline__ double dv_weight(float l, float m, double k) {
    return l == m ? 1. : dv_exp2(((double)l - (double)m) * k);
}

__device__ __forceinline__ double dv_sum64(double v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// N elements of a row from element i on (-infinity behind the end).
template <typename T, int N>
__device__ __forceinline__ void dv_load(const T *row, int i, int n, float (&x)[N]) {
    typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const float none = -__builtin_huge_valf();
    if (i + N <= n) {
        const vec v = *reinterpret_cast<const vec *>(row + i);
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = i + e < n ? (float)row[i + e] : none;
    }
}

// Whether sequence s has its rows among the call's.
__device__ __forceinline__ bool dv_rows(const SvVerify &a, int s, int *q0, int *n) {
    *q0 = a.q_start[s];
    *n = a.q_start[s + 1] - *q0;
    return *q0 >= 0 && *n > 0 && *n <= a.n_rows - *q0;
}
// A random number, within [0, 1) as the largest and smallest floats there (a NaN: 0).
__device__ __forceinline__ double dv_random(float u) { return fminf(fmaxf(u, 0.f), 0x1.fffffep-1f); }
// log2(e) over the temperature; 0: all weight on the largest logit.
__device__ __forceinline__ double dv_rate(const SvVerify &a, int s) {
    const double t = a.temperature ? a.temperature[s] : 1.;
    return t > 0. ? fmax(1.4426950408889634 / t, 1e-300) : 0.;
}

// Block x: chunk, row, and (draft) whose logits.  Bound by HBM and the exponentials' fp64.
template <typename T, int CH>
__global__ __launch_bounds__(DV_THREADS) void k_dv_stats(const SvVerify a, DvRec *__restrict__ rec) {
    constexpr int N = CH / DV_THREADS < 16 / (int)sizeof(T) ? CH / DV_THREADS : 16 / sizeof(T), R = CH / DV_THREADS / N;
    __shared__ float ms[DV_THREADS / 64];
    __shared__ int at[DV_THREADS / 64];
    __shared__ double sums[DV_THREADS / 64];
    const int c = blockIdx.x % a.chunks, r = blockIdx.x / a.chunks % a.n_rows, which = blockIdx.x / a.chunks / a.n_rows;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *row = (const T *)(which ? a.draft : a.logits) + r * (which ? a.dstride : a.stride);
    const int v0 = c * CH + (int)threadIdx.x * N;
    float x[R][N];
#pragma unroll
    for (int i = 0; i < R; i++) dv_load(row, v0 + i * DV_THREADS * N, a.vocab, x[i]);
    const int s = pg_seq_of(a.q_start, a.n_seqs, r);
    int q0, n;
    if (s >= a.n_seqs || !dv_rows(a, s, &q0, &n) || r < q0 || (which && r + 1 == q0 + n)) return;
    const double k = dv_rate(a, s);
    float m = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int e = 0; e < N; e++) m = fmaxf(m, x[i][e]);
    m = wave_max(m);
    if (lane == 0) ms[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < DV_THREADS / 64; w++) m = fmaxf(m, ms[w]);
    int first = 0x7FFFFFFF;
    double sum = 0.;
    if (!(k > 0.)) {
#pragma unroll
        for (int i = R - 1; i >= 0; i--)
#pragma unroll
            for (int e = N - 1; e >= 0; e--)
                if (x[i][e] == m) first = v0 + i * DV_THREADS * N + e;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d));
    } else if (m > -__builtin_huge_valf()) {
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int e = 0; e < N; e++) sum += dv_weight(x[i][e], m, k);
        sum = dv_sum64(sum);
    }
    if (lane == 0) {
        sums[wave] = sum;
        at[wave] = first;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.;
#pragma unroll
        for (int w = 0; w < DV_THREADS / 64; w++) {
            sum += sums[w];
            first = min(first, at[w]);
        }
        rec[((long long)which * a.n_rows + r) * a.chunks + c] = {m, first, sum};
    }
}

// A row's records as one, by a wave.
__device__ __forceinline__ DvRow dv_row(const DvRec *rec, int chunks, double k) {
    const int lane = threadIdx.x & 63;
    float m = -__builtin_huge_valf();
    for (int c = lane; c < chunks; c += 64) m = fmaxf(m, rec[c].m);
    m = wave_max(m);
    int at = 0x7FFFFFFF;
    double sum = 0.;
    for (int c = lane; c < chunks; c += 64) {
        const DvRec x = rec[c];
        if (k > 0.) sum += x.sum * dv_weight(x.m, m, k);
        else if (x.m == m) at = min(at, x.at);
    }
    if (k > 0.) return {m, -1, dv_sum64(sum)};
#pragma unroll
    for (int d = 1; d < 64; d *= 2) at = min(at, __shfl_xor(at, d));
    return {m, at, 0.};
}

// What a sequence comes to: the row that its next token is drawn from, and from what.
struct DvChoice {
    int kept, n, x;      // drafts that stay, rows, the draft that was rejected (-1: none)
    int row;
    DvRow p, q;
    double k;            // dv_rate
    int rest;            // weights max(p - q, 0) rather than p
};

// The probability of token x where its row's logit is l.
__device__ __forceinline__ double dv_prob(const DvRow &r, float l, int x, double k) {
    if (!(k > 0.)) return x == r.at && r.m > -__builtin_huge_valf() ? 1. : 0.;
    return r.sum > 0. ? dv_weight(l, r.m, k) / r.sum : 0.;
}
template <typename T>
__device__ __forceinline__ float dv_logit(const void *base, long long stride, int r, int x) {
    return (float)((const T *)base)[r * stride + x];
}

// By a whole workgroup of WAVES waves, a row a wave at a time.
template <typename T, int WAVES>
__device__ __forceinline__ bool dv_choose(const SvVerify &a, const DvRec *rec, int s, DvChoice *out) {
    __shared__ DvChoice ch[WAVES];
    __shared__ int stays[WAVES];
    int q0, n;
    if (!dv_rows(a, s, &q0, &n)) return false;
    const int wave = threadIdx.x >> 6;
    const double k = dv_rate(a, s);
    for (int i0 = 0;; i0 += WAVES) {   // uniform
        const int i = i0 + wave, r = q0 + i;
        int stay = 0;
        if (i < n) {
            DvChoice c;
            c.kept = i;
            c.n = n;
            c.row = r;
            c.k = k;
            c.p = dv_row(rec + (long long)r * a.chunks, a.chunks, k);
            c.q = {0.f, -1, 0.};
            c.x = -1;
            c.rest = 0;
            if (i + 1 < n) {
                const int x = a.tokens[r + 1];
                const bool is = (unsigned)x < (unsigned)a.vocab;
                double px = 0., qx = is ? 1. : 0.;
                if (is) px = dv_prob(c.p, dv_logit<T>(a.logits, a.stride, r, x), x, k);
                if (a.draft) {
                    c.q = dv_row(rec + (long long)(a.n_rows + r) * a.chunks, a.chunks, k);
                    qx = is ? dv_prob(c.q, dv_logit<T>(a.draft, a.dstride, r, x), x, k) : 0.;
                }
                stay = dv_random(a.u_accept[r]) * qx < px;
                c.x = x;
                c.rest = 1;
            }
            if ((threadIdx.x & 63) == 0) ch[wave] = c;
        }
        if ((threadIdx.x & 63) == 0) stays[wave] = stay;
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < WAVES; w++)
            if (!stays[w]) {   // (the last row of a sequence never stays)
                *out = ch[w];
                return true;
            }
        __syncthreads();
    }
}

// The weight of token v in max(p - q, 0), or in p; pi, qi: 1 / the rows' sums (0: no weight).
__device__ __forceinline__ double dv_rest(const DvChoice &c, double pi, double qi, bool draft, float l, float d, int v) {
    const double p = dv_weight(l, c.p.m, c.k) * pi;
    if (!c.rest) return p;
    if (!draft) return v == c.x ? 0. : p;
    return fmax(p - dv_weight(d, c.q.m, c.k) * qi, 0.);
}

// With a draft model: what each sequence comes to, and the sums of its weights a chunk.  x: chunk,
// sequence.
template <typename T, int CH>
__global__ __launch_bounds__(DV_THREADS) void k_dv_rest(const SvVerify a, const DvRec *__restrict__ rec,
                                                        DvChoice *__restrict__ choice, double *__restrict__ rest) {
    constexpr int N = CH / DV_THREADS < 16 / (int)sizeof(T) ? CH / DV_THREADS : 16 / sizeof(T), R = CH / DV_THREADS / N;
    __shared__ double sums[DV_THREADS / 64];
    const int ck = blockIdx.x % a.chunks, s = blockIdx.x / a.chunks;
    DvChoice c;
    if (!dv_choose<T, DV_THREADS / 64>(a, rec, s, &c)) return;
    if (ck == 0 && threadIdx.x == 0) choice[s] = c;
    if (!c.rest || !(c.k > 0.) || !(c.p.sum > 0.)) return;   // the draw does without
    const T *l = (const T *)a.logits + c.row * a.stride, *d = (const T *)a.draft + c.row * a.dstride;
    const int v0 = ck * CH + (int)threadIdx.x * N;
    float x[R][N], y[R][N];
#pragma unroll
    for (int i = 0; i < R; i++) {
        dv_load(l, v0 + i * DV_THREADS * N, a.vocab, x[i]);
        dv_load(d, v0 + i * DV_THREADS * N, a.vocab, y[i]);
    }
    const double pi = 1. / c.p.sum, qi = c.q.sum > 0. ? 1. / c.q.sum : 0.;
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int e = 0; e < N; e++) sum += dv_rest(c, pi, qi, true, x[i][e], y[i][e], 0);
    sum = dv_sum64(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.;
#pragma unroll
        for (int w = 0; w < DV_THREADS / 64; w++) sum += sums[w];
        rest[(long long)s * a.chunks + ck] = sum;
    }
}

// Inclusive sum over the workgroup of DV_PICK threads, and the whole one.
__device__ __forceinline__ double dv_scan(double v, double *lds, double *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    double before = 0., all = 0.;
    for (int w = 0; w < DV_PICK / 64; w++) {
        before += w < wave ? lds[w] : 0.;
        all += lds[w];
    }
    *total = all;
    return before + v;
}

// The draw, a workgroup a sequence.
template <typename T, int CH>
__global__ __launch_bounds__(DV_PICK) void k_dv_pick(const SvVerify a, const DvRec *__restrict__ rec,
                                                     const DvChoice *__restrict__ choice, const double *__restrict__ rest) {
    constexpr int EACH = CH / DV_PICK;
    __shared__ double red[DV_PICK / 64], before;
    __shared__ int found, last;
    const int s = blockIdx.x, tid = threadIdx.x;
    DvChoice c;
    bool is;
    if (choice) {
        int q0, n;
        is = dv_rows(a, s, &q0, &n);
        if (is) c = choice[s];
    } else is = dv_choose<T, DV_PICK / 64>(a, rec, s, &c);
    int next = -1;
    if (is && !(c.k > 0.)) {
        if (c.p.m > -__builtin_huge_valf()) next = c.p.at;
    } else if (is && c.p.sum > 0.) {
        const T *l = (const T *)a.logits + c.row * a.stride;
        const T *d = a.draft ? (const T *)a.draft + c.row * a.dstride : nullptr;
        const double u = dv_random(a.u_next[s]), pi = 1. / c.p.sum, qi = c.q.sum > 0. ? 1. / c.q.sum : 0.;
        double w[EACH];
        // the weights of a chunk's elements, EACH side by side a thread, and their sum
        auto weights = [&](int ck) {
            const int v0 = ck * CH + tid * EACH;
            float x[EACH], y[EACH];
            dv_load(l, v0, a.vocab, x);
            if (d && c.rest) dv_load(d, v0, a.vocab, y);
            double sum = 0.;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                w[e] = dv_rest(c, pi, qi, d != nullptr, x[e], y[e], v0 + e);
                sum += w[e];
            }
            return sum;
        };
        // a chunk's sum: as the record has it, or k_dv_rest, or (the rejected guess's own chunk) anew
        const int own = c.rest && !d && (unsigned)c.x < (unsigned)a.vocab ? c.x / CH : -1;
        double anew = 0., total = 0.;
        if (own >= 0) dv_scan(weights(own), red, &anew);
        auto mass = [&](int k) {
            if (c.rest && d) return rest[(long long)s * a.chunks + k];
            if (c.rest && k == own) return anew;
            const DvRec r = rec[(long long)c.row * a.chunks + k];
            return r.sum * dv_weight(r.m, c.p.m, c.k) * pi;
        };
        // a thread's chunks lie side by side
        const int per = (a.chunks + DV_PICK - 1) / DV_PICK, k0 = min(tid * per, a.chunks), k1 = min(k0 + per, a.chunks);
        double mine = 0., run = 0.;
        for (int round = 0; round < 2; round++) {   // (nothing left of p - q: p itself)
            mine = 0.;
            for (int k = k0; k < k1; k++) mine += mass(k);
            run = dv_scan(mine, red, &total) - mine;
            if (total > 0.) break;
            c.rest = 0;
        }
        if (tid == 0) {
            found = 0x7FFFFFFF;
            last = -1;
        }
        __syncthreads();
        // the first chunk whose end is above u * total; the last that has any weight, where rounding
        // leaves none
        double at[2] = {0., 0.};
        int f = 0x7FFFFFFF, z = -1;
        for (int k = k0; k < k1; k++) {
            const double m = mass(k);
            if (m > 0. && run + m > u * total && f == 0x7FFFFFFF) {
                f = k;
                at[0] = run;
            }
            if (m > 0.) {
                z = k;
                at[1] = run;
            }
            run += m;
        }
        if (f != 0x7FFFFFFF) atomicMin(&found, f);
        if (z >= 0) atomicMax(&last, z);
        __syncthreads();
        const int ck = found != 0x7FFFFFFF ? found : last;
        if (ck == f) before = at[0];
        else if (found == 0x7FFFFFFF && ck >= 0 && ck == z) before = at[1];
        __syncthreads();
        if (ck >= 0) {
            if (tid == 0) {
                found = 0x7FFFFFFF;
                last = -1;
            }
            mine = weights(ck);
            double all;
            run = before + (dv_scan(mine, red, &all) - mine);
            f = 0x7FFFFFFF;
            z = -1;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                run += w[e];
                if (w[e] > 0.) {
                    z = e;
                    if (run > u * total && f == 0x7FFFFFFF) f = e;
                }
            }
            const int v0 = ck * CH + tid * EACH;
            if (f != 0x7FFFFFFF) atomicMin(&found, v0 + f);
            if (z >= 0) atomicMax(&last, v0 + z);
            __syncthreads();
            next = found != 0x7FFFFFFF ? found : last;
        }
    }
    if (tid == 0) {
        a.n_accept[s] = is ? c.kept : 0;
        a.next[s] = (unsigned)next < (unsigned)a.vocab ? next : -1;   // (falling starts: whatever the records hold)
        if (a.n_drop) a.n_drop[s] = is ? c.n - 1 - c.kept : 0;
    }
}

int verify_chunk(int n_rows, int vocab, bool draft) {
    return (long long)n_rows * (draft ? 2 : 1) * vocab <= 512ll * DV_LONG ? DV_SHORT : DV_LONG;
}

size_t verify_workspace_bytes(int n_seqs, int n_rows, int vocab, bool draft) {
    const size_t ch = verify_chunk(n_rows, vocab, draft), chunks = ((size_t)vocab + ch - 1) / ch;
    const size_t n = (size_t)n_rows * (draft ? 2 : 1) * chunks * sizeof(DvRec);
    return draft ? n + (size_t)n_seqs * (chunks * sizeof(double) + sizeof(DvChoice)) : n;
}

template <typename T, int CH>
static hipError_t verify(SvVerify a, void *ws, hipStream_t st) {
    a.chunks = (a.vocab + CH - 1) / CH;
    const long long wgs = (long long)a.n_rows * (a.draft ? 2 : 1) * a.chunks;
    if (wgs > (1ll << 32) / DV_THREADS - 1 || (long long)a.n_seqs * a.chunks > (1ll << 32) / DV_THREADS - 1)
        return hipErrorInvalidConfiguration;
    DvRec *rec = (DvRec *)ws;
    DvChoice *choice = a.draft ? (DvChoice *)(rec + wgs) : nullptr;
    double *rest = a.draft ? (double *)(choice + a.n_seqs) : nullptr;
    if (wgs > 0) hipLaunchKernelGGL((k_dv_stats<T, CH>), dim3((unsigned)wgs), dim3(DV_THREADS), 0, st, a, rec);
    if (a.draft && wgs > 0)
        hipLaunchKernelGGL((k_dv_rest<T, CH>), dim3((unsigned)(a.n_seqs * a.chunks)), dim3(DV_THREADS), 0, st, a, rec, choice,
                           rest);
    hipLaunchKernelGGL((k_dv_pick<T, CH>), dim3(a.n_seqs), dim3(DV_PICK), 0, st, a, rec, choice, rest);
    return hipGetLastError();
}

template <typename T>
static hipError_t verify_t(const SvVerify &a, void *ws, hipStream_t st) {
    return verify_chunk(a.n_rows, a.vocab, a.draft != nullptr) == DV_SHORT ? verify<T, DV_SHORT>(a, ws, st)
                                                                          : verify<T, DV_LONG>(a, ws, st);
}

hipError_t launch_verify(const SvVerify &a, int type, void *ws, hipStream_t st) {
    return type == TBQ_KV_F32 ? verify_t<float>(a, ws, st) : type == TBQ_KV_F16 ? verify_t<pg_f16>(a, ws, st) : verify_t<pg_bf16>(a, ws, st);
}

}  // namespace tbq
