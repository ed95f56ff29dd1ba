// tbq_verify.hip -- drafted tokens against the target's logits from given random
// numbers (include/tbq_kv.h, tbq_draft_verify) on gfx950.
//
// p = softmax(l / T).  A draft x stays where u q(x) < p(x); behind the first that
// does not, the next token is drawn from max(p - q, 0), behind the last draft from
// p: the first token whose cumulative weight, in the order of the vocabulary, is above u times the
// whole.  Which token that is changes at as many borders as there are tokens, so
// weights and sums are fp64, and the weights exact to it: with fp32's 1e-7 one draw in
// thirty over 150000 tokens would depend on roundings, with fp64 one in 10^10.
//
// Three launches: a chunk's largest logit and sum of exponentials, for all rows;
// with a draft model, the sums of max(p - q, 0) a chunk for the one row of a
// sequence that is drawn from; and the draw, which looks for its token in one chunk.
// (A launch of its own says, with a draft model, which row that is: in every workgroup of
// the sums' launch it cost more than it spared.)
#include "tbq_kernels.h"
#include "tbq_serve.hpp"

namespace tbq {

constexpr int DV_THREADS = 256, DV_WIDE = 128, DV_CHOOSE = 1024, DV_PICK = 512;
constexpr int DV_MANY = 4096;   // chunks

struct DvRec {      // of a chunk of a row: the largest logit, where first, and the sum of the weights 2^(k (l - m))
    float m;
    int at;         // (of rows without a temperature only)
    double sum;
};
typedef DvRec DvRow;   // of a row: the same

// The weights exp((l - m) / T) of a row whose largest logit is m, by k = log2(e) / T: 2^t, t = k (l - m).
// t is split into the nearest whole number, which adding 1.5 * 2^52 leaves in the low bits, and r, |r| <= 1/2;
// 2^r is the polynomial of degree 10 that meets it at the eleven Chebyshev points, off by 4e-16 of it at most with the
// roundings (degree 8: 1.1e-12, which moves the borders by up to 4e-9 of the whole in all, and 1 to 3 us less in the case
// below); the whole number goes to the exponent.  Logits from none on have no weight (2^-1000 of the largest, -infinity, NaN); where
// m is infinite, all below it; k is 0 where only m itself has weight.  Those below low count as low: it is none, but for
// temperatures so high that every finite logit has weight (all).  With Least set, logits without weight have up to
// 2^-999, for sums alone (k > 0 and not all).
// (218 + 154 rows of 151936: 113 us with the library's exp, 55 with this.)
struct DvLaw {
    double k, m;
    float low, none;
    __device__ bool all() const { return none < low; }
};
__device__ __forceinline__ DvLaw dv_law(float m, double k) {
    const float most = 3.402823466e38f, inf = __builtin_huge_valf();
    if (!(m <= most)) return {0., most, most, most};
    const double x = (double)m - 1000. * __builtin_amdgcn_rcp(k);   // (the instruction's reciprocal: 1000 or nearly)
    if (x < -(double)most) return {k, m, -most, -inf};
    float low = (float)x;
    if ((double)low < x) low = nextafterf(low, most);   // (not below x)
    // where that leaves no float below m, m alone has weight
    if (low < m) return {k, m, low, low};
    low = nextafterf(m, -inf);
    return {0., m, low, low};
}
template <bool Least = false>
__device__ __forceinline__ double dv_weight(const DvLaw &w, float l) {
    const double t = ((double)__builtin_amdgcn_fmed3f(l, w.low, 3.402823466e38f) - w.m) * w.k, magic = 6755399441055744.;
    const double n = t + magic, r = t - (n - magic);
    double p = 7.072585949269223e-9;
    p = fma(p, r, 1.0208690299958306e-7);
    p = fma(p, r, 1.321544258792169e-6);
    p = fma(p, r, 1.5252657260200837e-5);
    p = fma(p, r, 1.540353044173605e-4);
    p = fma(p, r, 1.3333558230164974e-3);
    p = fma(p, r, 9.618129107606888e-3);
    p = fma(p, r, 5.550410866444772e-2);
    p = fma(p, r, 2.4022650695910097e-1);
    p = fma(p, r, 6.9314718055995e-1);
    p = fma(p, r, 1.);
    const uint64_t b = __builtin_bit_cast(uint64_t, p) + ((uint64_t)(uint32_t)__builtin_bit_cast(uint64_t, n) << 52);
    return Least || l > w.none ? __builtin_bit_cast(double, b) : 0.;
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
    return t > 0. ? fmax(1.4426950408889634 / t, 1e-60) : 0.;   // (1e-60 of any two finite ones is alike)
}

// Block x: chunk, row, and (draft) whose logits.  Bound by the vector units, which have 20 instructions a
// logit to do, 16 of them fp64, and about 170 a wave (218 + 154 rows of 151936, fp32: 55-58 us, 4.0 TB/s, busy for
// 85% of the cycles; with 16 logits a thread and two instructions a logit fewer 59; loads past the caches changed nothing).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_dv_stats(const SvVerify a, DvRec *__restrict__ rec,
                                                         float *__restrict__ drafted, double *__restrict__ others) {
    constexpr int N = 16 / sizeof(T), R = DV_CHUNK / THREADS / N;
    __shared__ float ms[THREADS / 64];
    __shared__ int at[THREADS / 64];
    __shared__ double sums[THREADS / 64], buts[THREADS / 64];
    const int c = blockIdx.x % a.chunks, r = blockIdx.x / a.chunks % a.n_rows, which = blockIdx.x / a.chunks / a.n_rows;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *row = (const T *)(which ? a.draft : a.logits) + r * (which ? a.dstride : a.stride);
    const int v0 = c * DV_CHUNK + (int)threadIdx.x * N;
    float x[R][N];
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < R; i++) dv_load(row, v0 + i * THREADS * N, a.vocab, x[i]);
    };
    if (!which) load();   // (nearly all of the target's rows are some sequence's)
    const int behind = a.tokens[min(r + 1, a.n_rows - 1)];
    const int s = pg_seq_of(a.q_start, a.n_seqs, r);
    int q0, n;
    if (s >= a.n_seqs || !dv_rows(a, s, &q0, &n) || r < q0 || (which && r + 1 == q0 + n)) return;
    if (which) load();
    const double k = dv_rate(a, s);
    const int guess = r + 1 < q0 + n ? behind : -1;   // judged by this row
    const bool has = (unsigned)guess < (unsigned)a.vocab && guess / DV_CHUNK == c, apart = has && !a.draft;
    float m = -__builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int e = 0; e < N; e++) m = fmaxf(m, x[i][e]);
    m = wave_max(m);
    if (lane == 0) ms[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) m = fmaxf(m, ms[w]);
    int first = 0x7FFFFFFF;
    double sum = 0., but = 0.;   // of all; of all but the guess, which the draw takes (not a difference: it may be nearly all)
    if (!(k > 0.)) {
#pragma unroll
        for (int i = R - 1; i >= 0; i--)
#pragma unroll
            for (int e = N - 1; e >= 0; e--)
                if (x[i][e] == m) first = v0 + i * THREADS * N + e;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d));
    } else if (m > -__builtin_huge_valf()) {
        const DvLaw law = dv_law(m, k);
        if (apart || law.all()) {   // uniform
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const double w = dv_weight(law, x[i][e]);
                    sum += w;
                    but += v0 + i * THREADS * N + e == guess ? 0. : w;
                }
            but = group_sum<64>(but);
        } else if (law.k > 0.) {
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int e = 0; e < N; e++) sum += dv_weight<true>(law, x[i][e]);
        } else {
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int e = 0; e < N; e++) sum += x[i][e] == m ? 1. : 0.;
        }
        sum = group_sum<64>(sum);
    }
    if (lane == 0) {
        sums[wave] = sum;
        buts[wave] = but;
        at[wave] = first;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = but = 0.;
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) {
            sum += sums[w];
            but += buts[w];
            first = min(first, at[w]);
        }
        rec[((long long)which * a.n_rows + r) * a.chunks + c] = {m, first, sum};
        if (apart) others[r] = but;
    }
    // the guess's logit, for the choice
    if (threadIdx.x == 64 && has) drafted[(long long)which * a.n_rows + r] = (float)row[guess];
}

// A row's records as one, by a wave; mine: the lane's first (lane below chunks).
__device__ __forceinline__ DvRow dv_row(const DvRec *rec, const DvRec &mine, int chunks, double k) {
    const int lane = threadIdx.x & 63;
    float m = mine.m;
    for (int c = lane + 64; c < chunks; c += 64) m = fmaxf(m, rec[c].m);
    m = wave_max(m);
    const DvLaw law = dv_law(m, k);
    int at = 0x7FFFFFFF;
    double sum = 0.;
    for (int c = lane; c < chunks; c += 64) {
        const DvRec x = c == lane ? mine : rec[c];
        if (k > 0.) sum += x.sum * dv_weight(law, x.m);
        else if (x.m == m) at = min(at, x.at);
    }
    if (k > 0.) return {m, -1, group_sum<64>(sum)};
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
    return r.sum > 0. ? dv_weight(dv_law(r.m, k), l) / r.sum : 0.;
}
// By a whole workgroup of WAVES waves, a row a wave at a time (n 0: no rows).
template <int WAVES>
__device__ __forceinline__ DvChoice dv_choose(const SvVerify &a, const DvRec *rec, const float *drafted, int s) {
    __shared__ DvRow lp[WAVES], lq[WAVES];
    __shared__ int stays[WAVES];
    int q0, n;
    if (!dv_rows(a, s, &q0, &n)) return {0, 0, -1, 0, {}, {}, 0., 0};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double k = dv_rate(a, s);
    for (int i0 = 0;; i0 += WAVES) {   // uniform
        const int r = q0 + i0 + wave;
        const bool judges = i0 + wave + 1 < n;
        if (i0 + wave < n) {
            const int x = judges ? a.tokens[r + 1] : -1;
            const bool is = (unsigned)x < (unsigned)a.vocab;
            const float u = judges ? a.u_accept[r] : 0.f, lx = is ? drafted[r] : 0.f;
            const float ly = is && a.draft ? drafted[a.n_rows + r] : 0.f;
            const DvRec *rp = rec + (long long)r * a.chunks, *rq = rec + (long long)(a.n_rows + r) * a.chunks;
            const DvRec none = {-__builtin_huge_valf(), 0x7FFFFFFF, 0.};
            const DvRec mp = lane < a.chunks ? rp[lane] : none, mq = lane < a.chunks && judges && a.draft ? rq[lane] : none;
            const DvRow p = dv_row(rp, mp, a.chunks, k);
            DvRow q = {0.f, -1, 0.};
            double qx = 1.;
            if (judges && a.draft) {
                q = dv_row(rq, mq, a.chunks, k);
                qx = dv_prob(q, ly, x, k);
            }
            if (lane == 0) {
                lp[wave] = p;
                lq[wave] = q;
                stays[wave] = is && dv_random(u) * qx < dv_prob(p, lx, x, k);
            }
        } else if (lane == 0) stays[wave] = 1;
        __syncthreads();
        // the first row that does not stay (the last row of a sequence never does)
        const uint64_t ends = __builtin_amdgcn_ballot_w64(lane < WAVES && !stays[lane % WAVES]);
        if (ends) {   // uniform
            const int w = __builtin_ctzll(ends);
            const int row = q0 + i0 + w, rest = i0 + w + 1 < n;
            return {i0 + w, n, rest ? a.tokens[row + 1] : -1, row, lp[w], lq[w], k, rest};
        }
        __syncthreads();
    }
}

// The weight of token v in max(p - q, 0), or in p; pi, qi: 1 / the rows' sums (0: no weight).
__device__ __forceinline__ double dv_rest(const DvChoice &c, const DvLaw &p, const DvLaw &q, double pi, double qi, bool draft,
                                          float l, float d, int v) {
    const double w = dv_weight(p, l) * pi;
    if (!c.rest) return w;
    if (!draft) return v == c.x ? 0. : w;
    return fmax(w - dv_weight(q, d) * qi, 0.);
}

// With a draft model: what each sequence comes to (n 0: no rows), by a workgroup each.
__global__ __launch_bounds__(DV_CHOOSE) void k_dv_choose(const SvVerify a, const DvRec *__restrict__ rec,
                                                       const float *__restrict__ drafted, DvChoice *__restrict__ choice) {
    const DvChoice c = dv_choose<DV_CHOOSE / 64>(a, rec, drafted, blockIdx.x);
    if (threadIdx.x == 0) choice[blockIdx.x] = c;
}

// And the sums of its weights a chunk.  x: chunk, sequence.
template <typename T>
__global__ __launch_bounds__(DV_THREADS) void k_dv_rest(const SvVerify a, const DvChoice *__restrict__ choice,
                                                        double *__restrict__ rest) {
    constexpr int N = 16 / sizeof(T), R = DV_CHUNK / DV_THREADS / N;
    __shared__ double sums[DV_THREADS / 64];
    const int ck = blockIdx.x % a.chunks, s = blockIdx.x / a.chunks;
    const DvChoice c = choice[s];
    if (!c.rest || !(c.k > 0.) || !(c.p.sum > 0.)) return;   // the draw does without
    const T *l = (const T *)a.logits + c.row * a.stride, *d = (const T *)a.draft + c.row * a.dstride;
    const int v0 = ck * DV_CHUNK + (int)threadIdx.x * N;
    float x[R][N], y[R][N];
#pragma unroll
    for (int i = 0; i < R; i++) {
        dv_load(l, v0 + i * DV_THREADS * N, a.vocab, x[i]);
        dv_load(d, v0 + i * DV_THREADS * N, a.vocab, y[i]);
    }
    const double pi = 1. / c.p.sum, qi = c.q.sum > 0. ? 1. / c.q.sum : 0.;
    const DvLaw p = dv_law(c.p.m, c.k), q = dv_law(c.q.m, c.k);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int e = 0; e < N; e++) sum += dv_rest(c, p, q, pi, qi, true, x[i][e], y[i][e], 0);
    sum = group_sum<64>(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.;
#pragma unroll
        for (int w = 0; w < DV_THREADS / 64; w++) sum += sums[w];
        rest[(long long)s * a.chunks + ck] = sum;
    }
}

// Inclusive sum over the workgroup of WAVES waves, and the whole one; lds: of this call only.
template <int WAVES>
__device__ __forceinline__ double dv_scan(double v, double *lds, double *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    double before = 0., all = 0.;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        if (w == wave) before = all;
        all += lds[w];
    }
    *total = all;
    return before + v;
}
// The first thread that says yes (LAST: the last one): its value (and x); -1 where none does.  lds: of this call only,
// and of one with LAST behind it.
template <int WAVES>
struct DvWho {
    int v[WAVES];
    double x[WAVES];
};
template <int WAVES, bool LAST>
__device__ __forceinline__ int dv_which(bool yes, int v, double x, DvWho<WAVES> *lds, double *out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t b = __builtin_amdgcn_ballot_w64(yes);
    const int l = b ? LAST ? 63 - __builtin_clzll(b) : __builtin_ctzll(b) : 0;
    if (LAST) __syncthreads();
    if (lane == l) {
        lds->v[wave] = b ? v : -1;
        lds->x[wave] = x;
    }
    __syncthreads();
    const int found = lds->v[lane % WAVES];
    const uint64_t w = __builtin_amdgcn_ballot_w64(lane < WAVES && found >= 0);
    if (!w) return -1;   // uniform
    const int at = LAST ? 63 - __builtin_clzll(w) : __builtin_ctzll(w);
    *out = lds->x[at];
    return __builtin_amdgcn_readlane(found, at);
}

// The draw, a workgroup a sequence: a chain of records, the scan of the chunks, one chunk's logits and
// the scan of its weights (5 rows of 151936, the choice within: 6.6 us; with sums by shuffles and the
// guess's chunk formed again 9.4).
template <typename T>
__global__ __launch_bounds__(DV_PICK) void k_dv_pick(const SvVerify a, const DvRec *__restrict__ rec,
                                                     const float *__restrict__ drafted,
                                                     const DvChoice *__restrict__ choice, const double *__restrict__ rest,
                                                     const double *__restrict__ others) {
    constexpr int EACH = DV_CHUNK / DV_PICK, WAVES = DV_PICK / 64;
    __shared__ double red[3][WAVES];
    __shared__ DvWho<WAVES> who[2];
    const int s = blockIdx.x, tid = threadIdx.x;
    DvChoice c = choice ? choice[s] : dv_choose<WAVES>(a, rec, drafted, s);
    const bool is = c.n > 0;
    int next = -1;
    if (is && !(c.k > 0.)) {
        if (c.p.m > -__builtin_huge_valf()) next = c.p.at;
    } else if (is && c.p.sum > 0.) {
        const T *l = (const T *)a.logits + c.row * a.stride;
        const T *d = a.draft ? (const T *)a.draft + c.row * a.dstride : nullptr;
        const double u = dv_random(a.u_next[s]), pi = 1. / c.p.sum, qi = c.q.sum > 0. ? 1. / c.q.sum : 0.;
        const DvLaw p = dv_law(c.p.m, c.k), q = dv_law(c.q.m, c.k);
        double w[EACH];
        // the weights of a chunk's elements, EACH side by side a thread, and their sum
        auto weights = [&](int ck) {
            const int v0 = ck * DV_CHUNK + tid * EACH;
            double sum = 0.;
            float x[EACH], y[EACH];
            dv_load(l, v0, a.vocab, x);
            if (d && c.rest) dv_load(d, v0, a.vocab, y);
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                w[e] = dv_rest(c, p, q, pi, qi, d != nullptr, x[e], y[e], v0 + e);
                sum += w[e];
            }
            return sum;
        };
        // a chunk's sum: as the record has it, or k_dv_rest, or (the rejected guess's own chunk) without the guess
        const int own = c.rest && !d && (unsigned)c.x < (unsigned)a.vocab ? c.x / DV_CHUNK : -1;
        const double but = own >= 0 ? others[c.row] : 0.;
        double total = 0.;
        auto mass = [&](int k) {
            if (c.rest && d) return rest[(long long)s * a.chunks + k];
            const DvRec r = rec[(long long)c.row * a.chunks + k];
            return (c.rest && k == own ? but : r.sum) * dv_weight(p, r.m) * pi;
        };
        // a thread's chunks lie side by side
        const int per = (a.chunks + DV_PICK - 1) / DV_PICK, k0 = min(tid * per, a.chunks), k1 = min(k0 + per, a.chunks);
        double run = 0., mine = 0.;
        for (int round = 0; round < 2; round++) {   // (nothing left of p - q: p itself)
            mine = 0.;
            for (int k = k0; k < k1; k++) mine += mass(k);
            run = dv_scan<WAVES>(mine, red[round], &total) - mine;
            if (total > 0.) break;
            c.rest = 0;
        }
        // the first chunk whose end is above u * total; the last that has any weight, where rounding
        // leaves none
        double at = 0., end = 0., before = 0.;
        int f = -1, z = -1;
        for (int k = k0; k < k1; k++) {
            const double m = per == 1 ? mine : mass(k);
            if (m > 0. && run + m > u * total && f < 0) {
                f = k;
                at = run;
            }
            if (m > 0.) {
                z = k;
                end = run;
            }
            run += m;
        }
        int ck = dv_which<WAVES, false>(f >= 0, f, at, &who[0], &before);
        if (ck < 0) ck = dv_which<WAVES, true>(z >= 0, z, end, &who[0], &before);
        if (ck >= 0) {
            mine = weights(ck);
            double all;
            run = before + (dv_scan<WAVES>(mine, red[2], &all) - mine);
            f = z = -1;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                run += w[e];
                if (w[e] > 0.) {
                    z = e;
                    if (run > u * total && f < 0) f = e;
                }
            }
            const int v0 = ck * DV_CHUNK + tid * EACH;
            next = dv_which<WAVES, false>(f >= 0, v0 + f, 0., &who[1], &before);
            if (next < 0) next = dv_which<WAVES, true>(z >= 0, v0 + z, 0., &who[1], &before);
        }
    }
    if (tid == 0) {
        a.n_accept[s] = is ? c.kept : 0;
        a.next[s] = (unsigned)next < (unsigned)a.vocab ? next : -1;   // (falling starts: whatever the records hold)
        if (a.n_drop) a.n_drop[s] = is ? c.n - 1 - c.kept : 0;
    }
}

// Records, choices and sums of the rest a chunk or (no draft model) of a chunk without the guess, the drafts' logits.
struct DvWs {
    DvRec *rec;
    DvChoice *choice;
    double *rest, *others;
    float *drafted;
    size_t bytes;
};
static DvWs verify_ws(void *ws, int n_seqs, int n_rows, int vocab, bool draft) {
    const size_t chunks = ((size_t)vocab + DV_CHUNK - 1) / DV_CHUNK;
    const size_t rows = (size_t)n_rows * (draft ? 2 : 1);
    DvWs w{};
    w.rec = (DvRec *)ws;
    size_t at = rows * chunks * sizeof(DvRec);
    if (draft) {
        w.choice = (DvChoice *)((char *)ws + at);
        at += (size_t)n_seqs * sizeof(DvChoice);
        w.rest = (double *)((char *)ws + at);
        at += (size_t)n_seqs * chunks * sizeof(double);
    } else {
        w.others = (double *)((char *)ws + at);
        at += (size_t)n_rows * sizeof(double);
    }
    w.drafted = (float *)((char *)ws + at);
    w.bytes = at + rows * sizeof(float);
    return w;
}
size_t verify_workspace_bytes(int n_seqs, int n_rows, int vocab, bool draft) {
    return verify_ws(nullptr, n_seqs, n_rows, vocab, draft).bytes;
}

template <typename T>
static hipError_t verify(const SvVerify &a, void *ws, hipStream_t st) {
    const long long wgs = (long long)a.n_rows * (a.draft ? 2 : 1) * a.chunks;
    if (wgs > (1ll << 32) / DV_THREADS - 1 || (long long)a.n_seqs * a.chunks > (1ll << 32) / DV_THREADS - 1)
        return hipErrorInvalidConfiguration;
    const DvWs w = verify_ws(ws, a.n_seqs, a.n_rows, a.vocab, a.draft != nullptr);
    // Many chunks: 32 logits a thread, for fewer instructions a logit (218 + 154 rows of 151936, fp32, with weights of degree 8:
    // 59 -> 53.5 us; 64 logits 55).  Few are spread further (5 rows 4.4 us, in 32 logits 5.3).
    if (wgs >= DV_MANY)
        hipLaunchKernelGGL((k_dv_stats<T, DV_WIDE>), dim3((unsigned)wgs), dim3(DV_WIDE), 0, st, a, w.rec, w.drafted, w.others);
    else if (wgs > 0)
        hipLaunchKernelGGL((k_dv_stats<T, DV_THREADS>), dim3((unsigned)wgs), dim3(DV_THREADS), 0, st, a, w.rec, w.drafted,
                           w.others);
    if (a.draft) {
        hipLaunchKernelGGL(k_dv_choose, dim3(a.n_seqs), dim3(DV_CHOOSE), 0, st, a, w.rec, w.drafted, w.choice);
        hipLaunchKernelGGL(k_dv_rest<T>, dim3((unsigned)(a.n_seqs * a.chunks)), dim3(DV_THREADS), 0, st, a, w.choice,
                           w.rest);
    }
    hipLaunchKernelGGL(k_dv_pick<T>, dim3(a.n_seqs), dim3(DV_PICK), 0, st, a, w.rec, w.drafted, w.choice, w.rest,
                       w.others);
    return hipGetLastError();
}

hipError_t launch_verify(const SvVerify &a, int type, void *ws, hipStream_t st) {
    return type == TBQ_KV_F32 ? verify<float>(a, ws, st) : type == TBQ_KV_F16 ? verify<pg_f16>(a, ws, st) : verify<pg_bf16>(a, ws, st);
}

}  // namespace tbq
