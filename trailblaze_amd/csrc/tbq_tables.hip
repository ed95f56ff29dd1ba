// tbq_tables.hip -- a step's page tables, slots and positions from request lengths
// (include/tbq_kv.h, tbq_kv_build_tables) on gfx950.
//
// All of it is prefix sums over the sequences: of the pages that go back to the
// free list, of the pages that are taken from its end, of the new tokens.  One
// workgroup forms them, 1024 sequences at a time, and moves the pages (whose number
// is small beside the tables); a launch over tokens and table entries follows.
// Bound by the first one's chain of dependent loads and barriers: lengths, pages that go
// back, the list's end (64 sequences of 8000 positions: 4.0 + 2.5 us; 1000 of 6000, 30
// prompts among them: 6.7 + 4).  LDS is what the 16 waves of one workgroup wait for: with
// wave sums that every thread adds for itself and searches in waves without an entry,
// 6.0 and 10.6 in the first launch; with a scan each for pages given, pages taken and tokens
// 11 and 20 in all.
#include <type_traits>

#include "tbq_kernels.h"
#include "tbq_serve.hpp"

namespace tbq {

constexpr int TB_THREADS = 1024, TB_WAVES = TB_THREADS / 64, TB_EACH = 4;   // most entries of a thread at a time
struct TbLds {
    int3 wave[2][TB_WAVES];                   // sums of the waves' sequences (by turns)
    int count[2][TB_EACH * TB_WAVES];
    int3 fail[TB_WAVES];                      // a wave's first sequence that is not served, pages taken and tokens before it
    // of a chunk's sequences, inclusive sums of the entries that each gives back and takes, and its first entry less
    // those before it
    int given[TB_THREADS], give[TB_THREADS], taken[TB_THREADS], take[TB_THREADS];
};

constexpr int TB_MOST = 1 << 30;   // tokens of a call; sums of them stop behind it
__device__ __forceinline__ int3 tb_add(int3 a, int3 b) {
    return make_int3(a.x + b.x, a.y + b.y, (int)min((unsigned)a.z + (unsigned)b.z, (unsigned)TB_MOST + 1u));
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int tb_dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int3 tb_dpp(int3 v) {
    return make_int3(tb_dpp<CTRL, ROWS>(v.x), tb_dpp<CTRL, ROWS>(v.y), tb_dpp<CTRL, ROWS>(v.z));
}
__device__ __forceinline__ int tb_add(int a, int b) { return a + b; }
__device__ __forceinline__ int tb_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ int3 tb_lane(int3 v, int l) { return make_int3(tb_lane(v.x, l), tb_lane(v.y, l), tb_lane(v.z, l)); }
// Inclusive sums over rows of 16 lanes; over the wave.
template <typename T>
__device__ __forceinline__ T tb_row_scan(T v) {
    v = tb_add(v, tb_dpp<0x111>(v));   // row_shr 1, 2, 4, 8
    v = tb_add(v, tb_dpp<0x112>(v));
    v = tb_add(v, tb_dpp<0x114>(v));
    return tb_add(v, tb_dpp<0x118>(v));
}
template <typename T>
__device__ __forceinline__ T tb_wave_scan(T v) {
    v = tb_row_scan(v);
    v = tb_add(v, tb_dpp<0x142, 0xA>(v));   // row_bcast 15, 31
    return tb_add(v, tb_dpp<0x143, 0xC>(v));
}
// Sums over the workgroup, in front of each thread, of pages given, pages taken (below 2^31: a table has no more
// entries) and tokens; and the whole ones.  One barrier; turn: 0 and 1 by turns.
__device__ __forceinline__ int3 tb_scan(int3 own, TbLds *lds, int turn, int3 *total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int3 v = tb_wave_scan(own), before = tb_dpp<0x138>(v);   // wave_shr 1
    if (lane == 63) lds->wave[turn][wave] = v;
    __syncthreads();
    const int3 w = tb_row_scan(lds->wave[turn][lane % TB_WAVES]);
    *total = tb_lane(w, TB_WAVES - 1);
    return wave ? tb_add(tb_lane(w, wave - 1), before) : before;
}
// How many yeses there are before each of the threads' N, the threads' first ones coming first; and how many in all.
template <int N>
__device__ __forceinline__ void tb_count(const bool (&yes)[N], TbLds *lds, int turn, int (&before)[N], int *total) {
    static_assert(N * TB_WAVES <= 64, "a lane a count");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint64_t b = __builtin_amdgcn_ballot_w64(yes[i]);
        before[i] = __builtin_popcountll(b & ((1ull << lane) - 1));
        if (lane == 0) lds->count[turn][TB_WAVES * i + wave] = __builtin_popcountll(b);
    }
    __syncthreads();
    const int own = lds->count[turn][lane % (N * TB_WAVES)], sum = N == 1 ? tb_row_scan(own) : tb_wave_scan(own);
    *total = tb_lane(sum, N * TB_WAVES - 1);
#pragma unroll
    for (int i = 0; i < N; i++) before[i] += tb_lane(sum - own, TB_WAVES * i + wave);
}

// The sequences (of n, 1 to 1024) that the entries j belong to: the first whose end is above j, which there is.
template <int N>
__device__ __forceinline__ void tb_find(const int *end, int n, const int (&j)[N], int (&at)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) at[i] = 0;
    for (int step = 512; step; step >>= 1) {
        if (step >= n) continue;   // uniform
#pragma unroll
        for (int i = 0; i < N; i++)
            if (end[min(at[i] + step, n) - 1] <= j[i]) at[i] += step;
    }
}

// Sequence s before the call: positions kept, pages of them and of all, new tokens; the pages it needs
// then (-1: more than the table has).
struct TbSeq {
    int base, held, kept, add, need;
};
__device__ __forceinline__ TbSeq tb_seq(const SvTables &a, int s, bool there) {
    if (!there) return {0, 0, 0, 0, 0};
    const int round = (1 << a.shift) - 1, room = a.t.max_pages << a.shift;
    const int len = min(max(a.t.kv_len[s], 0), room);
    const int drop = a.t.n_drop ? min(max(a.t.n_drop[s], 0), len) : 0, add = max(a.t.n_new[s], 0), base = len - drop;
    return {base, (len + round) >> a.shift, (base + round) >> a.shift, min(add, TB_MOST + 1),
            add > room - base ? -1 : (base + add + round) >> a.shift};
}
__device__ __forceinline__ int3 tb_sums(const TbSeq &q) {
    return make_int3(q.held - q.kept, q.need < 0 ? 0 : q.need - q.kept, q.add);
}

__global__ __launch_bounds__(TB_THREADS) void k_tables_plan(const SvTables a) {
    __shared__ TbLds lds;
    const tbq_kv_tables &t = a.t;
    const int tid = threadIdx.x, lane = tid & 63, listed = min(max(t.n_free[0], 0), t.n_pages);
    TbSeq q{};
    int3 own{}, sum{}, all{};   // the sequence's, those before it, the chunk's
    int turn = 0;
    // a chunk's sequences and where their entries begin
    auto chunk = [&](int s0, int n) {
        q = tb_seq(a, s0 + tid, tid < n);
        own = tb_sums(q);
        sum = tb_scan(own, &lds, turn ^= 1, &all);
        lds.given[tid] = sum.x + own.x;
        lds.give[tid] = q.kept - sum.x;
        lds.taken[tid] = sum.y + own.y;
        lds.take[tid] = q.kept - sum.y;
        __syncthreads();
    };
    // n entries: one a thread, or TB_EACH while there are more than threads
    auto rounds = [&](int n, auto f) {
        int j0 = 0;
        for (; n - j0 > TB_THREADS; j0 += TB_EACH * TB_THREADS) f(j0, std::integral_constant<int, TB_EACH>{});
        if (j0 < n) f(j0, std::integral_constant<int, 1>{});
    };
    // pages behind the last kept position go to the list, in the sequences' order
    int have = listed;
    for (int s0 = 0; s0 < t.n_seqs; s0 += TB_THREADS) {
        const int n = min(TB_THREADS, t.n_seqs - s0);
        chunk(s0, n);
        rounds(all.x, [&](int j0, auto each) {
            constexpr int N = decltype(each)::value;
            int j[N], i[N], page[N], before[N], count;
            bool is[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                j[e] = min(j0 + e * TB_THREADS + tid, all.x - 1);
                page[e] = -1;
            }
            if (j0 + (tid & ~63) < all.x) {   // the wave has some
                tb_find(lds.given, n, j, i);
#pragma unroll
                for (int e = 0; e < N; e++)
                    page[e] = t.page_table[(long long)(s0 + i[e]) * t.max_pages + lds.give[i[e]] + j[e]];
            }
#pragma unroll
            for (int e = 0; e < N; e++)
                is[e] = j0 + e * TB_THREADS + tid < all.x && (unsigned)page[e] < (unsigned)t.n_pages;
            tb_count(is, &lds, turn ^= 1, before, &count);
#pragma unroll
            for (int e = 0; e < N; e++)
                if (is[e] && have + before[e] < t.n_pages) t.free_out[have + before[e]] = page[e];
            have = min(have + count, t.n_pages);
        });
        if (t.n_seqs > TB_THREADS) __syncthreads();   // the sums are rewritten
    }
    __threadfence_block();
    // then sequences take pages from its end, until one does not get what it needs
    int taken = 0, rows = 0, served = 0;
    bool going = true;
    for (int s0 = 0; s0 < t.n_seqs; s0 += TB_THREADS) {
        const int n = min(TB_THREADS, t.n_seqs - s0);
        if (t.n_seqs > TB_THREADS) chunk(s0, n);
        const bool fails = tid < n && (!going || q.need < 0 || sum.y + own.y > have - taken || tb_add(sum, own).z > t.n_tokens - rows);
        const uint64_t b = __builtin_amdgcn_ballot_w64(fails);
        if (lane == (b ? __builtin_ctzll(b) : 0)) lds.fail[tid >> 6] = b ? make_int3(tid, sum.y, sum.z) : make_int3(n, 0, 0);
        __syncthreads();
        const int3 f = lds.fail[lane % TB_WAVES];
        const uint64_t w = __builtin_amdgcn_ballot_w64(f.x < n);
        const int3 first = tb_lane(f, w ? __builtin_ctzll(w) : 0);   // (a wave's fails are behind those of the waves before)
        const int fail = w ? first.x : n, all_take = w ? first.y : all.y, all_rows = w ? first.z : all.z;
        if (tid < n) {
            t.kv_len_out[s0 + tid] = q.base + (tid < fail ? q.add : 0);
            t.q_start[s0 + tid + 1] = rows + (tid < fail ? sum.z + own.z : all_rows);
        }
        rounds(all_take, [&](int j0, auto each) {
            constexpr int N = decltype(each)::value;
            if (j0 + (tid & ~63) >= all_take) return;   // the wave has none
            int j[N], i[N], page[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                j[e] = min(j0 + e * TB_THREADS + tid, all_take - 1);
                const int at = have - 1 - taken - j[e];
                page[e] = *(at < listed ? t.free_pages + at : t.free_out + at);
            }
            tb_find(lds.taken, n, j, i);
#pragma unroll
            for (int e = 0; e < N; e++)
                if (j0 + e * TB_THREADS + tid < all_take)
                    t.page_table_out[(long long)(s0 + i[e]) * t.max_pages + lds.take[i[e]] + j[e]] = page[e];
        });
        taken += all_take;
        rows += all_rows;
        served += fail;
        going = going && fail == n;
        if (t.n_seqs > TB_THREADS) __syncthreads();   // the sums are rewritten
    }
    if (tid == 0) {
        t.q_start[0] = 0;
        t.n_free_out[0] = have - taken;
        if (t.served) t.served[0] = served;
    }
}

// Workgroups of 256: those of the tokens, those of the list, then max_pages / 1024 a
// sequence.
constexpr int TF_THREADS = 256, TF_ENTRIES = 4;
__global__ __launch_bounds__(TF_THREADS) void k_tables_fill(const SvTables a, int token_wgs, int list_wgs,
                                                           int per_seq) {
    const tbq_kv_tables &t = a.t;
    const int round = (1 << a.shift) - 1;
    if ((int)blockIdx.x >= token_wgs + list_wgs) {
        const int x = blockIdx.x - token_wgs - list_wgs, s = x / per_seq;
        const int len = t.kv_len_out[s], base = len - (t.q_start[s + 1] - t.q_start[s]);
        const int kept = (base + round) >> a.shift, need = (len + round) >> a.shift;
        const int *in = t.page_table + (long long)s * t.max_pages;
        int *out = t.page_table_out + (long long)s * t.max_pages;
#pragma unroll
        for (int i = 0; i < TF_ENTRIES; i++) {
            const int e = (x % per_seq * TF_ENTRIES + i) * TF_THREADS + threadIdx.x;
            if (e >= t.max_pages) break;
            if (e >= need) out[e] = -1;
            else if (e < kept && out != in) out[e] = in[e];
        }
        return;
    }
    if ((int)blockIdx.x >= token_wgs) {   // the list: what is left of it, -1 behind
        const bool copy = t.free_out != t.free_pages;
        const int left = t.n_free_out[0], listed = copy ? t.n_free[0] : 0;
#pragma unroll
        for (int i = 0; i < TF_ENTRIES; i++) {
            const int e = ((blockIdx.x - token_wgs) * TF_ENTRIES + i) * TF_THREADS + threadIdx.x;
            if (e >= t.n_pages) break;
            if (e >= left) t.free_out[e] = -1;
            else if (copy && e < listed) t.free_out[e] = t.free_pages[e];
        }
        return;
    }
    const int t0 = blockIdx.x * TF_THREADS, row = t0 + threadIdx.x;
    int lo = pg_seq_of(t.q_start, t.n_seqs, t0), hi = pg_seq_of(t.q_start, t.n_seqs, t0 + TF_THREADS - 1);
    if (row >= t.n_tokens) return;
    while (lo < hi) {   // the number of sequences that end at or before the row
        const int mid = (lo + hi) >> 1;
        if (t.q_start[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    int pos = -1, slot = -1;
    if (lo < t.n_seqs) {
        const int len = t.kv_len_out[lo], base = len - (t.q_start[lo + 1] - t.q_start[lo]);
        pos = base + row - t.q_start[lo];
        const int e = pos >> a.shift;
        const int page = (e < (base + round) >> a.shift ? t.page_table : t.page_table_out)[(long long)lo * t.max_pages + e];
        slot = (unsigned)page < (unsigned)t.n_pages ? page << a.shift | (pos & round) : -1;
    }
    if (t.positions) t.positions[row] = pos;
    if (t.slots) t.slots[row] = slot;
}

hipError_t launch_tables(const SvTables &a, hipStream_t st) {
    hipLaunchKernelGGL(k_tables_plan, dim3(1), dim3(TB_THREADS), 0, st, a);
    const int token_wgs = a.t.slots || a.t.positions ? (a.t.n_tokens + TF_THREADS - 1) / TF_THREADS : 0;
    const int each = TF_THREADS * TF_ENTRIES, list_wgs = (a.t.n_pages + each - 1) / each;
    const int per_seq = (a.t.max_pages + each - 1) / each;
    const long long wgs = token_wgs + list_wgs + (long long)a.t.n_seqs * per_seq;
    if (wgs > (1ll << 32) / TF_THREADS - 1) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(k_tables_fill, dim3((unsigned)wgs), dim3(TF_THREADS), 0, st, a, token_wgs, list_wgs, per_seq);
    return hipGetLastError();
}

}  // namespace tbq
