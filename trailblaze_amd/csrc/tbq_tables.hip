// tbq_tables.hip -- a step's page tables, slots and positions from request lengths
// (include/tbq_kv.h, tbq_kv_build_tables) on gfx950.
//
// All of it is prefix sums over the sequences: of the pages that go back to the
// free list, of the pages that are taken from its end, of the new tokens.  One
// workgroup forms them, 1024 sequences at a time, and moves the pages (whose number
// is small beside the tables); a launch over tokens and table entries follows.
// Bound by the first one's chain of dependent loads: lengths, pages that go back, the
// list's end (64 sequences of 8000 positions: 6.0 + 2.5 us; 1000 of 6000, 30 prompts among
// them: 10.6 + 4.  A scan each for pages given, pages taken and tokens, instead of one: 11
// and 20 in all.)
#include "tbq_kernels.h"
#include "tbq_serve.hpp"

namespace tbq {

constexpr int TB_THREADS = 1024, TB_WAVES = TB_THREADS / 64;
struct TbLds {
    int3 wave[2][TB_WAVES];                   // sums of the waves' sequences (by turns)
    int count[2][TB_WAVES];
    int end[TB_THREADS], first[TB_THREADS];   // inclusive sums of a chunk's entries; each sequence's first entry
    int fail, take, tokens;
};

constexpr int TB_MOST = 1 << 30;   // tokens of a call; sums of them stop behind it
__device__ __forceinline__ int3 tb_add(int3 a, int3 b) {
    return make_int3(a.x + b.x, a.y + b.y, (int)min((unsigned)a.z + (unsigned)b.z, (unsigned)TB_MOST + 1u));
}
// Inclusive sums over the workgroup of pages given, pages taken (below 2^31: a table has no more entries)
// and tokens; and the whole ones.  One barrier; turn: 0 and 1 by turns.
__device__ __forceinline__ int3 tb_scan(int3 v, TbLds *lds, int turn, int3 *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int3 o = make_int3(__shfl_up(v.x, d), __shfl_up(v.y, d), __shfl_up(v.z, d));
        if (lane >= d) v = tb_add(v, o);
    }
    if (lane == 63) lds->wave[turn][wave] = v;
    __syncthreads();
    int3 before = make_int3(0, 0, 0), all = before;
#pragma unroll
    for (int w = 0; w < TB_WAVES; w++) {
        if (w == wave) before = all;
        all = tb_add(all, lds->wave[turn][w]);
    }
    *total = all;
    return tb_add(before, v);
}
// How many threads up to this one say yes, and how many do.
__device__ __forceinline__ int tb_count(bool yes, TbLds *lds, int turn, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t b = __builtin_amdgcn_ballot_w64(yes);
    if (lane == 0) lds->count[turn][wave] = __builtin_popcountll(b);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < TB_WAVES; w++) {
        if (w == wave) before = all;
        all += lds->count[turn][w];
    }
    *total = all;
    return before + __builtin_popcountll(b & (lane == 63 ? ~0ull : (2ull << lane) - 1));
}

// The sequence of a chunk that entry j belongs to: the first whose end is above j.
__device__ __forceinline__ int tb_find(const TbLds *lds, int n, int j) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (lds->end[mid] > j) hi = mid;
        else lo = mid + 1;
    }
    return lo;
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
    const int tid = threadIdx.x, listed = min(max(t.n_free[0], 0), t.n_pages);
    TbSeq q{};
    int3 sum{}, all{};
    // pages behind the last kept position go to the list, in the sequences' order
    int have = listed, turn = 0;
    for (int s0 = 0; s0 < t.n_seqs; s0 += TB_THREADS) {
        const int n = min(TB_THREADS, t.n_seqs - s0);
        q = tb_seq(a, s0 + tid, tid < n);
        sum = tb_scan(tb_sums(q), &lds, turn ^= 1, &all);
        if (all.x == 0) continue;   // uniform
        lds.end[tid] = sum.x;
        lds.first[tid] = q.kept - (sum.x - (q.held - q.kept));
        __syncthreads();
        for (int j0 = 0; j0 < all.x; j0 += TB_THREADS) {
            const int j = j0 + tid;
            int page = -1, count;
            if (j < all.x) {
                const int i = tb_find(&lds, n, j);
                page = t.page_table[(long long)(s0 + i) * t.max_pages + lds.first[i] + j];
            }
            const bool is = (unsigned)page < (unsigned)t.n_pages;
            const int at = have + tb_count(is, &lds, turn ^= 1, &count) - 1;
            if (is && at < t.n_pages) t.free_out[at] = page;
            have = min(have + count, t.n_pages);
        }
    }
    __threadfence_block();
    // then sequences take pages from its end, until one does not get what it needs
    long long taken = 0, rows = 0;
    int served = 0;
    bool going = true;
    for (int s0 = 0; s0 < t.n_seqs; s0 += TB_THREADS) {
        const int n = min(TB_THREADS, t.n_seqs - s0);
        if (t.n_seqs > TB_THREADS) {
            q = tb_seq(a, s0 + tid, tid < n);
            sum = tb_scan(tb_sums(q), &lds, turn ^= 1, &all);
        }
        if (tid == 0) lds.fail = n;
        __syncthreads();
        if (tid < n && (!going || q.need < 0 || taken + sum.y > have || rows + sum.z > t.n_tokens)) atomicMin(&lds.fail, tid);
        __syncthreads();
        const int fail = lds.fail, take = q.need < 0 ? 0 : q.need - q.kept;
        if (tid == fail) lds.take = sum.y - take;
        // (the tokens before the first that fails are its predecessor's sum: its own may have stopped)
        if (tid + 1 == fail) lds.tokens = sum.z;
        lds.end[tid] = tid < fail ? sum.y : 0x7FFFFFFF;
        lds.first[tid] = q.kept - (sum.y - take);
        __syncthreads();
        int all_take = all.y, all_rows = all.z;
        if (fail < n) {
            all_take = lds.take;
            all_rows = fail == 0 ? 0 : lds.tokens;
        }
        if (tid < n) {
            t.kv_len_out[s0 + tid] = q.base + (tid < fail ? q.add : 0);
            t.q_start[s0 + tid + 1] = (int)(rows + (tid < fail ? sum.z : all_rows));
        }
        for (int j = tid; j < all_take; j += TB_THREADS) {
            const int i = tb_find(&lds, n, j), at = have - 1 - (int)taken - j;
            t.page_table_out[(long long)(s0 + i) * t.max_pages + lds.first[i] + j] =
                at < listed ? t.free_pages[at] : t.free_out[at];
        }
        taken += all_take;
        rows += all_rows;
        served += fail;
        going = going && fail == n;
    }
    if (tid == 0) {
        t.q_start[0] = 0;
        t.n_free_out[0] = have - (int)taken;
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
