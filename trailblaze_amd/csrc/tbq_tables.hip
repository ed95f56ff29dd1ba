// tbq_tables.hip -- a step's page tables, slots and positions from request lengths
// (include/tbq_kv.h, tbq_kv_build_tables) on gfx950.
//
// All of it is prefix sums over the sequences: of the pages that go back to the
// free list, of the pages that are taken from its end, of the new tokens.  One
// workgroup forms them, 1024 sequences at a time, and moves the pages (whose number
// is small beside the tables); a launch over tokens and table entries follows.
#include "tbq_kernels.h"
#include "tbq_serve.hpp"

namespace tbq {

constexpr int TB_THREADS = 1024;
struct TbLds {
    long long wave[TB_THREADS / 64];
    int end[TB_THREADS], first[TB_THREADS];   // inclusive sums of a chunk's entries; each sequence's first entry
    int fail;
    long long take, tokens;
};

// Inclusive sum over the workgroup, and the whole one.
__device__ __forceinline__ long long tb_scan(long long v, TbLds *lds, long long *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const long long o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) lds->wave[wave] = v;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < TB_THREADS / 64; w++) {
        const long long x = lds->wave[w];
        before += w < wave ? x : 0;
        all += x;
    }
    *total = all;
    return before + v;
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

// Sequence s before the call: positions kept and held, pages of both, new tokens.
struct TbSeq {
    int base, held, kept, add;
};
__device__ __forceinline__ TbSeq tb_seq(const SvTables &a, int s) {
    const int round = (1 << a.shift) - 1, room = a.t.max_pages << a.shift;
    const int len = min(max(a.t.kv_len[s], 0), room);
    const int drop = a.t.n_drop ? min(max(a.t.n_drop[s], 0), len) : 0;
    return {len - drop, (len + round) >> a.shift, (len - drop + round) >> a.shift, max(a.t.n_new[s], 0)};
}

__global__ __launch_bounds__(TB_THREADS) void k_tables_plan(const SvTables a) {
    __shared__ TbLds lds;
    const tbq_kv_tables &t = a.t;
    const int tid = threadIdx.x, listed = min(max(t.n_free[0], 0), t.n_pages);
    long long total;
    // pages behind the last kept position go to the list, in the sequences' order
    int have = listed;
    for (int s0 = 0; s0 < t.n_seqs; s0 += TB_THREADS) {
        const int n = min(TB_THREADS, t.n_seqs - s0);
        const TbSeq q = tid < n ? tb_seq(a, s0 + tid) : TbSeq{0, 0, 0, 0};
        const int end = (int)tb_scan(q.held - q.kept, &lds, &total);   // (sums of entries stay below 2^31: the table has no more)
        lds.end[tid] = end;
        lds.first[tid] = q.kept - (end - (q.held - q.kept));
        __syncthreads();
        const int back = (int)total;
        for (int j0 = 0; j0 < back; j0 += TB_THREADS) {
            const int j = j0 + tid;
            int page = -1;
            if (j < back) {
                const int i = tb_find(&lds, n, j);
                page = t.page_table[(long long)(s0 + i) * t.max_pages + lds.first[i] + j];
            }
            const bool is = (unsigned)page < (unsigned)t.n_pages;
            const int at = have + (int)tb_scan(is, &lds, &total) - 1;
            if (is && at < t.n_pages) t.free_out[at] = page;
            have = min(have + (int)total, t.n_pages);
        }
        __syncthreads();
    }
    __threadfence_block();
    __syncthreads();
    // then sequences take pages from its end, until one does not get what it needs
    long long taken = 0, rows = 0;
    int served = 0;
    bool going = true;
    for (int s0 = 0; s0 < t.n_seqs; s0 += TB_THREADS) {
        const int n = min(TB_THREADS, t.n_seqs - s0);
        const TbSeq q = tid < n ? tb_seq(a, s0 + tid) : TbSeq{0, 0, 0, 0};
        const long long len = (long long)q.base + q.add, need = (len + (1 << a.shift) - 1) >> a.shift;
        const bool fits = need <= t.max_pages;
        const int take = fits ? (int)need - q.kept : 0;
        long long all_take, all_rows;
        const long long end = tb_scan(take, &lds, &all_take), end_rows = tb_scan(q.add, &lds, &all_rows);
        if (tid == 0) lds.fail = n;
        __syncthreads();
        if (tid < n && (!going || !fits || taken + end > have || rows + end_rows > t.n_tokens)) atomicMin(&lds.fail, tid);
        __syncthreads();
        const int fail = lds.fail;
        if (tid == fail) {
            lds.take = end - take;
            lds.tokens = end_rows - q.add;
        }
        lds.end[tid] = tid < fail ? (int)end : 0x7FFFFFFF;
        lds.first[tid] = q.kept - (int)(end - take);
        __syncthreads();
        if (fail < n) {
            all_take = lds.take;
            all_rows = lds.tokens;
        }
        if (tid < n) {
            t.kv_len_out[s0 + tid] = q.base + (tid < fail ? q.add : 0);
            t.q_start[s0 + tid + 1] = (int)(rows + (tid < fail ? end_rows : all_rows));
        }
        for (int j = tid; j < (int)all_take; j += TB_THREADS) {
            const int i = tb_find(&lds, n, j), at = have - 1 - (int)taken - j;
            t.page_table_out[(long long)(s0 + i) * t.max_pages + lds.first[i] + j] = at < listed ? t.free_pages[at] : t.free_out[at];
        }
        taken += all_take;
        rows += all_rows;
        served += fail;
        going = going && fail == n;
        __syncthreads();
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
