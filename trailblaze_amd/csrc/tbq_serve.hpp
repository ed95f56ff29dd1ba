// tbq_serve.hpp -- what a serving step keeps on the device beside the cache
// (include/tbq_kv.h): page tables from request lengths, and the verification of
// drafted tokens.  Internal to libtbq.
#pragma once

#include "tbq_paged.hpp"

namespace tbq {

struct SvTables {
    tbq_kv_tables t;
    int shift;   // log2 of the page size
};
hipError_t launch_tables(const SvTables &a, hipStream_t st);

struct SvVerify {
    int n_seqs, n_rows, vocab, chunks;   // chunks of a row of logits
    const int *q_start, *tokens;
    const void *logits, *draft;          // [n_rows][vocab], rows apart by stride, dstride elements; draft may be null
    long long stride, dstride;
    const float *temperature, *u_accept, *u_next;
    int *n_accept, *next, *n_drop;
};
// Elements of a row that a workgroup takes at a time.  (Calls, on one card: 218 + 154 rows of 151936, fp32, 93 us in 8192,
// 85 in 4096, 91 in 2048; 146 + 113 rows of 50257, bf16, 38.6, 33.5 and 31.4; 5 rows of 151936 14.6, 13 and 12.)
constexpr int DV_CHUNK = 4096;
size_t verify_workspace_bytes(int n_seqs, int n_rows, int vocab, bool draft);
hipError_t launch_verify(const SvVerify &a, int type, void *ws, hipStream_t st);

}  // namespace tbq
