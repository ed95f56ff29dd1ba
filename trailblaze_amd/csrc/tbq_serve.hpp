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
// Elements of a row that a workgroup takes at a time: the longer ones where there are many.
constexpr int DV_SHORT = 2048, DV_LONG = 8192;
int verify_chunk(int n_rows, int vocab, bool draft);
size_t verify_workspace_bytes(int n_seqs, int n_rows, int vocab, bool draft);
hipError_t launch_verify(const SvVerify &a, int type, void *ws, hipStream_t st);

}  // namespace tbq
