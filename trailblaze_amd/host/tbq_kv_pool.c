/*
 * tbq_kv_pool.c -- the page pool of a paged key/value cache (include/tbq_kv.h):
 * how many holders each page has.  Host bookkeeping only; the pages' contents
 * are moved by tbq_kv_copy_pages.
 */
#include <stdlib.h>

#include "../../include/tbq_kv.h"

int tbq_host_fail(const char *msg);   /* tbq_api.hip (hidden): sets tbq_last_error, returns 0 */

struct tbq_kv_pool {
    int n, n_free;
    int low;      /* no page below it is free */
    int *holders;
    int *named;   /* scratch of one call: how often each page is named in it */
};

tbq_kv_pool *tbq_kv_pool_create(int n_pages) {
    if (n_pages < 1) {
        tbq_host_fail("tbq_kv_pool_create: n_pages < 1");
        return NULL;
    }
    tbq_kv_pool *p = calloc(1, sizeof *p);
    if (p) {
        p->holders = calloc((size_t)n_pages, sizeof *p->holders);
        p->named = calloc((size_t)n_pages, sizeof *p->named);
    }
    if (!p || !p->holders || !p->named) {
        tbq_kv_pool_destroy(p);
        tbq_host_fail("tbq_kv_pool_create: out of host memory");
        return NULL;
    }
    p->n = p->n_free = n_pages;
    return p;
}

void tbq_kv_pool_destroy(tbq_kv_pool *p) {
    if (!p) return;
    free(p->holders);
    free(p->named);
    free(p);
}

int tbq_kv_pool_free_pages(const tbq_kv_pool *p) { return p ? p->n_free : 0; }

int tbq_kv_pool_holders(const tbq_kv_pool *p, int page) { return p && page >= 0 && page < p->n ? p->holders[page] : -1; }

int tbq_kv_pool_alloc(tbq_kv_pool *p, int n, int *pages) {
    if (!p || n < 0 || (n > 0 && !pages)) return tbq_host_fail("tbq_kv_pool_alloc: bad argument");
    if (n > p->n_free) return tbq_host_fail("tbq_kv_pool_alloc: not enough free pages");
    int i = p->low;
    for (int got = 0; got < n; i++) {
        if (p->holders[i]) continue;
        p->holders[i] = 1;
        pages[got++] = i;
    }
    if (n > 0) p->low = i;
    p->n_free -= n;
    return 1;
}

/* Whether every page named exists and has at least as many holders as it is
 * named times (spend), or one (share). */
static int nameable(tbq_kv_pool *p, int n, const int *pages, int spend) {
    int i, ok = 1;
    for (i = 0; i < n && ok; i++) {
        ok = pages[i] >= 0 && pages[i] < p->n && p->holders[pages[i]] > (spend ? p->named[pages[i]] : 0);
        if (ok) p->named[pages[i]]++;
    }
    for (int j = 0; j < i; j++)
        if (pages[j] >= 0 && pages[j] < p->n) p->named[pages[j]] = 0;
    return ok;
}

int tbq_kv_pool_share(tbq_kv_pool *p, int n, const int *pages) {
    if (!p || n < 0 || (n > 0 && !pages)) return tbq_host_fail("tbq_kv_pool_share: bad argument");
    if (!nameable(p, n, pages, 0)) return tbq_host_fail("tbq_kv_pool_share: a page is free or not there");
    for (int i = 0; i < n; i++) p->holders[pages[i]]++;
    return 1;
}

int tbq_kv_pool_release(tbq_kv_pool *p, int n, const int *pages) {
    if (!p || n < 0 || (n > 0 && !pages)) return tbq_host_fail("tbq_kv_pool_release: bad argument");
    if (!nameable(p, n, pages, 1)) return tbq_host_fail("tbq_kv_pool_release: a page is free, named too often or not there");
    for (int i = 0; i < n; i++) {
        if (--p->holders[pages[i]]) continue;
        p->n_free++;
        if (pages[i] < p->low) p->low = pages[i];
    }
    return 1;
}

int tbq_kv_pool_fork(tbq_kv_pool *p, int positions, int page_size, const int *pages, int *child, int copy[2]) {
    if (!p || positions < 0 || page_size < 1 || !copy || (positions > 0 && (!pages || !child)))
        return tbq_host_fail("tbq_kv_pool_fork: bad argument");
    const int full = positions / page_size, part = positions % page_size != 0;
    copy[0] = copy[1] = -1;
    if (!nameable(p, full + part, pages, 0)) return tbq_host_fail("tbq_kv_pool_fork: a page is free or not there");
    int fresh = -1;
    if (part && !tbq_kv_pool_alloc(p, 1, &fresh)) return 0;
    for (int i = 0; i < full; i++) {
        p->holders[pages[i]]++;
        child[i] = pages[i];
    }
    if (part) {
        copy[0] = pages[full];
        copy[1] = child[full] = fresh;
    }
    return 1;
}

int tbq_kv_pool_defrag(tbq_kv_pool *p, int max, int *src, int *dst) {
    if (!p || max < 0 || (max > 0 && (!src || !dst))) {
        tbq_host_fail("tbq_kv_pool_defrag: bad argument");
        return -1;
    }
    /* the highest used page into the lowest free one, while that is lower */
    int n = 0, lo = p->low, hi = p->n - 1;
    while (n < max) {
        while (lo < p->n && p->holders[lo]) lo++;
        while (hi >= 0 && !p->holders[hi]) hi--;
        if (lo >= hi) break;
        p->holders[lo] = p->holders[hi];
        p->holders[hi] = 0;
        src[n] = hi--;
        dst[n++] = lo++;
    }
    p->low = lo < p->n ? lo : p->n;
    return n;
}
