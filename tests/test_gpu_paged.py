"""GPU checks of the paged key/value cache's operators (include/tbq_kv.h)
against 64-bit references (paged_ref.py), through the package's entry points.
Pools hold NaN wherever a call has no business to look, so a read of a free
page, of a row behind a sequence or of a masked position shows."""
import math

import numpy as np
import pytest

import trailblaze_amd as tb
from paged_ref import (TYPES, attention, attention_tolerance, frequencies, half_step, least, make_table, page_of, rmsnorm,
                       rotate, tokens)
from trailblaze_amd import paged

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def _init():
    print("device:", tb.init(), flush=True)


def _torch():
    import torch
    return torch


def ints(v):
    torch = _torch()
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(lens):
    return [0] + [int(x) for x in np.cumsum(lens)]


def make_batch(q_lens, kv_len, table, rows=None, **kw):
    st = starts(q_lens)
    return paged.kv_batch(ints(st), ints(kv_len), ints(table), st[-1] if rows is None else rows, **kw)


# ---- append ----------------------------------------------------------------------
def run_append(act, qact, cache, D, NQ, NKV, page, q_lens, past, layout="half", rot=None, norm=True, scaling="none",
               factor=1.0, orig=0, positions=None, pad=0, layers=2, layer=1, wide=0, spoil=None, q_none=False, theta=1e6,
               inplace=False, seed=0):
    """Runs one append and compares q_out and the whole pools with the reference."""
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    T, rot = sum(q_lens), D if rot is None else rot
    rows = T + pad
    kv = [n + p for n, p in zip(q_lens, past)]
    table, P = make_table(kv, page, g, spare=2)
    if spoil:
        spoil(table, P)
    ti, tq, tc = TYPES[act], TYPES[qact], TYPES[cache]
    width = (NQ + 2 * NKV) * D + wide
    qkv = torch.randn(rows, width, generator=g).to(ti)
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2)) if norm else (None, None)
    K0, V0 = (torch.randn(layers, P, NKV, page, D, generator=g).to(tc) for _ in range(2))
    k, v, x = K0.cuda(), V0.cuda(), qkv.cuda()
    parts = x[:, :(NQ + 2 * NKV) * D].unflatten(1, (NQ + 2 * NKV, D)).split((NQ, NKV, NKV), 1)
    q, kn, vn = parts
    if inplace:
        q = q.contiguous()
    q_out = q if inplace else torch.full((rows, NQ, D), 7.0, device="cuda", dtype=tq)
    old = q_out.cpu().clone()
    rp = None
    if rot:
        rp = paged.rope(rot, theta, layout=layout, scaling=scaling, factor=factor, orig_ctx=orig)
    b = make_batch(q_lens, kv, table, rows)
    pos_t = None if positions is None else ints(positions + [0] * pad)
    paged.kv_append(paged.kv_cache(k, v), layer, b, None if q_none else q, kn, vn, None if q_none else q_out, rope=rp,
                    q_norm=None if wq is None else wq.cuda(), k_norm=None if wk is None else wk.cuda(), eps=EPS,
                    positions=pos_t)
    torch.cuda.synchronize()
    # reference
    st = starts(q_lens)
    toks = tokens(st, kv)
    where = torch.tensor([p if positions is None else positions[t] for t, _, p in toks] + [0] * pad)
    X = qkv[:, :(NQ + 2 * NKV) * D].double().view(rows, NQ + 2 * NKV, D)
    Q, K = rmsnorm(X[:, :NQ], wq, EPS), rmsnorm(X[:, NQ:NQ + NKV], wk, EPS)
    m = 1.0
    if rot:
        f, m = frequencies(rot, theta, scaling, factor, orig)
        Q, K = rotate(Q, where, f, m, layout), rotate(K, where, f, m, layout)
    KN, VN = K0.double().clone(), V0.double().clone()
    tolK = torch.zeros_like(KN)
    QN = old.double().clone()

    # norm: 9 roundings of 2^-24 in 1 / sqrt, 2 of the products; angle 2^-26
    # turns = 1.6 of 2^-24, sin and cos 2 ulp, m 1, the pair's sum 2: below 24
    # of 2^-24 of the pair's length (at most the row's largest pair)
    def tol(y, t):
        return 24 * 2.0 ** -24 * math.sqrt(2) * y.abs().amax(-1, keepdim=True) + half_step(t) * y.abs() + least(t)

    for t, s, p in toks:
        if p < 0:
            continue
        QN[t] = Q[t]
        pg = page_of(table, s, p, page, P)
        if pg >= 0:
            KN[layer, pg, :, p % page], VN[layer, pg, :, p % page] = K[t], X[t, NQ + NKV:].to(tc).double()
            tolK[layer, pg, :, p % page] = tol(K[t], tc)
    dk = (k.cpu().double() - KN).abs()
    assert bool((dk <= tolK).all()), float((dk - tolK).max())
    assert torch.equal(v.cpu(), VN.to(tc))
    if not q_none:
        dq = (q_out.cpu().double() - QN).abs()
        seen = torch.zeros(rows, 1, 1, dtype=torch.bool)
        for t, s, p in toks:
            seen[t] = p >= 0
        tq_ = torch.where(seen, tol(QN, tq), torch.zeros(()).double())
        assert bool((dq <= tq_).all()), float((dq - tq_).max())


TYPE_SETS = [("f32", "f32", "f16"), ("f32", "f16", "f16"), ("f16", "f16", "f16"), ("f32", "f32", "bf16"),
             ("f32", "bf16", "bf16"), ("bf16", "bf16", "bf16")]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("act,qact,cache", TYPE_SETS)
def test_append_types(act, qact, cache, D):
    run_append(act, qact, cache, D, 4, 2, 16, [1, 5, 0, 18], [30, 0, 4, 15])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (128, 8), (128, 104), (64, 64), (64, 24), (64, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rotations(layout, D, rot, norm):
    run_append("f32", "f32", "f16", D, 3, 1, 32, [7, 2], [60, 0], layout=layout, rot=rot, norm=norm)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=8.0), dict(scaling="yarn", factor=4.0, orig=4096)])
def test_append_scalings(kw):
    run_append("f32", "f32", "f16", 128, 4, 2, 64, [3, 1], [1000, 5], **kw)


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 5), (24, 4), (64, 8), (40, 1), (128, 16)])
def test_append_head_counts(heads, kv):
    """Head counts around the 16 (head_dim 128) and 32 (64) that a workgroup takes at a time."""
    for D in (64, 128):
        run_append("bf16", "bf16", "bf16", D, heads, kv, 16, [2, 1], [3, 16], layers=1, layer=0)


def test_append_far_positions():
    """Angles of positions up to 2^31 - 1, given apart from the cache's (the
    reference's 64-bit angle of 2e9 is exact to 2e9 * 2^-53 = 2e-7 radians,
    2 of the test's 24 roundings)."""
    run_append("f32", "f32", "f16", 128, 2, 1, 16, [4], [0], positions=[0, 131071, 1 << 24, 2147483647], norm=False)


def test_append_strides_padding_and_bad_pages():
    """Rows wider than the heads, rows behind the last sequence, pages outside
    the pool, a table that is too short, tokens at negative positions."""
    def spoil(table, P):
        table[0][0] = -1
        table[1][0] = P
        table[2][0] = 2 ** 31 - 1
    run_append("f16", "f16", "f16", 128, 4, 2, 16, [17, 3, 2], [0, 0, 0], pad=5, wide=24, spoil=spoil)
    run_append("f32", "f32", "f16", 64, 4, 2, 16, [6, 3], [-4, -3], pad=1)


def test_append_without_q_and_in_place():
    run_append("f16", "f16", "f16", 128, 4, 2, 16, [5, 1], [9, 0], q_none=True)
    run_append("bf16", "bf16", "bf16", 64, 6, 3, 32, [5, 1], [9, 0], inplace=True)
    run_append("f32", "f32", "f16", 128, 33, 11, 32, [5, 1], [9, 0], inplace=True, layout="interleaved")


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 200])
def test_append_many_sequences(seqs):
    """Token to sequence lookups around the wave's 64 lanes, empty sequences among them."""
    run_append("f16", "f16", "f16", 64, 1, 1, 16, [(i * 7) % 4 for i in range(seqs)], [i % 20 for i in range(seqs)],
               layers=1, layer=0)


@pytest.mark.parametrize("seqs", [4095, 4096, 4097, 5000])
def test_append_thousands_of_sequences(seqs):
    """Lookups of one, two and three rounds, a long run of empty sequences among them."""
    run_append("f16", "f16", "f16", 64, 1, 1, 16, [0 if 100 < i < 1500 else (i * 7) % 3 for i in range(seqs)],
               [i % 5 for i in range(seqs)], layers=1, layer=0)


@pytest.mark.parametrize("T", [300, 2500])
def test_append_long_prompt(T):
    run_append("f32", "f16", "f16", 128, 4, 2, 64, [T], [100], scaling="yarn", factor=4.0, orig=1024)


# ---- attention ----------------------------------------------------------------------
def fill_seen(shape, table, kv, page, dtype, g):
    """A pool of NaN with random rows at every sequence's positions (all layers)."""
    torch = _torch()
    out = []
    for _ in range(2):
        t = torch.full(shape, float("nan"), dtype=dtype)
        for s, n in enumerate(kv):
            for p in range(n):
                pg = page_of(table, s, p, page, shape[1])
                if pg >= 0:
                    t[:, pg, :, p % page] = torch.randn(shape[0], shape[2], shape[4], generator=g).to(dtype)
        out.append(t)
    return out


def run_attention(act, cache, D, NQ, NKV, page, q_lens, past, window=0, sinks=0, scale=0.0, pad=0, layers=1, layer=0,
                  spoil=None, spoil_pool=None, wide=0, peak=1.0, seed=0, max_q=0, max_kv=0):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    kv = [n + p for n, p in zip(q_lens, past)]
    table, P = make_table([max(n, 0) for n in kv], page, g, spare=1)
    ta, tc = TYPES[act], TYPES[cache]
    K, V = fill_seen((layers, P, NKV, page, D), table, kv, page, tc, g)
    if spoil:
        spoil(table, P)
    if spoil_pool:
        spoil_pool(K, V, table, kv)
    st = starts(q_lens)
    rows = st[-1] + pad
    Q = (peak * torch.randn(rows, NQ * D + wide, generator=g)).to(ta)
    q = Q.cuda()[:, :NQ * D].unflatten(1, (NQ, D))
    out = torch.full((rows, NQ, D), 7.0, dtype=ta, device="cuda")
    c, b = paged.kv_cache(K.cuda(), V.cuda()), make_batch(q_lens, kv, table, rows, max_q=max_q, max_kv=max_kv)
    paged.attn_paged(c, layer, b, q, out, window=window, sinks=sinks, scale=scale)
    got = out.cpu().double()
    ref = attention(K, V, layer, st, kv, table, Q[:, :NQ * D].unflatten(1, (NQ, D)), window, sinks, scale)
    for t in range(rows):
        if t not in ref:
            assert bool((got[t] == 7.0).all()), t
            continue
        o, spread, size = ref[t]
        tol = attention_tolerance(o, spread, size, ta, tc)
        # a row that sees a NaN or an infinity is not finite there (which of them it is depends
        # on the order of its sums)
        fine = torch.isfinite(o)
        bad = torch.where(fine, ~((got[t] - o).abs() <= tol), torch.isfinite(got[t]))
        assert not bool(bad.any()), (t, float((got[t] - o).abs().max()), float(tol.min()))
    return got


ATTN_TYPES = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("act,cache", ATTN_TYPES)
@pytest.mark.parametrize("heads,kv", [(4, 1), (4, 4), (6, 2), (8, 1), (16, 1), (7, 1), (40, 2)])
def test_attention_single_tokens(act, cache, D, heads, kv):
    """A decode step: ragged lengths from one position on, one sequence without
    a new token, one without any position."""
    run_attention(act, cache, D, heads, kv, 16, [1, 1, 1, 0, 1, 1], [0, 30, 31, 5, 100, 290])


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
@pytest.mark.parametrize("heads,kv,D", [(4, 2, 64), (6, 2, 128), (8, 1, 128), (5, 5, 64)])
def test_attention_chunks(act, cache, heads, kv, D):
    """Chunks and single tokens in one batch, rows behind the last sequence."""
    run_attention(act, cache, D, heads, kv, 32, [70, 1, 3, 17, 0, 129], [0, 77, 5, 200, 9, 1], pad=4)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_page_sizes(page):
    for act, cache in ATTN_TYPES:
        run_attention(act, cache, 64, 4, 2, page, [1, 40, 90], [300, 60, 0], layers=2, layer=1)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (16, 0), (17, 4), (64, 1), (100, 33), (64, 64), (63, 70),
                                          (5, 1000), (1000, 4)])
def test_attention_windows(window, sinks):
    for act, cache in (("f32", "f16"), ("bf16", "bf16")):
        run_attention(act, cache, 64, 4, 2, 16, [1, 1, 37, 100], [299, 3, 250, 60], window=window, sinks=sinks)


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
def test_attention_long_context(act, cache):
    """Contexts split over many workgroups, single tokens and a chunk."""
    run_attention(act, cache, 128, 4, 1, 64, [1, 2], [4000, 9])
    run_attention(act, cache, 64, 4, 1, 64, [33], [3000])


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
@pytest.mark.parametrize("q,heads,kv,past", [(9, 4, 1, 700), (17, 8, 4, 2300), (40, 4, 1, 5000), (33, 6, 2, 1100)])
def test_attention_chunks_split_over_the_positions(act, cache, q, heads, kv, past):
    """A few tokens over a long context, in one to dozens of splits, beside a single token."""
    run_attention(act, cache, 64, heads, kv, 64, [q, 1], [past, 900])


@pytest.mark.parametrize("heads,kv,D", [(12, 3, 128), (33, 3, 64), (4, 1, 64)])
def test_attention_joins_of_few_and_of_many_splits(heads, kv, D):
    """As many splits as a row's lanes add in turn, and more (a workgroup a row); heads that leave a
    joining workgroup partly empty."""
    run_attention("f16", "f16", D, heads, kv, 64, [16], [9 * 64 * 4])
    run_attention("f16", "f16", D, heads, kv, 64, [16], [36 * 64 * 4])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("act,cache", ATTN_TYPES)
def test_attention_drafts(act, cache, wide):
    """Rows around the 16 and the 32 that a sequence of few rows has at most, in batches that may hold
    little and more than 256 MiB of keys and values (wide tables)."""
    def widen(table, P):
        for r in table:
            r.extend([-1] * 200)
    for window in (0, 150):
        run_attention(act, cache, 64, 16, 8, 256, [1, 4, 5, 8, 9, 16, 17], [300, 20, 0, 511, 300, 100, 250],
                      window=window, spoil=widen if wide else None)


def test_attention_bounds_leave_out_what_lies_beyond():
    """Lengths above max_q and max_kv: the rows within them are as ever where nothing of theirs is
    left out, nothing else is written or read."""
    torch = _torch()
    g = torch.Generator().manual_seed(2)
    q_lens, kv = [1, 60, 2], [90, 70, 200]
    table, P = make_table(kv, 16, g)
    K, V = fill_seen((1, P, 2, 16, 64), table, kv, 16, torch.float16, g)
    Q = torch.randn(63, 4, 64, generator=g).half()
    c, out = paged.kv_cache(K.cuda(), V.cuda()), torch.full((63, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    b = make_batch(q_lens, kv, table, max_q=2, max_kv=100)
    paged.attn_paged(c, 0, b, Q.cuda(), out)
    ref = attention(K, V, 0, starts(q_lens), kv, table, Q)
    o, spread, size = ref[0]
    assert bool(((out[0].cpu().double() - o).abs() <= attention_tolerance(o, spread, size, torch.float16, torch.float16)).all())
    assert bool((out[1:61] == 7.0).all())          # more tokens than max_q
    assert bool(torch.isfinite(out[61:]).all())    # positions from 100 on left out


def test_attention_bad_pages_are_not_seen():
    def spoil(table, P):
        table[0][1] = -1                 # a hole
        table[1] = [P] * len(table[1])   # nothing left: rows of zeros
        table[2][0] = 2 ** 31 - 1
    for act, cache in ATTN_TYPES:
        got = run_attention(act, cache, 64, 4, 2, 16, [1, 3, 20], [60, 9, 30], spoil=spoil)
        assert bool((got[1:4] == 0).all())


def test_attention_rows_that_see_nothing():
    """Tokens before position 0 (a sequence shorter than its chunk) are zeros."""
    for act, cache in ATTN_TYPES:
        got = run_attention(act, cache, 128, 8, 2, 16, [3, 40], [-2, -30])
        assert bool((got[:2] == 0).all()) and bool((got[3:33] == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_unseen_values_have_no_influence(bad, which):
    """A position that holds NaN or an infinity changes the rows that see it
    and no other: tokens before it, and tokens whose window has passed it."""
    def spoil_pool(K, V, table, kv):
        t = K if which == "k" else V
        for s, p in ((0, 50), (1, 99), (2, 3)):
            t[:, table[s][p // 16], :, p % 16] = bad
    for act, cache in ATTN_TYPES:
        for window, sinks in ((0, 0), (7, 2)):
            if window == 0 and which == "k" and bad == -float("inf"):
                continue   # scores of either infinity: the reference's own NaN rows
            run_attention(act, cache, 64, 4, 2, 16, [60, 9, 1, 6], [0, 91, 40, 3], window=window, sinks=sinks,
                          spoil_pool=spoil_pool)


@pytest.mark.parametrize("past", [40, 900])
def test_attention_keys_of_minus_infinity_weigh_nothing(past):
    """A key that a 16-bit cache holds as -infinity in one place, where every row of q is positive: the
    formula gives it the weight 0 and a finite row, in few rows and in many, split or not."""
    torch = _torch()
    g = torch.Generator().manual_seed(past)
    q_lens, kv = [1, 3, 60], [1 + past, 3 + past, 60 + past]
    for act, cache in ATTN_TYPES:
        table, P = make_table(kv, 16, g)
        K, V = fill_seen((1, P, 2, 16, 64), table, kv, 16, TYPES[cache], g)
        K0 = K.clone()
        for s in range(3):
            for p in (5, 33, past - 1):
                K[0, table[s][p // 16], :, p % 16, 7] = -float("inf")
                K0[0, table[s][p // 16], :, p % 16, 7] = 0
        Q = torch.randn(64, 8, 64, generator=g).to(TYPES[act])
        Q[:, :, 7] = Q[:, :, 7].abs() + 0.1
        out = torch.empty(64, 8, 64, dtype=TYPES[act], device="cuda")
        paged.attn_paged(paged.kv_cache(K.cuda(), V.cuda()), 0, make_batch(q_lens, kv, table), Q.cuda(), out)
        ref, sizes = (attention(k, V, 0, starts(q_lens), kv, table, Q) for k in (K, K0))
        for t in ref:
            o, spread, _ = ref[t]
            tol = attention_tolerance(o, spread, sizes[t][2], TYPES[act], TYPES[cache])   # finite scores' sizes
            assert bool(torch.isfinite(o).all()) and bool(((out[t].cpu().double() - o).abs() <= tol).all()), (act, t)


def test_attention_unseen_values_in_one_of_several_splits():
    """A chunk over a context long enough to be split: the last split holds a NaN that only the
    last token sees, the first one what a window has passed; the other rows join as if they were
    not there."""
    def last(K, V, table, kv):
        for t in (K, V):
            t[:, table[0][(kv[0] - 1) // 64], :, (kv[0] - 1) % 64] = float("nan")
    for act, cache in ATTN_TYPES:
        run_attention(act, cache, 64, 4, 1, 64, [40], [2500], spoil_pool=last)

    def early(K, V, table, kv):
        V[:, table[0][20], :, 40:] = float("inf")   # positions 1320..1343 of a window of 1200
    for act, cache in ATTN_TYPES:
        run_attention(act, cache, 64, 4, 1, 64, [40], [2510], window=1200, sinks=70, spoil_pool=early)


@pytest.mark.parametrize("peak", [0.0, 30.0])
def test_attention_score_sizes(peak):
    """All scores alike, and one position that takes nearly all of a row."""
    for act, cache in ATTN_TYPES:
        run_attention(act, cache, 128, 4, 2, 16, [1, 50], [200, 10], peak=peak)


@pytest.mark.parametrize("peak,scale", [(1e-37, 0.0), (1e-37, 1e-37), (1.0, 1e-38), (1e30, 1e-32), (6e4, 1e-6)])
def test_attention_sizes_at_the_ends_of_the_types(peak, scale):
    """Rows and scales whose product leaves fp32's normal numbers, or whose scores come near its end."""
    for act, cache in ATTN_TYPES:
        p = min(peak, 1e4) if act == "f16" else peak
        run_attention(act, cache, 64, 4, 2, 16, [1, 50], [200, 10], peak=p, scale=scale if p == peak else 1e-6)


def test_attention_scale_strides_and_bounds():
    for act, cache in ATTN_TYPES:
        run_attention(act, cache, 64, 4, 2, 16, [1, 20], [50, 3], scale=0.5, wide=16, max_q=20, max_kv=51)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129])
def test_attention_lengths_around_tiles(n):
    run_attention("f16", "f16", 64, 2, 1, 16, [1, n, 2], [n, 0, n])


def test_attention_many_sequences():
    run_attention("f16", "f16", 64, 2, 2, 16, [1 if i % 3 else i % 7 for i in range(130)], [i % 40 for i in range(130)])


def test_cache_beyond_32_bits():
    """Pages whose elements lie behind 2^32 of the pool: 40000 pages of 8 heads."""
    torch = _torch()
    P, NKV, page, D = 40000, 8, 64, 128
    k, v = (torch.empty(2, P, NKV, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    c = paged.kv_cache(k, v)
    kv, table = [100, 3], [[P - 1, 17], [P - 3, -1]]
    g = torch.Generator().manual_seed(1)
    x = torch.randn(103, 12 * D * 2, generator=g).cuda().view(103, 24, D)
    b = make_batch([100, 3], kv, table)
    q_out = torch.empty(103, 8, D, device="cuda")
    paged.kv_append(c, 1, b, x[:, :8], x[:, 8:16], x[:, 16:], q_out)
    out = torch.empty_like(q_out)
    paged.attn_paged(c, 1, b, q_out, out)
    paged.kv_copy_pages(c, [P - 1, P - 3], [P - 2, P - 5])
    torch.cuda.synchronize()
    pages = [P - 1, 17, P - 3]
    K, V = k[:, pages].cpu(), v[:, pages].cpu()
    assert torch.equal(k[1, P - 2], k[1, P - 1]) and torch.equal(v[1, P - 5], v[1, P - 3])
    assert torch.equal(K[1, 0], x[:64, 8:16].half().transpose(0, 1).cpu())
    ref = attention(K, V, 1, [0, 100, 103], kv, [[0, 1], [2, -1]], q_out.cpu())
    for t in ref:
        o, spread, size = ref[t]
        tol = attention_tolerance(o, spread, size, torch.float32, torch.float16)
        assert bool(((out[t].cpu().double() - o).abs() <= tol).all()), t


# ---- copies and compaction -------------------------------------------------------------
@pytest.mark.parametrize("D,NKV,page,layers", [(64, 1, 16, 1), (128, 8, 64, 3), (64, 3, 256, 2), (128, 5, 32, 2)])
@pytest.mark.parametrize("n", [1, 3, 130])
def test_copy_pages(D, NKV, page, layers, n):
    torch = _torch()
    g = torch.Generator().manual_seed(n)
    P = 2 * n + 1
    K, V = (torch.randn(layers, P, NKV, page, D, generator=g).half() for _ in range(2))
    k, v = K.cuda(), V.cuda()
    ids = torch.randperm(P, generator=g).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    if n > 2:
        src[1] = src[0]   # one page to two places
    paged.kv_copy_pages(paged.kv_cache(k, v), src, dst)
    K[:, dst], V[:, dst] = K[:, src], V[:, src]
    assert torch.equal(k.cpu(), K) and torch.equal(v.cpu(), V)


@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 64), (64, 256)])
@pytest.mark.parametrize("lens,kept", [([5], [5]), ([40, 1, 33], [0, 1, 20]), ([700], [333]), ([1000, 300], [999, 150]),
                                       ([260], [129])])
def test_compact(D, page, lens, kept):
    torch = _torch()
    g = torch.Generator().manual_seed(sum(lens))
    layers, NKV = 2, 3
    table, P = make_table(lens, page, g, spare=1)
    K, V = (torch.randn(layers, P, NKV, page, D, generator=g).bfloat16() for _ in range(2))
    keep = [sorted(torch.randperm(n, generator=g)[:m].tolist()) for n, m in zip(lens, kept)]
    k, v = K.cuda(), V.cuda()
    flat = [x for r in keep for x in r]
    paged.kv_compact(paged.kv_cache(k, v), ints(table), ints(starts(kept)), ints(flat or [0]))
    for t, dev in ((K, k), (V, v)):
        old = t.clone()
        for s, r in enumerate(keep):
            for j, p in enumerate(r):
                t[:, table[s][j // page], :, j % page] = old[:, table[s][p // page], :, p % page]
        assert torch.equal(dev.cpu(), t)


def test_compact_of_nothing():
    """No row of any sequence kept: nothing to move, and keep is an empty tensor."""
    torch = _torch()
    k = torch.randn(1, 4, 1, 16, 64).half().cuda()
    old = k.clone()
    paged.kv_compact(paged.kv_cache(k, k.clone()), ints([[0, 1], [2, 3]]), ints([0, 0, 0]), ints([]))
    assert torch.equal(k, old)


def test_compact_skips_bad_pages():
    """Rows without a page, as source or as destination, are left out."""
    torch = _torch()
    K = torch.randn(1, 4, 1, 16, 64).half()
    k, v = K.cuda(), K.cuda()
    paged.kv_compact(paged.kv_cache(k, v), ints([[0, -1, 2, 9]]), ints([0, 18]), ints(list(range(24, 40)) + [-5, 63]))
    want = K.clone()
    want[0, 0, :, 8:16] = K[0, 2, :, 0:8]   # sources 24..31 have no page, 32..39 are page 2's
    assert torch.equal(k.cpu(), want)


# ---- graphs, streams, devices -------------------------------------------------------------
def _decode_state(seed, cache="f16", act="f32"):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    kv = [70, 200]
    table, P = make_table([256, 256], 16, g)
    K, V = (torch.randn(1, P, 2, 16, 64, generator=g).to(TYPES[cache]).cuda() for _ in range(2))
    c, b = paged.kv_cache(K, V), make_batch([1, 1], kv, table, max_q=1, max_kv=256)
    x = torch.randn(2, 8, 64, generator=g).to(TYPES[act]).cuda()
    n = paged.attn_workspace_size(c, b, 4, x.dtype)
    return dict(c=c, b=b, x=x, K=K, V=V, q=torch.empty(2, 4, 64, device="cuda", dtype=x.dtype),
                out=torch.empty(2, 4, 64, device="cuda", dtype=x.dtype),
                ws=torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), rope=paged.rope(64, 1e4))


def _step(s):
    paged.kv_append(s["c"], 0, s["b"], s["x"][:, :4], s["x"][:, 4:6], s["x"][:, 6:], s["q"], rope=s["rope"])
    paged.attn_paged(s["c"], 0, s["b"], s["q"], s["out"], workspace=s["ws"])
    return s["out"]


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
def test_captured_decode_steps_follow_the_lengths(act, cache):
    """One capture replayed while the sequences grow (device lengths), with
    eager work between, against eager calls on a copy of the state; two such
    graphs with workspaces of their own, replayed in turn."""
    torch = _torch()
    graphs = []
    for seed in (1, 2):
        s, e = _decode_state(seed, cache, act), _decode_state(seed, cache, act)
        _step(s)   # warm-up; the same row is appended again below
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            _step(s)
        graphs.append((gr, s, e))
    for r in range(4):
        for gr, s, e in graphs:
            new = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(r)).to(s["x"].dtype)
            for st in (s, e):
                st["x"].copy_(new)
                st["b"]._keep[1].copy_(ints([70 + r, 200 + 13 * r]))
            gr.replay()
            want = _step(e).clone()
            torch.cuda.synchronize()
            assert torch.equal(s["out"], want) and torch.equal(s["K"], e["K"]) and torch.equal(s["V"], e["V"])


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
def test_captured_chunks(act, cache):
    """A chunk's append and attention, split and joined, captured with a workspace from the call itself
    and replayed over new rows, with eager calls between."""
    torch = _torch()
    g = torch.Generator().manual_seed(9)
    kv, q_lens = [2500, 30], [40, 1]
    table, P = make_table(kv, 64, g)
    K, V = (torch.randn(1, P, 2, 64, 128, generator=g).to(TYPES[cache]).cuda() for _ in range(2))
    c, b = paged.kv_cache(K, V), make_batch(q_lens, kv, table)
    x = torch.randn(41, 12, 128, generator=g).to(TYPES[act]).cuda()
    q, out = torch.empty_like(x[:, :8]).contiguous(), torch.empty(41, 8, 128, device="cuda", dtype=TYPES[act])
    rope = paged.rope(128, 1e4)

    def step(o):
        paged.kv_append(c, 0, b, x[:, :8], x[:, 8:10], x[:, 10:], q, rope=rope)
        paged.attn_paged(c, 0, b, q, o)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        step(out)
    for r in range(3):
        x.copy_(torch.randn(41, 12, 128, generator=g))
        gr.replay()
        want = torch.empty_like(out)
        step(want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_another_stream():
    torch = _torch()
    a, b = _decode_state(3), _decode_state(3)
    want = _step(a).clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _step(b)
    st.synchronize()
    assert torch.equal(b["out"], want)


def test_calls_repeat_bit_for_bit():
    torch = _torch()
    s = _decode_state(5)
    want = _step(s).clone()
    for _ in range(3):
        assert torch.equal(_step(s), want)


def test_python_refusals():
    torch = _torch()
    s = _decode_state(6)
    x, c, b = s["x"], s["c"], s["b"]
    with pytest.raises(ValueError, match="cpu"):
        paged.attn_paged(c, 0, b, s["q"].cpu(), s["out"])
    with pytest.raises(ValueError, match="device"):
        paged.kv_cache(s["K"].cpu(), s["V"].cpu())
    with pytest.raises(ValueError, match="device"):
        paged.kv_batch(b._keep[0].cpu(), b._keep[1], b._keep[2], 2)
    with pytest.raises(ValueError, match="out"):
        paged.attn_paged(c, 0, b, s["q"], s["out"].half())
    with pytest.raises(ValueError, match="side by side"):
        paged.kv_append(c, 0, b, x[:, ::2], x[:, 4:6], x[:, 6:], s["q"])
    with pytest.raises(ValueError, match="one type"):
        paged.kv_append(c, 0, b, x[:, :4], x[:, 4:6].half(), x[:, 6:].half(), s["q"])
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        paged.kv_cache(s["K"].float(), s["V"].float())
    with pytest.raises(ValueError, match="int32"):
        paged.kv_batch(b._keep[0].long(), b._keep[1], b._keep[2], 2)
    with pytest.raises(tb.TbqError, match="layer"):
        paged.attn_paged(c, 1, b, s["q"], s["out"])
    if paged.attn_workspace_size(c, b, 4, torch.float32) > 16:
        with pytest.raises(tb.TbqError, match="workspace"):
            paged.attn_paged(c, 0, b, s["q"], s["out"], workspace=s["ws"][:16])


@pytest.mark.parametrize("act,cache,size", [("bf16", "bf16", 3e38), ("f16", "f16", 65504.0), ("f32", "f16", 65504.0)])
@pytest.mark.parametrize("past", [60, 2500])
def test_attention_values_at_the_end_of_their_type(act, cache, size, past):
    """Averages of values whose sum fp32 does not hold: few rows and many, split or not."""
    def big(K, V, table, kv):
        V.copy_(_torch().where(_torch().isnan(V), V, V.sign() * size))
        V[:, :, :, :, :8] = V[:, :, :, :, :8].abs()   # dims where they are all alike
    run_attention(act, cache, 64, 4, 1, 64, [1, 40], [past, past], spoil_pool=big)


# ---- long loops: lists, lookups and splits that follow the first ------------------------------
def check_sampled(got, K, V, layer, st, kv, table, Q, rows, window, sinks, ta, tc):
    """The sampled token rows against the 64-bit form, each as a batch of its own."""
    for t, s, pos in tokens(st, kv):
        if t in rows:
            o, spread, size = attention(K, V, layer, [0, 1], [pos + 1], [table[s]], Q[t:t + 1], window, sinks)[0]
            tol = attention_tolerance(o, spread, size, ta, tc)
            assert bool(((got[t].double() - o).abs() <= tol).all()), (t, s, pos)


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (3001, 150)])
def test_attention_chunk_of_many_tiles(act, cache, window, sinks):
    """A prompt's chunk of enough blocks that none is split (100 of 8 kv heads): up to 91 tiles one after
    the other on shuffled pages, looked up 16 at a time, the sinks' in front of a window's."""
    torch = _torch()
    g = torch.Generator().manual_seed(31)
    T, past, page, NQ, NKV, D = 3200, 2600, 64, 32, 8, 64
    ta, tc = TYPES[act], TYPES[cache]
    table, P = make_table([T + past], page, g, spare=3)
    K, V = (torch.full((1, P, NKV, page, D), float("nan"), dtype=tc) for _ in range(2))
    for t in (K, V):
        t[:, table[0]] = torch.randn(1, len(table[0]), NKV, page, D, generator=g).to(tc)
        t[:, table[0][-1], :, (T + past - 1) % page + 1:] = float("nan")
    Q = torch.randn(T, NQ, D, generator=g).to(ta)
    out = torch.empty(T, NQ, D, dtype=ta, device="cuda")
    b = make_batch([T], [T + past], table)
    paged.attn_paged(paged.kv_cache(K.cuda(), V.cuda()), 0, b, Q.cuda(), out, window=window, sinks=sinks)
    rows = {0, 1, 31, 32, 700, 1023, 1555, 2048, 3000, 3198, 3199}
    assert bool(torch.isfinite(out).all())
    check_sampled(out.cpu(), K, V, 0, [0, T], [T + past], table, Q, rows, window, sinks, ta, tc)


@pytest.mark.parametrize("act,cache", ATTN_TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (6000, 70)])
def test_attention_single_tokens_of_many_tiles(act, cache, window, sinks):
    """Enough workgroups (400 sequences of 8 kv heads) that a split has 192 tiles, 48 a wave, whose pages
    are looked up 32 tiles at a time; the sequences share a few pages in orders of their own."""
    torch = _torch()
    g = torch.Generator().manual_seed(32)
    S, page, P, NQ, NKV, D, most = 400, 256, 40, 16, 8, 64, 30
    ta, tc = TYPES[act], TYPES[cache]
    K, V = (torch.randn(1, P, NKV, page, D, generator=g).to(tc) for _ in range(2))
    kv = torch.randint(1, most * page + 1, (S,), generator=g).tolist()
    kv[:6] = [most * page, 4096, 4097, 4128, 6144, 6145]
    table = [torch.randint(0, P, (most,), generator=g).tolist() for _ in range(S)]
    Q = torch.randn(S, NQ, D, generator=g).to(ta)
    out = torch.empty(S, NQ, D, dtype=ta, device="cuda")
    b = make_batch([1] * S, kv, table)
    paged.attn_paged(paged.kv_cache(K.cuda(), V.cuda()), 0, b, Q.cuda(), out, window=window, sinks=sinks)
    rows = set(range(6)) | set(range(50, S, 60))
    check_sampled(out.cpu(), K, V, 0, list(range(S + 1)), kv, table, Q, rows, window, sinks, ta, tc)


# layers and sequences that give a workgroup 1, 2, 3, 5, 16, 33 and 64 columns; rows beyond one and two lists
@pytest.mark.parametrize("D,NKV,layers,lens,kept", [
    (64, 1, 1, [4000], [2500]), (128, 1, 512, [1500], [1100]), (64, 3, 512, [1300], [1030]), (64, 5, 512, [1200], [1001]),
    (128, 8, 512, [1200], [1030]), (64, 33, 32, [90, 40, 70, 7] * 4, [50, 1, 70, 0] * 4),
    (128, 32, 32, [90, 40, 70, 7] * 4, [50, 1, 69, 3] * 4)])
def test_compact_many_rows_and_columns(D, NKV, layers, lens, kept):
    torch = _torch()
    g = torch.Generator().manual_seed(sum(lens) + NKV)
    page = 16
    table, P = make_table(lens, page, g, spare=1)
    gg = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randint(-2 ** 15, 2 ** 15, (layers, P, NKV, page, D), generator=gg, device="cuda", dtype=torch.int16)
            for _ in range(2))
    keep = [sorted(torch.randperm(n, generator=g)[:m].tolist()) for n, m in zip(lens, kept)]
    want = []
    for t in (k, v):
        w = t.clone()
        for s, r in enumerate(keep):
            at = lambda ps: (torch.tensor([table[s][p // page] for p in ps], dtype=torch.int64).cuda(),   # noqa: E731
                             torch.tensor([p % page for p in ps], dtype=torch.int64).cuda())
            if r:
                (ps, rs), (pd, rd) = at(r), at(range(len(r)))
                w.transpose(2, 3)[:, pd, rd] = t.transpose(2, 3)[:, ps, rs]
        want.append(w)
    c = paged.kv_cache(k.view(torch.float16), v.view(torch.float16))
    paged.kv_compact(c, ints(table), ints(starts(kept)), ints([x for r in keep for x in r]))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("D,heads,kv,q_lens,past", [(128, 32, 8, [1, 1, 1], [299, 4999, 8]), (64, 8, 1, [1], [20000]),
                                                    (64, 4, 1, [8, 3, 1], [700, 40, 5000]), (128, 17, 1, [1], [3000])])
@pytest.mark.parametrize("window", [0, 256])
def test_attention_of_few_rows_rounds_only_its_output(act, D, heads, kv, q_lens, past, window):
    """Single tokens and drafts (up to 32 rows a kv head) of 16-bit rows: the probabilities are pairs (each
    half off by half a step of what it rounds), so what is left is fp32's (attention_tolerance's first terms)
    and the one rounding of the output."""
    torch = _torch()
    g = torch.Generator().manual_seed(D + heads)
    t, page, kvl = TYPES[act], 64, [n + p for n, p in zip(q_lens, past)]
    table, P = make_table(kvl, page, g)
    K, V = (torch.randn(1, P, kv, page, D, generator=g).to(t) for _ in range(2))
    T = sum(q_lens)
    Q = torch.randn(T, heads, D, generator=g).to(t)
    out = torch.empty(T, heads, D, dtype=t, device="cuda")
    paged.attn_paged(paged.kv_cache(K.cuda(), V.cuda()), 0, make_batch(q_lens, kvl, table), Q.cuda(), out, window=window)
    ref = attention(K, V, 0, starts(q_lens), kvl, table, Q, window)
    for r in ref:
        o, spread, size = ref[r]
        tol = attention_tolerance(o, spread, size, torch.float32, t)
        tol = tol + half_step(t) ** 2 * spread
        tol = tol + half_step(t) * (o.abs() + tol) + least(t)
        assert bool(((out[r].cpu().double() - o).abs() <= tol).all()), r


def test_named_stream_without_a_workspace():
    """Calls on a stream that is not the current one, workspaces their own, while the current one's
    memory comes and goes."""
    torch = _torch()
    a, b = _decode_state(3), _decode_state(3)
    want, st = _step(a).clone(), torch.cuda.Stream()
    for _ in range(3):
        st.wait_stream(torch.cuda.current_stream())
        paged.kv_append(b["c"], 0, b["b"], b["x"][:, :4], b["x"][:, 4:6], b["x"][:, 6:], b["q"], rope=b["rope"], stream=st)
        paged.attn_paged(b["c"], 0, b["b"], b["q"], b["out"], stream=st)
        for _ in range(4):
            torch.full((1 << 16,), float("nan"), device="cuda")
        st.synchronize()
        assert torch.equal(b["out"], want)
    X, W = torch.randn(40, 2048, device="cuda").half(), torch.randn(64, 2048, device="cuda").half()
    got = [torch.empty(40, 64, device="cuda") for _ in range(2)]
    st.wait_stream(torch.cuda.current_stream())
    tb.gemm(W, 1, X, 40, 64, 2048, got[0], stream=st)
    tb.gemm(W, 1, X, 40, 64, 2048, got[1])
    st.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(*got)
