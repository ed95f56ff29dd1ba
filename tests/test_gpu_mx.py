"""GPU checks of the MXFP4 cache (include/tbq_kv.h) against the format's
definition (mx_ref.py) and 64-bit formulas (paged_ref.py), through the package's
entry points.  Pages that nobody has written hold 0xFF (codes of -6 under a NaN
scale), so a read of what a call has no business to look at shows."""
import math

import numpy as np
import pytest

import mx_ref
import trailblaze_amd as tb
from paged_ref import (TYPES, attention, attention_tolerance, frequencies, half_step, least, make_table, page_of, rmsnorm,
                       rotate, tokens)
from trailblaze_amd import paged

pytestmark = pytest.mark.gpu
EPS = 1e-6
ACTS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module", autouse=True)
def _init():
    print("device:", tb.init(), flush=True)


def _torch():
    import torch
    return torch


def ints(v):
    return _torch().tensor(v, dtype=_torch().int32, device="cuda")


def starts(lens):
    return [0] + [int(x) for x in np.cumsum(lens)]


def make_batch(q_lens, kv_len, table, rows=None, **kw):
    st = starts(q_lens)
    return paged.kv_batch(ints(st), ints(kv_len), ints(table), st[-1] if rows is None else rows, **kw)


def empty_pool(layers, P, NKV, page, D):
    torch = _torch()
    return torch.full((layers, P, NKV, paged.kv_head_bytes(page, D)), 255, dtype=torch.uint8)


# ---- append ----------------------------------------------------------------------
def run_append(act, qact, D, NQ, NKV, page, q_lens, past, layout="half", rot=None, norm=True, scaling="none", factor=1.0,
               orig=0, positions=None, pad=0, layers=2, layer=1, wide=0, spoil=None, q_none=False, theta=1e6, seed=0,
               change=None):
    """One append: q_out within its roundings, both pools byte for byte.  (Keys are formed in 64 bits on both
    sides, 1e-15 apart; none of the seeded values lies that near a border between codes.)"""
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    T, rot = sum(q_lens), D if rot is None else rot
    rows = T + pad
    kv = [n + p for n, p in zip(q_lens, past)]
    table, P = make_table(kv, page, g, spare=2)
    if spoil:
        spoil(table, P)
    ti, tq = TYPES[act], TYPES[qact]
    width = (NQ + 2 * NKV) * D + wide
    qkv = torch.randn(rows, width, generator=g)
    if change:
        change(qkv)
    qkv = qkv.to(ti)
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2)) if norm else (None, None)
    K0, V0 = (torch.randint(0, 256, empty_pool(layers, P, NKV, page, D).shape, generator=g).to(torch.uint8) for _ in range(2))
    k, v, x = K0.cuda(), V0.cuda(), qkv.cuda()
    q, kn, vn = x[:, :(NQ + 2 * NKV) * D].unflatten(1, (NQ + 2 * NKV, D)).split((NQ, NKV, NKV), 1)
    q_out = torch.full((rows, NQ, D), 7.0, device="cuda", dtype=tq)
    rp = paged.rope(rot, theta, layout=layout, scaling=scaling, factor=factor, orig_ctx=orig) if rot else None
    b = make_batch(q_lens, kv, table, rows)
    paged.kv_append(paged.kv_cache(k, v, head_dim=D), layer, b, None if q_none else q, kn, vn, None if q_none else q_out,
                    rope=rp, q_norm=None if wq is None else wq.cuda(), k_norm=None if wk is None else wk.cuda(), eps=EPS,
                    positions=None if positions is None else ints(positions + [0] * pad))
    torch.cuda.synchronize()
    toks = tokens(starts(q_lens), kv)
    where = torch.tensor([p if positions is None else positions[t] for t, _, p in toks] + [0] * pad)
    X = qkv[:, :(NQ + 2 * NKV) * D].double().view(rows, NQ + 2 * NKV, D)
    eps = float(np.float32(EPS))
    Q, K = rmsnorm(X[:, :NQ], wq, eps), rmsnorm(X[:, NQ:NQ + NKV], wk, eps)
    if rot:
        f, m = frequencies(rot, theta, scaling, factor, orig)
        Q, K = rotate(Q, where, f, m, layout), rotate(K, where, f, m, layout)
    (KC, KS), (VC, VS) = (mx_ref.unpack(t, page, D, is_v) for t, is_v in ((K0, False), (V0, True)))
    kc, ks = mx_ref.blocks(K)
    vc, vs = mx_ref.blocks(X[:, NQ + NKV:])
    QN, seen = torch.full((rows, NQ, D), 7.0).double(), torch.zeros(rows, 1, 1, dtype=torch.bool)
    for t, s, p in toks:
        if p < 0:
            continue
        QN[t], seen[t] = Q[t], True
        pg = page_of(table, s, p, page, P)
        if pg >= 0:
            KC[layer, pg, :, p % page], KS[layer, pg, :, p % page] = kc[t], ks[t]
            VC[layer, pg, :, p % page], VS[layer, pg, :, p % page] = vc[t], vs[t]
    assert torch.equal(k.cpu(), mx_ref.pack(KC, KS, False))
    assert torch.equal(v.cpu(), mx_ref.pack(VC, VS, True))
    if not q_none:
        # as over 16-bit pages: below 24 of 2^-24 of the pair's length, and the output's rounding
        tol = 24 * 2.0 ** -24 * math.sqrt(2) * QN.abs().amax(-1, keepdim=True) + half_step(tq) * QN.abs() + least(tq)
        dq, tol = (q_out.cpu().double() - QN).abs(), torch.where(seen, tol, torch.zeros(()).double())
        bad = torch.where(torch.isfinite(QN), ~(dq <= tol), torch.isfinite(q_out.cpu()))
        assert not bool(bad.any())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("act,qact", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
def test_append_types(act, qact, D):
    run_append(act, qact, D, 4, 2, 16, [1, 5, 0, 18], [30, 0, 4, 15])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (128, 8), (128, 104), (64, 64), (64, 24), (64, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rotations(layout, D, rot, norm):
    run_append("f32", "f32", D, 3, 1, 32, [7, 2], [60, 0], layout=layout, rot=rot, norm=norm)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=8.0), dict(scaling="yarn", factor=4.0, orig=4096)])
def test_append_scalings(kw):
    run_append("f32", "f32", 128, 4, 2, 64, [3, 1], [1000, 5], **kw)


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 5), (24, 4), (64, 8), (40, 1), (128, 16), (15, 5), (47, 1)])
def test_append_head_counts(heads, kv):
    """Head counts around the 16 (head_dim 128) and 32 (64) that a workgroup takes at a time."""
    for D in (64, 128):
        run_append("bf16", "bf16", D, heads, kv, 16, [2, 1], [3, 16], layers=1, layer=0)


def test_append_strides_padding_and_bad_pages():
    """Rows wider than the heads, rows behind the last sequence, pages outside the pool, a table that is
    too short, tokens at negative positions, positions of their own."""
    def spoil(table, P):
        table[0][0] = -1
        table[1][0] = P
        table[2][0] = 2 ** 31 - 1
    run_append("f16", "f16", 128, 4, 2, 16, [17, 3, 2], [0, 0, 0], pad=5, wide=24, spoil=spoil)
    run_append("f32", "f32", 64, 4, 2, 16, [6, 3], [-4, -3], pad=1)
    run_append("f32", "f32", 128, 2, 1, 16, [4], [0], positions=[0, 9, 70001, 1000003], norm=False, pad=2)
    run_append("bf16", "bf16", 64, 2, 2, 128, [5, 1], [9, 0], q_none=True)


@pytest.mark.parametrize("T", [300, 2500])
def test_append_long_prompt(T):
    run_append("f32", "f16", 128, 4, 2, 64, [T], [100], scaling="yarn", factor=4.0, orig=1024)


def test_append_many_sequences():
    run_append("f16", "f16", 64, 1, 1, 16, [(i * 7) % 4 for i in range(200)], [i % 20 for i in range(200)], layers=1, layer=0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("act,qact", [("f32", "f16"), ("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv,D,T", [(32, 8, 128, 700), (16, 4, 128, 1100), (50, 5, 128, 600), (32, 8, 64, 1100),
                                          (64, 16, 64, 700), (100, 10, 64, 600)])
def test_append_long_prompts_of_many_heads(heads, kv, D, T, act, qact, layout):
    """Prompts and heads enough for two and for three heads a lane, the last workgroup of a token full, partly and all but
    empty."""
    run_append(act, qact, D, heads, kv, 64, [T, 3], [100, 9], layout=layout, rot=D if T > 700 else D // 2, layers=1, layer=0,
               pad=2)


@pytest.mark.parametrize("act", ACTS)
def test_append_sizes_of_values(act):
    """Blocks of zeros, of values below every scale and beyond the largest one, on the borders between two
    codes and between two scales, with infinities and NaN (in k and v; not rotated)."""
    torch = _torch()
    D, page, NKV = 64, 16, 2
    x = torch.randn(9, 2 * NKV * D)
    x[0] = 0
    x[1] *= 1e-9
    x[2] *= 6e4
    x[3, ::32] = 7.0 * 2 ** 3
    x[3, 1::32] = 5 * 2 ** 3
    x[4, ::32] = 7.0
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    x[4, 1:25] = torch.cat([ties, -ties, ties * 0.996])
    x[5, 5] = float("inf")
    x[5, 200] = float("nan")
    x[6, 40] = -float("inf")
    x[7, ::32] = 7.0 * (1 + 2 ** -7)   # just beyond a scale's largest
    x[8] *= 2.0 ** -24
    run_append(act, act, D, 1, NKV, page, [9], [0], rot=0, norm=False, layers=1, layer=0,
               change=lambda q: q[:, D:].copy_(x))


# ---- values read back ---------------------------------------------------------------
@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("page,D,NKV", [(16, 64, 1), (16, 128, 3), (32, 128, 2), (64, 64, 5), (256, 128, 1)])
def test_dequant(page, D, NKV, out):
    """All codes under all the scales that append writes, and NaN; all pages and a list of them."""
    torch = _torch()
    g = torch.Generator().manual_seed(1)
    P, L = 7, 2
    pages = []
    for is_v in (False, True):
        code = torch.randint(0, 16, (L, P, NKV, page, D), generator=g)
        scale = torch.randint(104, 142, (L, P, NKV, page, D // 32), generator=g)
        pages.append(mx_ref.pack(code, torch.where(scale == 141, 255, scale), is_v))
    c = paged.kv_cache(pages[0].cuda(), pages[1].cuda(), head_dim=D)
    for ids in (None, [3, 0, -1, 6, 3, P, 2 ** 31 - 1]):
        n = P if ids is None else len(ids)
        o = [torch.full((n, NKV, page, D), 7.0, dtype=TYPES[out], device="cuda") for _ in range(2)]
        paged.kv_dequant(c, 1, *o, pages=None if ids is None else ints(ids))
        for t, b, is_v in zip(o, pages, (False, True)):
            want = mx_ref.values(b[1], page, D, is_v)
            if ids is not None:
                want = torch.stack([want[i] if 0 <= i < P else torch.zeros_like(want[0]) for i in ids])
            assert torch.equal(t.cpu().double().nan_to_num(1e30), want.nan_to_num(1e30))
    few = [torch.empty((2, NKV, page, D), dtype=TYPES[out], device="cuda") for _ in range(2)]
    paged.kv_dequant(c, 0, *few)
    assert torch.equal(few[1].cpu().double().nan_to_num(1e30), mx_ref.values(pages[1][0, :2], page, D, True).nan_to_num(1e30))


@pytest.mark.parametrize("out", ACTS)
@pytest.mark.parametrize("page,D,NKV", [(16, 64, 3), (16, 128, 2), (32, 64, 1), (32, 128, 2), (64, 64, 1), (64, 128, 4), (128, 64, 2),
                                        (256, 64, 1), (256, 128, 2)])
def test_dequant_of_many_pages(page, D, NKV, out):
    """Enough rows for several of them a thread; a list of pages with invalid ones, and all pages."""
    torch = _torch()
    g = torch.Generator().manual_seed(page + D)
    n = 32768 // (page * NKV) + 3
    P = n + 2
    pages, want = [], []
    for is_v in (False, True):
        code = torch.randint(0, 16, (1, P, NKV, page, D), generator=g)
        scale = torch.randint(104, 142, (1, P, NKV, page, D // 32), generator=g)
        pages.append(mx_ref.pack(code, torch.where(scale == 141, 255, scale), is_v))
        want.append(mx_ref.values(pages[-1][0], page, D, is_v).nan_to_num(1e30))
    c = paged.kv_cache(pages[0].cuda(), pages[1].cuda(), head_dim=D)
    ids = torch.randint(0, P, (n,), generator=g)
    ids[5], ids[7], ids[n - 1] = -1, P, 2 ** 31 - 1
    there = (ids >= 0) & (ids < P)
    for list_ in (ids, None):
        o = [torch.full((n, NKV, page, D), 7.0, dtype=TYPES[out], device="cuda") for _ in range(2)]
        paged.kv_dequant(c, 0, *o, pages=None if list_ is None else ints(ids.tolist()))
        for t, w in zip(o, want):
            w = w[:n] if list_ is None else torch.where(there[:, None, None, None], w[torch.where(there, ids, 0)], 0.0)
            assert torch.equal(t.cpu().double().nan_to_num(1e30), w)


# ---- attention ----------------------------------------------------------------------
def fill_seen(L, P, NKV, page, D, table, kv, g):
    """Pools of 0xFF with random rows at every sequence's positions: bytes, and the values they hold."""
    torch = _torch()
    out = []
    for is_v in (False, True):
        code, scale = mx_ref.unpack(empty_pool(L, P, NKV, page, D), page, D, is_v)
        for s, n in enumerate(kv):
            for p in range(n):
                pg = page_of(table, s, p, page, P)
                if pg >= 0:
                    c, e = mx_ref.blocks(torch.randn(L, NKV, D, generator=g))
                    code[:, pg, :, p % page], scale[:, pg, :, p % page] = c, e
        out.append((code, scale))
    return out


def tolerance(o, spread, size, ta, V, keys):
    """attention_tolerance, and what it leaves out, which shows where the large probabilities meet values that
    are 0: probabilities, scaled by 2^14, are sums of halves, whose least step is 2^-24, so each is off by up to
    2^-25 besides: 2^-39 of the row's largest, which the sum of all is at least; times |V| of up to `keys` keys."""
    big = float(V[_torch().isfinite(V)].abs().max()) if V.numel() else 0.0
    return attention_tolerance(o, spread, size, ta, _torch().float16) + keys * big * 2.0 ** -39


def run_attention(act, D, NQ, NKV, page, q_lens, past, window=0, sinks=0, scale=0.0, pad=0, layers=1, layer=0, spoil=None,
                  spoil_pool=None, wide=0, peak=1.0, seed=0, max_q=0, max_kv=0):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    kv = [n + p for n, p in zip(q_lens, past)]
    table, P = make_table([max(n, 0) for n in kv], page, g, spare=1)
    ta = TYPES[act]
    (kc, ks), (vc, vs) = fill_seen(layers, P, NKV, page, D, table, kv, g)
    if spoil:
        spoil(table, P)
    if spoil_pool:
        spoil_pool(ks, vs, table, kv)
    st = starts(q_lens)
    rows = st[-1] + pad
    Q = (peak * torch.randn(rows, NQ * D + wide, generator=g)).to(ta)
    q = Q.cuda()[:, :NQ * D].unflatten(1, (NQ, D))
    out = torch.full((rows, NQ, D), 7.0, dtype=ta, device="cuda")
    c = paged.kv_cache(mx_ref.pack(kc, ks, False).cuda(), mx_ref.pack(vc, vs, True).cuda(), head_dim=D)
    paged.attn_paged(c, layer, make_batch(q_lens, kv, table, rows, max_q=max_q, max_kv=max_kv), q, out, window=window,
                     sinks=sinks, scale=scale)
    got = out.cpu().double()
    K, V = mx_ref.unblock(kc, ks), mx_ref.unblock(vc, vs)
    ref = attention(K, V, layer, st, kv, table, Q[:, :NQ * D].unflatten(1, (NQ, D)), window, sinks, scale)
    for t in range(rows):
        if t not in ref:
            assert bool((got[t] == 7.0).all()), t
            continue
        o, spread, size = ref[t]
        tol = tolerance(o, spread, size, ta, V, max(kv))
        fine = torch.isfinite(o)   # a row that sees a NaN is not finite there
        bad = torch.where(fine, ~((got[t] - o).abs() <= tol), torch.isfinite(got[t]))
        assert not bool(bad.any()), (t, float((got[t] - o).abs().max()), float(tol.min()))
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("heads,kv", [(4, 1), (4, 4), (6, 2), (8, 1), (16, 1), (7, 1), (40, 2)])
def test_attention_single_tokens(act, D, heads, kv):
    """A decode step: ragged lengths from one position on, one sequence without a new token, one without
    any position."""
    run_attention(act, D, heads, kv, 16, [1, 1, 1, 0, 1, 1], [0, 30, 31, 5, 100, 290])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("heads,kv,D", [(4, 2, 64), (6, 2, 128), (8, 1, 128), (5, 5, 64)])
def test_attention_chunks(act, heads, kv, D):
    """Chunks and single tokens in one batch, rows behind the last sequence."""
    run_attention(act, D, heads, kv, 32, [70, 1, 3, 17, 0, 129], [0, 77, 5, 200, 9, 1], pad=4)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_page_sizes(page):
    for act in ACTS:
        run_attention(act, 64, 4, 2, page, [1, 40, 90], [300, 60, 0], layers=2, layer=1)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (16, 0), (17, 4), (64, 1), (100, 33), (64, 64), (63, 70),
                                          (5, 1000), (1000, 4)])
def test_attention_windows(window, sinks):
    for act in ("f32", "bf16"):
        run_attention(act, 64, 4, 2, 16, [1, 1, 37, 100], [299, 3, 250, 60], window=window, sinks=sinks)


@pytest.mark.parametrize("act", ACTS)
def test_attention_long_context(act):
    """Contexts split over many workgroups, single tokens and a chunk."""
    run_attention(act, 128, 4, 1, 64, [1, 2], [4000, 9])
    run_attention(act, 64, 4, 1, 64, [33], [3000])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("q,heads,kv,past", [(9, 4, 1, 700), (17, 8, 4, 2300), (40, 4, 1, 5000), (33, 6, 2, 1100)])
def test_attention_chunks_split_over_the_positions(act, q, heads, kv, past):
    run_attention(act, 64, heads, kv, 64, [q, 1], [past, 900])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("act", ACTS)
def test_attention_drafts(act, wide):
    """Rows around the 16 and the 32 that a sequence of few rows has at most, in batches that may hold little
    and more than 256 MiB of keys and values (wide tables)."""
    def widen(table, P):
        for r in table:
            r.extend([-1] * 900)
    for window in (0, 150):
        run_attention(act, 64, 16, 8, 256, [1, 4, 5, 8, 9, 16, 17], [300, 20, 0, 511, 300, 100, 250], window=window,
                      spoil=widen if wide else None)


@pytest.mark.parametrize("wide", [0, 20, 100, 900])
@pytest.mark.parametrize("act", ACTS)
def test_attention_longer_drafts(act, wide):
    """Rows around the 48 and the 64 that a sequence of few rows has at most in short batches, and the same in batches
    that may hold more (tables up to every limit)."""
    def widen(table, P):
        for r in table:
            r.extend([-1] * wide)
    run_attention(act, 64, 16, 8, 256, [24, 25, 32, 33, 1, 3], [300, 20, 0, 511, 250, 600], spoil=widen)
    run_attention(act, 128, 32, 8, 64, [12, 13, 16, 17], [70, 5, 100, 200], window=90, sinks=3, spoil=widen)


def test_attention_bounds_leave_out_what_lies_beyond():
    """Lengths above max_q and max_kv: as over 16-bit pages, what lies beyond is left out."""
    torch = _torch()
    g = torch.Generator().manual_seed(2)
    q_lens, kv = [1, 60, 2], [90, 70, 200]
    table, P = make_table(kv, 16, g)
    (kc, ks), (vc, vs) = fill_seen(1, P, 2, 16, 64, table, kv, g)
    Q = torch.randn(63, 4, 64, generator=g).half()
    out = torch.full((63, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    c = paged.kv_cache(mx_ref.pack(kc, ks, False).cuda(), mx_ref.pack(vc, vs, True).cuda(), head_dim=64)
    paged.attn_paged(c, 0, make_batch(q_lens, kv, table, max_q=2, max_kv=100), Q.cuda(), out)
    o, spread, size = attention(mx_ref.unblock(kc, ks), mx_ref.unblock(vc, vs), 0, starts(q_lens), kv, table, Q)[0]
    assert bool(((out[0].cpu().double() - o).abs() <= attention_tolerance(o, spread, size, torch.float16, torch.float16)).all())
    assert bool((out[1:61] == 7.0).all())
    assert bool(torch.isfinite(out[61:]).all())


def rounds_only_its_output(o, spread, size, ta, V, keys):
    """tolerance() without the rounding of the probabilities: they are pairs of halves, each off by half a step of what
    it rounds, so what is left of them is half a step squared; then the one rounding of the output."""
    torch = _torch()
    tol = tolerance(o, spread, size, torch.float32, V, keys) + half_step(torch.float16) ** 2 * spread
    return tol + half_step(ta) * (o.abs() + tol) + least(ta)


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("D,heads,kv,q_lens,past", [
    (128, 32, 8, [1, 1, 1], [299, 999, 8]), (64, 8, 1, [1, 1], [2000, 3]), (64, 4, 2, [4, 3, 1], [70, 0, 500]),
    (64, 9, 1, [1, 1], [700, 40]), (128, 17, 1, [1], [900]), (64, 4, 1, [8, 3, 1], [700, 40, 500]),
    (64, 16, 8, [24, 1], [300, 9]),   # few rows
    (128, 4, 2, [70, 1, 3], [150, 77, 5]), (64, 6, 2, [129, 20], [10, 400]), (64, 4, 1, [33], [3000])])   # many rows
def test_attention_of_16_bit_rows_rounds_only_its_output(act, D, heads, kv, q_lens, past):
    """Scores near each other and values of alternating sign, whose average is small beside them, so that the rounding of
    the output hides no other; and random values."""
    torch = _torch()
    g = torch.Generator().manual_seed(D + heads)
    ta, page, kvl = TYPES[act], 64, [n + p for n, p in zip(q_lens, past)]
    table, P = make_table(kvl, page, g)
    K, V = (torch.randn(1, P, kv, page, D, generator=g) for _ in range(2))
    V[..., :D // 2] = torch.where(torch.arange(page) % 2 == 0, 1.0, -1.0)[:, None]
    T = sum(q_lens)
    Q = torch.randn(T, heads, D, generator=g).to(ta)
    out = torch.empty(T, heads, D, dtype=ta, device="cuda")
    c = paged.kv_cache(mx_ref.pool(K, False).cuda(), mx_ref.pool(V, True).cuda(), head_dim=D)
    paged.attn_paged(c, 0, make_batch(q_lens, kvl, table), Q.cuda(), out, scale=0.01)
    K, V = mx_ref.rounded(K), mx_ref.rounded(V)
    ref = attention(K, V, 0, starts(q_lens), kvl, table, Q, scale=0.01)
    for r in ref:
        o, spread, size = ref[r]
        assert bool(((out[r].cpu().double() - o).abs() <= rounds_only_its_output(o, spread, size, ta, V, max(kvl))).all()), r


@pytest.mark.parametrize("act,big,small,k_big,k_small", [("f16", 8, -14, -14, 8), ("bf16", 8, -24, -22, 13),
                                                         ("bf16", 8, -31, -22, 14), ("bf16", 8, -37, -22, 14)])
@pytest.mark.parametrize("heads,kv,q_lens,past", [(4, 1, [1, 1], [299, 8]), (32, 2, [1], [700]), (8, 4, [5, 1], [90, 40]),
                                                  (4, 2, [70, 1], [30, 77])])
def test_attention_of_rows_with_far_apart_elements(heads, kv, q_lens, past, act, big, small, k_big, k_small):
    """Every other row of q has elements that are 2^32 to 2^45 times smaller than its others, where the keys are up to 2^36
    times larger, so that both count in the scores.  (fp16 rows: 2^22 times, as far as that type goes.)"""
    torch = _torch()
    g = torch.Generator().manual_seed(heads - small)
    ta, page, D, kvl = TYPES[act], 64, 64, [n + p for n, p in zip(q_lens, past)]
    table, P = make_table(kvl, page, g)
    K, V = (torch.randn(1, P, kv, page, D, generator=g) for _ in range(2))
    K[..., :32] *= 2.0 ** k_big
    K[..., 32:] *= 2.0 ** k_small
    T = sum(q_lens)
    Q = torch.randn(T, heads, D, generator=g)
    Q[:, 0::2, :32] *= 2.0 ** big
    Q[:, 0::2, 32:] *= 2.0 ** small
    Q[:, 1::2] *= 2.0 ** (small - 3)
    Q = Q.to(ta)
    scale = 2.0 ** -(big + k_big) / 4
    out = torch.empty(T, heads, D, dtype=ta, device="cuda")
    c = paged.kv_cache(mx_ref.pool(K, False).cuda(), mx_ref.pool(V, True).cuda(), head_dim=D)
    paged.attn_paged(c, 0, make_batch(q_lens, kvl, table), Q.cuda(), out, scale=scale)
    K, V = mx_ref.rounded(K), mx_ref.rounded(V)
    ref = attention(K, V, 0, starts(q_lens), kvl, table, Q, scale=scale)
    for r in ref:
        o, spread, size = ref[r]
        assert bool(((out[r].cpu().double() - o).abs() <= rounds_only_its_output(o, spread, size, ta, V, max(kvl))).all()), r


def test_attention_bad_pages_are_not_seen():
    def spoil(table, P):
        table[0][1] = -1                 # a hole
        table[1] = [P] * len(table[1])   # nothing left: rows of zeros
        table[2][0] = 2 ** 31 - 1
    for act in ACTS:
        run_attention(act, 64, 4, 2, 16, [1, 2, 60], [40, 30, 0], spoil=spoil)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("D,past,max_q", [(64, 90, 2), (64, 90, 80), (128, 700, 80), (128, 3000, 2)])
def test_attention_ends_at_max_kv(act, D, past, max_q):
    """Sequences longer than max_kv (here 100 below the longest): each token attends over the positions below it that
    there are up to max_kv, whether it stands there or behind; few rows and a chunk, in one range and in several."""
    torch = _torch()
    g = torch.Generator().manual_seed(past + D)
    q_lens = [2, 1, 2] if max_q == 2 else [2, 1, 80]
    kv = [past + 110, 40, past + 120]
    most = max(kv) - 100
    ta = TYPES[act]
    table, P = make_table(kv, 64, g)
    K, V = (torch.randn(1, P, 2, 64, D, generator=g) for _ in range(2))
    c = paged.kv_cache(mx_ref.pool(K, False).cuda(), mx_ref.pool(V, True).cuda(), head_dim=D)
    K, V = mx_ref.rounded(K), mx_ref.rounded(V)
    Q = torch.randn(sum(q_lens), 4, D, generator=g).to(ta)
    out = torch.full((sum(q_lens), 4, D), 7.0, dtype=ta, device="cuda")
    paged.attn_paged(c, 0, make_batch(q_lens, kv, table, max_q=max_q, max_kv=most), Q.cuda(), out)
    got = out.cpu().double()
    beyond = 0
    for t, s, p in tokens(starts(q_lens), kv):
        n = min(p + 1, most)
        beyond += p >= most
        o, spread, size = attention(K, V, 0, [0, 1], [n], [table[s]], Q[t:t + 1])[0]
        assert bool(((got[t] - o).abs() <= rounds_only_its_output(o, spread, size, ta, V, n) if act != "f32" else
                     (got[t] - o).abs() <= tolerance(o, spread, size, ta, V, n)).all()), (t, p)
    assert beyond >= 4


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("heads,kv", [(4, 1), (8, 1)])
def test_attention_nan_blocks_reach_only_rows_that_see_them(act, heads, kv):
    """NaN blocks of keys and values: later tokens' (causal), before the window, between sinks and window;
    rows that see one are not finite, the others exact.  Single tokens, drafts and chunks."""
    def nan(ks, vs, table, kvl):
        for s, p in ((0, 5), (1, 40), (2, 33), (2, 90)):
            pg = table[s][p // 16]
            vs[:, pg, :, p % 16, 0] = 255
        pg = table[2][3]
        ks[:, pg, :, 7, 1] = 255   # position 55: a key
    for window, sinks in ((0, 0), (20, 2), (7, 40)):
        run_attention(act, 64, heads, kv, 16, [1, 3, 70, 2], [40, 39, 30, 3], window=window, sinks=sinks, spoil_pool=nan)


@pytest.mark.parametrize("act", ACTS)
def test_attention_scales_and_peaks(act):
    """Sharp distributions, a scale of its own, q of very large and small elements, wide rows."""
    run_attention(act, 128, 4, 2, 16, [1, 20], [100, 60], peak=30.0, wide=24)
    run_attention(act, 64, 4, 2, 16, [1, 20], [100, 60], scale=1e-3, peak=100.0)
    run_attention(act, 64, 4, 2, 16, [2, 33], [100, 60], scale=3e4, peak=1e-5)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (3001, 150)])
def test_attention_long_loops(act, window, sinks):
    """More tiles a workgroup than one round of page lookups: 400 sequences of single tokens, and a chunk of
    enough blocks that none is split.  Sampled rows."""
    torch = _torch()
    g = torch.Generator().manual_seed(32)
    page, P, NQ, NKV, D = 256, 40, 16, 8, 64
    code, scale = [], []
    for is_v in (False, True):
        c, e = mx_ref.blocks(torch.randn(1, P, NKV, page, D, generator=g))
        code.append(c)
        scale.append(e)
    K, V = (mx_ref.unblock(c, e) for c, e in zip(code, scale))
    cache = paged.kv_cache(*(mx_ref.pack(c, e, v).cuda() for c, e, v in zip(code, scale, (False, True))), head_dim=D)
    for S, T, kv in ((400, 1, [int(n) for n in torch.randint(1, 30 * page + 1, (400,), generator=g)]), (1, 3200, [5800])):
        kv[:4] = [30 * page, 4097, 4128, 6145][:len(kv)] if S > 1 else kv
        table = [torch.randint(0, P, (30,), generator=g).tolist() for _ in range(S)]
        Q = torch.randn(S * T, NQ, D, generator=g).to(TYPES[act])
        out = torch.empty(S * T, NQ, D, dtype=TYPES[act], device="cuda")
        b = make_batch([T] * S, kv, table)
        paged.attn_paged(cache, 0, b, Q.cuda(), out, window=window, sinks=sinks)
        got = out.cpu().double()
        assert bool(torch.isfinite(got).all())
        for t, s, pos in tokens(starts([T] * S), kv):
            if t in (0, 1, 2, 3, 31, 32, 200, 399, 700, 2048, 3199):
                o, spread, size = attention(K, V, 0, [0, 1], [pos + 1], [table[s]], Q[t:t + 1], window, sinks)[0]
                tol = tolerance(o, spread, size, TYPES[act], V, pos + 1)
                assert bool(((got[t] - o).abs() <= tol).all()), (S, t, s, pos)


# ---- pages and rows moved -----------------------------------------------------------
@pytest.mark.parametrize("page,D,NKV", [(16, 64, 3), (16, 128, 1), (64, 128, 2)])
def test_copy_pages(page, D, NKV):
    torch = _torch()
    g = torch.Generator().manual_seed(3)
    K, V = (torch.randint(0, 256, (3, 9, NKV, paged.kv_head_bytes(page, D)), generator=g).to(torch.uint8) for _ in range(2))
    k, v = K.cuda(), V.cuda()
    paged.kv_copy_pages(paged.kv_cache(k, v, head_dim=D), [0, 5, 0], [8, 1, 3])
    for t in (K, V):
        t[:, [8, 1, 3]] = t[:, [0, 5, 0]]
    assert torch.equal(k.cpu(), K) and torch.equal(v.cpu(), V)


@pytest.mark.parametrize("page,D,NKV", [(16, 64, 2), (16, 128, 1), (64, 128, 2), (256, 64, 1)])
def test_compact(page, D, NKV):
    """Ragged sequences, one without kept rows, one that keeps all, one of several steps with far sources;
    rows without a page as source or destination stay."""
    torch = _torch()
    g = torch.Generator().manual_seed(4)
    L, lens = 2, [3, 70, 700, 17, 40]
    table, P = make_table(lens, page, g, spare=1)
    keep = [[2], [], sorted(torch.randperm(700, generator=g)[:333].tolist()), list(range(17)), list(range(9, 40))]
    K, V = (torch.randint(0, 256, (L, P, NKV, paged.kv_head_bytes(page, D)), generator=g).to(torch.uint8) for _ in range(2))
    k, v = K.cuda(), V.cuda()
    if page == 16:
        table[4][1] = -1
    paged.kv_compact(paged.kv_cache(k, v, head_dim=D), ints(table), ints(starts([len(x) for x in keep])), ints(sum(keep, [])))
    for got, t, is_v in ((k, K, False), (v, V, True)):
        code, scale = mx_ref.unpack(t, page, D, is_v)
        c, e = code.clone(), scale.clone()
        for s, rows in enumerate(keep):
            for j, p in enumerate(rows):
                a, b = page_of(table, s, p, page, P), page_of(table, s, j, page, P)
                if a >= 0 and b >= 0:
                    c[:, b, :, j % page], e[:, b, :, j % page] = code[:, a, :, p % page], scale[:, a, :, p % page]
        assert torch.equal(got.cpu(), mx_ref.pack(c, e, is_v))


# ---- graphs, streams, the dense model -------------------------------------------------
def _state(seed, act):
    torch = _torch()
    g = torch.Generator().manual_seed(seed)
    table, P = make_table([256, 256], 16, g)
    K, V = (mx_ref.pool(torch.randn(1, P, 2, 16, 64, generator=g), v).cuda() for v in (False, True))
    c, b = paged.kv_cache(K, V, head_dim=64), make_batch([1, 1], [70, 200], table, max_q=1, max_kv=256)
    x = torch.randn(2, 8, 64, generator=g).to(TYPES[act]).cuda()
    n = paged.attn_workspace_size(c, b, 4, x.dtype)
    return dict(c=c, b=b, x=x, K=K, V=V, q=torch.empty(2, 4, 64, device="cuda", dtype=x.dtype),
                out=torch.empty(2, 4, 64, device="cuda", dtype=x.dtype),
                kv=[torch.empty(P, 2, 16, 64, device="cuda", dtype=torch.float16) for _ in range(2)],
                ws=torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"), rope=paged.rope(64, 1e4))


def _step(s, stream=None):
    paged.kv_append(s["c"], 0, s["b"], s["x"][:, :4], s["x"][:, 4:6], s["x"][:, 6:], s["q"], rope=s["rope"], stream=stream)
    paged.attn_paged(s["c"], 0, s["b"], s["q"], s["out"], workspace=s["ws"], stream=stream)
    paged.kv_dequant(s["c"], 0, *s["kv"], stream=stream)
    return s["out"]


@pytest.mark.parametrize("act", ACTS)
def test_captured_steps_follow_the_lengths(act):
    """Two captures replayed in turn while the sequences grow, with eager work between, against eager calls."""
    torch = _torch()
    graphs = []
    for seed in (1, 2):
        s, e = _state(seed, act), _state(seed, act)
        _step(s)
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
            assert torch.equal(s["kv"][0], e["kv"][0])


def test_streams_and_repeats():
    torch = _torch()
    a, b = _state(3, "f32"), _state(3, "f32")
    want = _step(a).clone()
    for _ in range(3):
        assert torch.equal(_step(a), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    _step(b, stream=st)
    st.synchronize()
    assert torch.equal(b["out"], want) and torch.equal(b["K"], a["K"])


def test_offsets_beyond_32_bits():
    """Pages more than 4 GiB into a layer: prompts, single tokens, a page copied, rows moved and values read back as with
    the same pages at the front of a small cache."""
    torch = _torch()
    NQ, NKV, D, page = 16, 8, 128, 256
    big = 2 ** 32 // (NKV * paged.kv_head_bytes(page, D)) + 2
    assert big * NKV * paged.kv_head_bytes(page, D) > 2 ** 32
    rope, got = paged.rope(D, 1e6), []
    for P, ids in ((8, [0, 1, 2, 3, 4, 5]), (big + 8, [big, big + 1, 2, big + 5, big + 3, big + 7])):
        K, V = (torch.empty(1, P, NKV, paged.kv_head_bytes(page, D), dtype=torch.uint8, device="cuda") for _ in range(2))
        for t in (K, V):
            t[0, ids] = 255
        c, out = paged.kv_cache(K, V, head_dim=D), []
        table = [[ids[0], ids[1]], [ids[2], ids[3]]]
        g = torch.Generator().manual_seed(1)
        at = [0, 0]
        for new in ([300, 20], [1, 1], [5, 240]):
            at = [x + n for x, n in zip(at, new)]
            T = sum(new)
            x = torch.randn(T, NQ + 2 * NKV, D, generator=g).half().cuda()
            b = make_batch(new, at, table, max_q=max(new), max_kv=512)
            q, o = (torch.empty(T, NQ, D, dtype=torch.float16, device="cuda") for _ in range(2))
            paged.kv_append(c, 0, b, x[:, :NQ], x[:, NQ:NQ + NKV], x[:, NQ + NKV:], q, rope=rope)
            paged.attn_paged(c, 0, b, q, o)
            out += [q.cpu(), o.cpu()]
        paged.kv_copy_pages(c, [ids[1], ids[2]], [ids[4], ids[5]])
        paged.kv_compact(c, ints([[ids[4]], [ids[5]]]), ints([0, 3, 7]), ints([2, 5, 30, 0, 7, 8, 100]))
        kv = [torch.empty(6, NKV, page, D, device="cuda") for _ in range(2)]
        paged.kv_dequant(c, 0, *kv, pages=ints(ids))
        out += [t.cpu().nan_to_num(1e30) for t in kv]
        for t in (K, V):
            out.append(t[0, ids].cpu())
        got.append(out)
        del K, V, c
        torch.cuda.empty_cache()
    assert bool(torch.isfinite(got[0][1]).all())
    for x, y in zip(*got):
        assert torch.equal(x, y)


def test_two_steps_at_once():
    """Two caches' steps on two streams, none waiting for the other."""
    torch = _torch()
    sets = [_state(7, "f16"), _state(8, "bf16")]
    want = [_step(s).clone() for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in zip(sets, streams):
            _step(s, stream=st)
        torch.cuda.synchronize()
        for s, w in zip(sets, want):
            assert torch.equal(s["out"], w)


@pytest.mark.parametrize("act", ACTS)
def test_append_writes_over_its_own_q(act):
    torch = _torch()
    a, b = _state(9, act), _state(9, act)
    _step(a)
    q = b["x"][:, :4].clone()
    paged.kv_append(b["c"], 0, b["b"], q, b["x"][:, 4:6], b["x"][:, 6:], q, rope=b["rope"])
    torch.cuda.synchronize()
    assert torch.equal(q, a["q"]) and torch.equal(b["K"], a["K"]) and torch.equal(b["V"], a["V"])


@pytest.mark.parametrize("hidden", [256, 8448])
def test_dense_step_over_an_mxfp4_cache(oracle, hidden):
    """Prompts, chunks and single tokens of two sequences through the model's forward: the keys and values
    held are within a code's half step of the 64-bit ones, and the logits are those of the 64-bit forward
    that attends over the values held.  (hidden 8448: token by token, the decode step's path.)"""
    torch = _torch()
    from oracle.dense import DenseOracle, attention as attend, rmsnorm as rms, rope as turn, silu_mul
    from trailblaze_amd.dense import DenseConfig, SyntheticDense
    from conftest import rel_l2
    cfg = DenseConfig(n_layers=2, hidden=hidden, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=512, max_ctx=64)
    m = SyntheticDense(cfg, 3, keep_host=True)
    r = DenseOracle(oracle, cfg, m.host)
    page, P = 16, 12
    cache = m.paged_cache(P, page, mxfp4=True)
    for t in cache._keep:
        t.fill_(255)
    table = [[5, 0, 7], [2, 9, 4]]
    rng = np.random.default_rng(1)
    text = [rng.integers(0, 512, 40).tolist() for _ in range(2)]
    at = [0, 0]
    for new in ([20, 3], [1, 17], [1, 1], [2, 1]):
        logits = torch.empty(2, 512, device="cuda")
        toks = sum((text[s][at[s]:at[s] + n] for s, n in enumerate(new)), [])
        at = [a + n for a, n in zip(at, new)]
        m.step(cache, new, at, table, toks, logits)
        held = [[torch.empty(P, 2, page, 64, device="cuda") for _ in range(2)] for _ in range(2)]
        for l in range(2):
            paged.kv_dequant(cache, l, *held[l])
        for s in range(2):
            kv = [[t[table[s]].cpu().double().transpose(0, 1).reshape(2, 48, 64).numpy() for t in held[l]] for l in range(2)]
            xs = [r.lm[t].copy() for t in text[s][:at[s]]]
            for l, L in enumerate(r.layers):
                for p, x in enumerate(xs):
                    qkv = (L["wqkv"] @ rms(x, L["attn_norm"], cfg.norm_eps)).reshape(8, 64)
                    q = np.stack([turn(rms(v, L["q_norm"], cfg.norm_eps), p, cfg.rope_theta) for v in qkv[:4]])
                    k = np.stack([turn(rms(v, L["k_norm"], cfg.norm_eps), p, cfg.rope_theta) for v in qkv[4:6]])
                    # off by a code's half step, 2^E <= max / 3.5, and by the products' 1e-2
                    for h in range(2):
                        for got, y in ((kv[l][0][h, p], k[h]), (kv[l][1][h, p], qkv[6 + h])):
                            big = np.abs(y).reshape(2, 32).max(-1).repeat(32)
                            assert (np.abs(got - y) <= big * (1 / 3.5 + 0.03)).all()
                    xs[p] = x + L["wo"] @ attend(q, kv[l][0], kv[l][1], p + 1).reshape(-1)
                    gu = L["wgu"] @ rms(xs[p], L["ffn_norm"], cfg.norm_eps)
                    xs[p] = xs[p] + L["wdown"] @ silu_mul(gu[:512], gu[512:])
            want = r.lm @ rms(xs[-1], r.output_norm, cfg.norm_eps)
            assert rel_l2(logits[s].cpu().numpy(), want) <= 1e-2
