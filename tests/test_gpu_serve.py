"""GPU checks of a serving step's tables (tbq_kv_build_tables) and of the
verification of drafts (tbq_draft_verify) against serve_ref.py, which says the
same in lists and 64-bit numpy; and a run of them with the MXFP4 cache's append and
attention, as a server that drafts tokens uses them.  All outputs are whole
numbers and equal.  (A draw's border would have to lie within 1e-15 of the whole
to be decided differently; none of the seeded ones does.)"""
import numpy as np
import pytest

import serve_ref
import trailblaze_amd as tb
from paged_ref import TYPES
from trailblaze_amd import paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    print("device:", tb.init(), flush=True)


def _torch():
    import torch
    return torch


def ints(v):
    return _torch().tensor(v, dtype=_torch().int32, device="cuda")


NAMES = ("kv_len", "table", "free", "n_free", "q_start", "slots", "positions", "served")


def state(rng, seqs, page, past, spare, width=2, odd=False):
    """(kv_len, table, free, n_free) of a server's random moment."""
    lens = [int(rng.integers(0, past + 1)) for _ in range(seqs)]
    need = [-(-n // page) for n in lens]
    P = max(1, sum(need) + spare)
    ids = rng.permutation(P).tolist()
    W = max(need, default=0) + width
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + rng.integers(-5, P + 5, W - n).tolist())   # what lies behind does not count
        at += n
    free = ids[at:] + rng.integers(-5, P + 5, at).tolist()
    if odd and seqs > 4:
        lens[0], lens[1] = -3, W * page + 9
        for e in range(0, need[2], 2):
            table[2][e] = -1 if e % 4 else P
    return lens, table, free, spare


def build(page, rows, lens, drop, new, table, free, n_free, place="apart", optional=True):
    """One call; its outputs as lists."""
    torch = _torch()
    src = dict(kv_len=ints(lens), table=ints(table).view(len(lens), -1), free=ints(free), n_free=ints([n_free]))
    out = {k: torch.full_like(v, 77) for k, v in src.items()} if place == "apart" else src
    out = dict(out, q_start=ints([7] * (len(lens) + 1)))
    if optional:
        out.update(slots=ints([7] * rows), positions=ints([7] * rows), served=ints([7]))
    t = paged.kv_tables(page, src["kv_len"], ints(new), src["table"], src["free"], src["n_free"], q_start=out["q_start"],
                        n_drop=None if drop is None else ints(drop), kv_len_out=out["kv_len"], table_out=out["table"],
                        free_out=out["free"], n_free_out=out["n_free"], slots=out.get("slots"), positions=out.get("positions"),
                        served=out.get("served"))
    paged.kv_build_tables(t)
    return {k: v.tolist() for k, v in out.items()}


def check(page, rows, lens, drop, new, table, free, n_free, **kw):
    got = build(page, rows, lens, drop, new, table, free, n_free, **kw)
    want = serve_ref.tables(page, rows, lens, drop, new, table, free, n_free)
    for k in got:
        assert got[k] == want[k], k
    return want


@pytest.mark.parametrize("place", ["apart", "in place"])
@pytest.mark.parametrize("seqs,page,past,drop,new", [(1, 16, 0, 0, 1), (1, 256, 5000, 4, 5), (7, 16, 40, 8, 9), (64, 64, 900, 3, 4),
                                                     (300, 16, 60, 40, 30), (1024, 32, 50, 2, 3), (1025, 16, 33, 33, 2),
                                                     (2500, 16, 20, 1, 1), (3, 128, 10, 10, 4000)])
def test_tables(seqs, page, past, drop, new, place):
    rng = np.random.default_rng(seqs * 31 + past)
    lens, table, free, n = state(rng, seqs, page, past, 300 + seqs, width=2 + new // page)
    d, a = rng.integers(0, drop + 1, seqs).tolist(), rng.integers(0, new + 1, seqs).tolist()
    assert check(page, sum(a) + 5, lens, d, a, table, free, n, place=place)["served"] == [seqs]


@pytest.mark.parametrize("place", ["apart", "in place"])
@pytest.mark.parametrize("seqs,page,past,new", [(40, 16, 5000, 5000), (1030, 16, 200, 100), (1, 16, 150000, 150000), (65, 16, 1200, 1200)])
def test_tables_of_many_pages(seqs, page, past, new, place):
    """More pages given and taken in a call than the workgroup has threads, by some multiples."""
    rng = np.random.default_rng(seqs)
    lens, table, free, n = state(rng, seqs, page, past, seqs * (new // page + 1), width=2 + new // page)
    d, a = rng.integers(0, past + 1, seqs).tolist(), rng.integers(0, new + 1, seqs).tolist()
    assert check(page, sum(a), lens, d, a, table, free, n, place=place)["served"] == [seqs]
    check(page, sum(a), lens, [past] * seqs, a, table, free, 5, place=place)


@pytest.mark.parametrize("place", ["apart", "in place"])
@pytest.mark.parametrize("spare", [0, 1, 30])
def test_tables_not_all_served(spare, place):
    """Too few pages, rows or entries of a table: from the first sequence they do not suffice for on, none is
    served, and what was dropped is dropped."""
    for seqs in (9, 1500):
        rng = np.random.default_rng(spare + seqs)
        lens, table, free, n = state(rng, seqs, 16, 50, spare, width=3)
        d, a = rng.integers(0, 20, seqs).tolist(), rng.integers(0, 40, seqs).tolist()
        few = check(16, sum(a), lens, d, a, table, free, n, place=place)["served"][0]
        assert few < seqs or (seqs, spare) == (9, 30)   # (9 sequences do with 30 pages)
        check(16, sum(a) // 7, lens, d, a, table, free, n, place=place)
        a[seqs // 2] = 10 ** 6
        check(16, sum(a), lens, [0] * seqs, a, table, free, n, place=place) if sum(a) < 1 << 21 else None
        a[seqs // 2] = 2 ** 31 - 1
        check(16, 1000, lens, d, a, table, free, n, place=place)


@pytest.mark.parametrize("place", ["apart", "in place"])
def test_tables_of_odd_inputs(place):
    """Lengths below zero and beyond the table, drops of more than there is and of less than none, entries and
    lists that name no page, counts of free pages that cannot be."""
    rng = np.random.default_rng(5)
    lens, table, free, n = state(rng, 12, 16, 70, 40, width=4, odd=True)
    a = rng.integers(-2, 9, 12).tolist()
    check(16, 64, lens, rng.integers(-9, 99, 12).tolist(), a, table, free, n, place=place)
    check(16, 64, lens, None, a, table, free, n, place=place)
    check(16, 64, lens, [10 ** 9] * 12, a, table, free, n, place=place)
    for odd in (-4, 0, len(free), 10 ** 9):
        check(16, 64, lens, [2 ** 31 - 1, -2 ** 31] * 6, a, table, free, odd, place=place)


@pytest.mark.parametrize("place", ["apart", "in place"])
def test_tables_of_sequences_that_share_a_prefix(place):
    """Sequences whose first pages are the same ones drop and add behind them, and one leaves with length and drop 0: the
    shared pages stay where they are and never come to the list."""
    rng = np.random.default_rng(8)
    page, S, own = 16, 5, 4
    shared = [3, 0, 11]
    rest = [p for p in rng.permutation(12 + S * own).tolist() if p not in shared]
    lens = [48 + int(n) for n in rng.integers(1, 50, S)]
    table = [shared + rest[s * own:(s + 1) * own] + [-1] * 3 for s in range(S)]
    free, n = rest[S * own:] + [-1] * (12 + S * own - len(rest) + S * own), len(rest) - S * own
    for s, m in enumerate(lens):
        table[s][-(-m // page):] = [-1] * (10 - -(-m // page))
    for step in range(6):
        drop = [int(rng.integers(0, m - 48 + 1)) if m else 0 for m in lens]
        new = [int(rng.integers(0, 20)) if m else 0 for m in lens]
        want = check(page, 200, lens, drop, new, table, free, n, place=place)
        lens, table, free, n = want["kv_len"], want["table"], want["free"], want["n_free"][0]
        assert not set(shared) & set(free[:n])
        if step == 2:
            lens[1] = 0
        for s, m in enumerate(lens):
            assert table[s][:3] == shared or not m


def test_tables_without_rows_and_without_sequences():
    torch = _torch()
    rng = np.random.default_rng(6)
    lens, table, free, n = state(rng, 5, 32, 90, 20)
    got = build(32, 0, lens, [1] * 5, [3] * 5, table, free, n, optional=False)
    want = serve_ref.tables(32, 15, lens, [1] * 5, [3] * 5, table, free, n)
    for k in got:
        assert got[k] == want[k], k
    q, slots, served = ints([7]), ints([7, 7]), ints([7])
    t = paged.kv_tables(16, ints([]), ints([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), ints([2, 1, 0]), ints([2]),
                        q_start=q, slots=slots, served=served)
    paged.kv_build_tables(t)
    assert q.tolist() == [0] and slots.tolist() == [-1, -1] and served.tolist() == [0] and t._keep[4].tolist() == [2, 1, -1]


def test_captured_tables_go_on():
    """One capture, replayed in place: a server's steps one after the other, with eager work between."""
    torch = _torch()
    rng = np.random.default_rng(7)
    S, page, rows = 40, 16, 200
    lens, table, free, n = state(rng, S, page, 100, 80, width=6)
    t = dict(kv_len=ints(lens), table=ints(table), free=ints(free), n_free=ints([n]), drop=ints([0] * S), new=ints([1] * S),
             q_start=ints([0] * (S + 1)), slots=ints([0] * rows), positions=ints([0] * rows), served=ints([0]))
    h = paged.kv_tables(page, t["kv_len"], t["new"], t["table"], t["free"], t["n_free"], q_start=t["q_start"],
                        n_drop=t["drop"], slots=t["slots"], positions=t["positions"], served=t["served"])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        paged.kv_build_tables(h)
    for _ in range(6):
        d, a = rng.integers(0, 5, S).tolist(), rng.integers(0, 6, S).tolist()
        t["drop"].copy_(ints(d))
        t["new"].copy_(ints(a))
        gr.replay()
        want = serve_ref.tables(page, rows, lens, d, a, table, free, n)
        torch.cuda.synchronize()
        for k in NAMES:
            assert t[k].tolist() == want[k], k
        lens, table, free, n = want["kv_len"], want["table"], want["free"], want["n_free"][0]


# ---- verification ------------------------------------------------------------------
def run_verify(rng, n_rows, V, act="f32", draft=True, T="mixed", change=None, wide=0, near=0.5, good=0.6, u=None, starts=None, defined=True):
    """One call against the reference; returns it."""
    torch = _torch()
    S = len(n_rows)
    q_start = [0] + [int(x) for x in np.cumsum(n_rows)] if starts is None else starts
    R = sum(n_rows)
    base = rng.standard_normal((R, V + wide)).astype(np.float32) * 3
    logits = torch.tensor(base).to(TYPES[act])
    dl = torch.tensor(base + near * rng.standard_normal((R, V + wide)).astype(np.float32)).to(TYPES[act]) if draft else None
    temp = [float(rng.choice([0, 0.3, 1.0, 1.7])) for _ in range(S)] if T == "mixed" else T
    tokens = rng.integers(0, V, R)
    for r in range(1, R):   # often the best one of the row before
        if rng.random() < good:
            tokens[r] = int(logits[r - 1, :V].float().argmax())
    ua, un = rng.random(R).astype(np.float32), rng.random(S).astype(np.float32)
    if u is not None:
        ua[:], un[:] = u
    if change:
        change(logits, dl, tokens, ua, un)
    f32 = lambda v: torch.tensor(np.asarray(v, np.float32), device="cuda")   # noqa: E731
    out = [torch.full((S,), 77, dtype=torch.int32, device="cuda") for _ in range(3)]
    paged.draft_verify(ints(q_start), ints(tokens.tolist()), logits.cuda()[:, :V], f32(ua), f32(un), out[0], out[1], n_drop=out[2],
                       draft_logits=None if dl is None else dl.cuda()[:, :V],
                       temperature=None if temp is None else f32(temp))
    got = tuple(o.tolist() for o in out)
    if not defined:
        return got
    f64 = lambda t: t[:, :V].double().numpy()   # noqa: E731
    t64 = None if temp is None else np.asarray(temp, np.float32).astype(np.float64)
    want = serve_ref.verify(q_start, tokens, f64(logits), None if dl is None else f64(dl), t64, ua.astype(np.float64),
                            un.astype(np.float64))
    assert got == want
    return want


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 3, 17, 8191, 8192, 8193, 40009])
def test_verify(V, act, draft):
    rng = np.random.default_rng(V)
    for T in ("mixed", None):
        run_verify(rng, [1, 5, 0, 3, 9, 1, 2, 2, 2, 7], V, act, draft, T, wide=V % 3)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_rows_and_sequences(draft):
    """Many drafts (rounds of the workgroups' waves), many sequences, a vocabulary of more than 64 chunks."""
    rng = np.random.default_rng(1)
    got = run_verify(rng, [100, 3, 40, 17, 16, 18], 300, draft=draft, T=[0.0] * 6, good=1.0)
    assert got[0][0] == 99
    run_verify(rng, [100, 30, 33], 500, draft=draft, good=0.97, near=0.01)
    run_verify(rng, rng.integers(0, 4, 1500).tolist(), 100, draft=draft)
    run_verify(rng, [3, 1, 2], 600001, draft=draft)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("T", [[0.0] * 4, [-1.0] * 4, [float("nan")] * 4, [float("inf")] * 4, [1e-30] * 4, [1e30] * 4])
def test_verify_temperatures(T, draft):
    """Greedy ones (ties to the first), flat and sharp ones."""
    rng = np.random.default_rng(2)

    def ties(logits, dl, *_):
        logits[:, [30, 9000, 9001]] = 50.0
        if dl is not None:
            dl[:, [9000, 30]] = 50.0
    run_verify(rng, [4, 1, 6, 3], 10000, draft=draft, T=T, change=ties)
    run_verify(rng, [4, 1, 6, 3], 1000, draft=draft, T=T)


@pytest.mark.parametrize("u", [(0.0, 0.0), (1 - 2.0 ** -24, 1 - 2.0 ** -24), (0.0, 1 - 2.0 ** -24), (1.0, 1.0), (-3.0, float("inf")),
                               (float("nan"), float("nan"))])
@pytest.mark.parametrize("draft", [False, True])
def test_verify_edges_of_the_random_numbers(u, draft):
    rng = np.random.default_rng(3)
    run_verify(rng, [4, 1, 6, 3], 20000, draft=draft, u=u)
    run_verify(rng, [4, 1, 6, 3], 7, draft=draft, u=u)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_verify_infinite_and_missing_logits(act, draft):
    """-infinity (a grammar's mask), NaN, +infinity, rows of nothing else, drafts outside the vocabulary."""
    rng = np.random.default_rng(4)
    inf = float("inf")

    def odd(logits, dl, tokens, ua, un):
        for t in (logits,) if dl is None else (logits, dl):
            t[0:3, ::2] = -inf
            t[3] = -inf
            t[4, 5] = inf
            t[4, 8300] = inf
            t[5, 100:300] = float("nan")
            t[6] = float("nan")
            t[7, :8192] = -inf
            t[8, 8192:] = -inf
        if dl is not None:
            dl[9] = -inf
            logits[10] = -inf
        tokens[1], tokens[6], tokens[13], tokens[14], tokens[15] = 1, 200, -1, 9000, 2 ** 31 - 1
    for T in (None, [0.0] * 8, [0.7] * 8):
        run_verify(rng, [2, 2, 3, 2, 4, 1, 1, 3], 9000, act, draft, T, change=odd)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_verify_guesses_at_the_borders_of_chunks(act, draft):
    """Rejected guesses at the ends of the parts that a row is summed in, guesses that are the largest of their
    part or the only weight in it, and a part that has no other weight."""
    at = [0, 4095, 4096, 8191, 8192, 12287, 12288, 5, 5000]

    def change(logits, dl, tokens, ua, un):
        for i, x in enumerate(at):
            tokens[2 * i + 1] = x
            if i % 3 == 1:   # nearly all of the row's weight
                logits[2 * i, x] = 14.0
            if i % 3 == 2:   # the only weight of its part
                logits[2 * i, x // 4096 * 4096:(x // 4096 + 1) * 4096] = -float("inf")
                logits[2 * i, x] = 9.0
        tokens[-1] = 8190    # a row of nothing else, whose guess is outside its weight
        logits[-2] = -float("inf")
        logits[-2, 8189] = 1.0
    for T in (None, [0.05] * 10, [3.0] * 10):
        for seed in range(3):
            rng = np.random.default_rng(seed)
            run_verify(rng, [2] * 10, 12289, act, draft, T, change=change, u=(1 - 2.0 ** -24, float(rng.random())))


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("size", [1e-43, 1e-36, 1e-20, 1e20, 1e36])
def test_verify_sizes_of_logits_and_temperatures(size, draft):
    """Logits and temperatures far from 1, in proportion: the probabilities are ordinary ones."""
    def change(logits, dl, tokens, ua, un):
        for t in (logits,) if dl is None else (logits, dl):
            t *= size
    T = [float(np.float32(size * x)) for x in (0.5, 1.0, 2.0, 0.3)]
    run_verify(np.random.default_rng(11), [4, 1, 6, 3], 9000, draft=draft, T=T, change=change)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("T", [1e33, 1e35, 1e37, 3e38, float("inf")])
def test_verify_hot_temperatures_over_masks(T, draft):
    """Where every finite logit has weight, the lowest one too, masked ones (-infinity, NaN) still have none."""
    low = float(np.finfo(np.float32).min)

    def change(logits, dl, tokens, ua, un):
        for t in (logits,) if dl is None else (logits, dl):
            t[:, ::3] = -float("inf")
            t[:, 1::9] = low
            t[:, 2::27] = 1e35
            t[0:3, 50:6000] = float("nan")
            t[3, 4096:8192] = low
    run_verify(np.random.default_rng(12), [4, 1, 6, 3], 9000, draft=draft, T=[T] * 4, change=change)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_more_chunks_than_threads(draft):
    """A vocabulary of 537 parts."""
    run_verify(np.random.default_rng(8), [2, 1], 2200003, draft=draft, T=[0.8, 1.0], u=(1 - 2.0 ** -24, 0.75))


@pytest.mark.parametrize("V,at", [(2, (0, 1)), (9000, (3, 8200)), (4096, (4000, 4095))])
@pytest.mark.parametrize("draft", [False, True])
def test_verify_draws_next_to_borders(V, at, draft):
    """Two tokens with weight, 1 and w, of which the first ends within 1e-14 to 1e-13 of the random number: fp64's weights
    (off by a few 1e-16, and 2e-16 times the exponent) decide such a draw as the formula does."""
    torch = _torch()
    rng = np.random.default_rng(V)
    d, T = (rng.uniform(a, b, 20000000).astype(np.float32) for a, b in ((0.1, 3.0), (0.3, 2.0)))
    ends = 1 / (1 + np.exp(-d.astype(np.float64) / T)) * 2.0 ** 24
    near = np.abs(ends - np.rint(ends)) < 1.1e-13 * 2 ** 24
    d, T = d[near], T[near]
    ends = 1 / (1 + np.exp(-d.astype(np.longdouble) / T.astype(np.longdouble)))
    u = np.rint(ends * 2 ** 24) / 2 ** 24
    keep = (np.abs(ends - u) > 1e-14) & (np.abs(ends - u) < 1e-13)
    d, T, u, want = d[keep], T[keep], u[keep].astype(np.float32), np.where(u < ends, *at)[keep]
    S = len(d)
    assert S > 30 and len(set(want.tolist())) == 2
    logits = torch.full((S, V), -float("inf"))
    logits[:, at[0]], logits[:, at[1]] = 0.0, torch.tensor(-d)
    f32 = lambda v: torch.tensor(v, device="cuda")   # noqa: E731
    out = [torch.full((S,), 77, dtype=torch.int32, device="cuda") for _ in range(2)]
    l = logits.cuda()
    paged.draft_verify(ints(list(range(S + 1))), ints([0] * S), l, torch.zeros(S, device="cuda"), f32(u), out[0], out[1],
                       draft_logits=l if draft else None, temperature=f32(T))
    assert out[0].tolist() == [0] * S and out[1].tolist() == want.tolist()


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_verify_of_more_than_4096_parts(act, draft):
    """Hundreds of rows of several parts each and an odd vocabulary, in the launch of many parts: guesses at the parts' ends
    that are rejected, that are nearly all of their part or its only weight, greedy rows, masked rows, rows of nothing."""
    at = [0, 4095, 4096, 8191, 49151, 49152, 50256, 20000]
    inf = float("inf")

    def change(logits, dl, tokens, ua, un):
        R = len(tokens)
        ua[::4] = 1 - 2.0 ** -24
        for i, r in enumerate(range(0, R - 1, 3)):
            x = at[i % 8]
            tokens[r + 1] = x
            if i % 3 == 1:
                logits[r, x] = 14.0
            if i % 5 == 2:
                logits[r, x // 4096 * 4096:(x // 4096 + 1) * 4096] = -inf
                logits[r, x] = 9.0
        for t in (logits,) if dl is None else (logits, dl):
            t[1::17, ::2] = -inf
            t[2::23, :8192] = -inf
            t[4::29, 100:30000] = float("nan")
            t[7, :] = -inf
            t[8, 40000] = inf
    rng = np.random.default_rng(21)
    rows = rng.integers(1, 9, 80).tolist()
    assert sum(rows) * 13 >= 4096
    for T in ("mixed", [0.9] * 80):
        run_verify(rng, rows, 50257, act, draft, T, change=change, wide=3)


def test_verify_draft_equal_to_the_target():
    """p = q: nothing is rejected, whatever the numbers; where a draft has no weight at all, p is drawn from."""
    rng = np.random.default_rng(5)
    got = run_verify(rng, [9, 5], 9000, near=0.0, u=(1 - 2.0 ** -24, 0.3), T=None)
    assert got[0] == [8, 4]

    def never(logits, dl, tokens, ua, un):
        tokens[1] = 4
        logits[0, 4] = dl[0, 4] = -float("inf")
    assert run_verify(rng, [2], 300, near=0.0, T=None, change=never)[0] == [0]


def test_verify_rows_outside_the_call():
    """Starts below zero and beyond the rows: such a sequence has nothing, the others are as ever.  Falling
    ones: nothing defined, but no token outside the vocabulary."""
    run_verify(np.random.default_rng(6), [2, 3, 4], 100, starts=[0, 2, 5, 10])
    run_verify(np.random.default_rng(6), [2, 3, 4], 100, starts=[-1, 2, 5, 9])
    got = run_verify(np.random.default_rng(6), [2, 3, 4], 100, starts=[0, 5, 2, 9], defined=False)
    assert all(-1 <= v < 100 for v in got[1]) and got[0][1] == 0 and got[1][1] == -1 and got[2][1] == 0


def test_verify_is_captured_and_repeats():
    """Two captures with workspaces of their own, replayed in turn over new logits, against eager calls; another stream."""
    torch = _torch()
    g = torch.Generator().manual_seed(1)
    S, R, V = 6, 20, 9001
    q = ints([0, 3, 4, 9, 12, 19, 20])

    def make():
        s = dict(l=torch.empty(R, V, device="cuda"), d=torch.empty(R, V, device="cuda"), t=ints([0] * R),
                 ua=torch.empty(R, device="cuda"), un=torch.empty(S, device="cuda"), o=[ints([0] * S) for _ in range(3)])
        s["ws"] = torch.empty(paged.draft_verify_workspace_size(S, R, V, torch.float32, True), dtype=torch.uint8, device="cuda")
        return s

    def fill(s, seed):
        g.manual_seed(seed)
        l = 3 * torch.randn(R, V, generator=g)
        s["l"].copy_(l)
        s["d"].copy_(l + 0.3 * torch.randn(R, V, generator=g))
        s["t"].copy_(torch.cat([torch.zeros(1), l.argmax(-1)[:-1]]))
        s["ua"].copy_(torch.rand(R, generator=g))
        s["un"].copy_(torch.rand(S, generator=g))

    def call(s, stream=None):
        paged.draft_verify(q, s["t"], s["l"], s["ua"], s["un"], s["o"][0], s["o"][1], n_drop=s["o"][2], draft_logits=s["d"],
                           workspace=s["ws"], stream=stream)
    a, b, e = make(), make(), make()
    graphs = []
    for s in (a, b):
        fill(s, 0)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(s)
        graphs.append((gr, s))
    for seed in range(1, 5):
        for gr, s in graphs:
            fill(s, seed)
            fill(e, seed)
            gr.replay()
            call(e)
            torch.cuda.synchronize()
            assert [x.tolist() for x in s["o"]] == [x.tolist() for x in e["o"]]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    call(b, stream=st)
    st.synchronize()
    assert [x.tolist() for x in b["o"]] == [x.tolist() for x in e["o"]]


@pytest.mark.parametrize("draft", [False, True])
def test_verify_rows_beyond_32_bits(draft):
    """Rows more than 2^32 bytes apart, and 2^32 elements of 16 bits, as those of a small tensor."""
    torch = _torch()
    g = torch.Generator().manual_seed(9)
    V, R = 9001, 3
    for act, apart in (("f32", 2 ** 30 + 7), ("bf16", 2 ** 31 + 5)):
        ta = TYPES[act]
        near = [3 * torch.randn(R, V, generator=g) for _ in range(2)]
        near = [x.to(ta).cuda() for x in near]
        buf = torch.empty((R - 1) * apart + 2 * V + 3, dtype=ta, device="cuda")
        far = [buf.as_strided((R, V), (apart, 1), storage_offset=i * (V + 1)) for i in range(2)]
        for x, y in zip(far, near):
            x.copy_(y)
        tok = ints([0, int(near[0][0].float().argmax()), 17])
        u = torch.tensor([0.3, 0.999999, 0.5], device="cuda")
        res = []
        for x in (near, far):
            o = [ints([77]) for _ in range(3)]
            paged.draft_verify(ints([0, 3]), tok, x[0], u, u[:1], o[0], o[1], n_drop=o[2], draft_logits=x[1] if draft else None)
            res.append([t.item() for t in o])
        assert res[0] == res[1] and 0 <= res[0][1] < V
        del buf, far
        torch.cuda.empty_cache()


def test_two_verifications_and_tables_at_once():
    """Calls on two streams with workspaces and outputs of their own, none waiting for the other."""
    torch = _torch()
    g = torch.Generator().manual_seed(5)
    S, R, V = 8, 32, 50001
    q = ints(list(range(0, 33, 4)))
    l = 3 * torch.randn(R, V, generator=g).cuda()
    d = l + 0.5 * torch.randn(R, V, generator=g).cuda()
    tok = torch.cat([torch.zeros(1, device="cuda"), l.argmax(-1)[:-1].float()]).int()
    ua, un = torch.rand(R, generator=g).cuda(), torch.rand(S, generator=g).cuda()
    sets = []
    for dl in (d, None):
        n = paged.draft_verify_workspace_size(S, R, V, torch.float32, dl is not None)
        t = dict(kv_len=ints([100 * i for i in range(S)]), new=ints([4] * S), drop=ints([i % 3 for i in range(S)]),
                 table=ints([[64 * s + e for e in range(64)] for s in range(S)]), free=ints(list(range(512, 1024))), n_free=ints([500]),
                 q_start=ints([0] * (S + 1)), lens=ints([0] * S), out=ints([[0] * 64] * S), fo=ints([0] * 512), no=ints([0]))
        h = paged.kv_tables(16, t["kv_len"], t["new"], t["table"], t["free"], t["n_free"], q_start=t["q_start"], n_drop=t["drop"],
                            kv_len_out=t["lens"], table_out=t["out"], free_out=t["fo"], n_free_out=t["no"])
        sets.append((dl, torch.empty(n, dtype=torch.uint8, device="cuda"), [ints([77] * S) for _ in range(3)], t, h))

    def call(x, stream=None):
        dl, ws, o, t, h = x
        paged.draft_verify(q, tok, l, ua, un, o[0], o[1], n_drop=o[2], draft_logits=dl, workspace=ws, stream=stream)
        paged.kv_build_tables(h, stream=stream)
        return [*o, t["lens"], t["out"], t["fo"], t["no"], t["q_start"]]
    want = [[y.clone() for y in call(x)] for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for x, st in zip(sets, streams):
            call(x, stream=st)
        torch.cuda.synchronize()
    for x, w in zip(sets, want):
        for y, z in zip([*x[2], x[3]["lens"], x[3]["out"], x[3]["fo"], x[3]["no"], x[3]["q_start"]], w):
            assert torch.equal(y, z)


# ---- together ------------------------------------------------------------------------
def test_speculative_steps_on_the_device():
    """Tables, append, attention, logits, verification, and the drops into the next tables, without the host between: a
    model of one attention layer over an MXFP4 cache whose target is greedy gives, with drafts (right, wrong or
    sampled), the tokens that it gives one at a time."""
    torch = _torch()
    g = torch.Generator().manual_seed(3)
    S, NQ, NKV, D, V, page, P, drafts, most = 5, 4, 2, 64, 97, 16, 40, 3, 16
    emb = torch.randn(V, (NQ + 2 * NKV) * D, generator=g).cuda()
    head = torch.randn(NQ * D, V, generator=g).cuda()
    rope = paged.rope(D, 1e4)
    rng = np.random.default_rng(3)

    def server(k, text=None):
        """`most` tokens of each sequence, from steps of 1 + k tokens."""
        c = paged.kv_cache(*(torch.full((1, P, NKV, paged.kv_head_bytes(page, D)), 255, dtype=torch.uint8, device="cuda")
                             for _ in range(2)), head_dim=D)
        rows = S * (1 + k)
        t = dict(kv_len=ints([0] * S), table=ints([[-1] * 8] * S), free=ints(list(range(P))), n_free=ints([P]),
                 drop=ints([0] * S), new=ints([1 + k] * S), q_start=ints([0] * (S + 1)), slots=ints([0] * rows), served=ints([0]))
        h = paged.kv_tables(page, t["kv_len"], t["new"], t["table"], t["free"], t["n_free"], q_start=t["q_start"],
                            n_drop=t["drop"], slots=t["slots"], served=t["served"])
        b = paged.kv_batch(t["q_start"], t["kv_len"], t["table"], rows, max_q=1 + k)
        q, out = (torch.empty(rows, NQ, D, device="cuda") for _ in range(2))
        n_accept, nxt, ones = ints([0] * S), ints([0] * S), torch.ones(rows, device="cuda") * 0.5
        zero = torch.zeros(S, device="cuda")
        texts, cur = [[s + 1] for s in range(S)], [s + 1 for s in range(S)]
        while min(len(x) for x in texts) < most:
            toks = []
            for s in range(S):   # drafts: the true next tokens, spoilt at a random place
                guess = (text[s][len(texts[s]):len(texts[s]) + k] if text else [])[:k]
                guess = guess + [0] * (k - len(guess))
                if k and rng.random() < 0.6:
                    guess[rng.integers(0, k)] = int(rng.integers(0, V))
                toks += [cur[s]] + guess
            tok = ints(toks)
            paged.kv_build_tables(h)
            x = emb[tok.long()].view(rows, NQ + 2 * NKV, D)
            paged.kv_append(c, 0, b, x[:, :NQ], x[:, NQ:NQ + NKV], x[:, NQ + NKV:], q, rope=rope)
            paged.attn_paged(c, 0, b, q, out)
            logits = out.view(rows, -1) @ head
            paged.draft_verify(t["q_start"], tok, logits, ones, zero, n_accept, nxt, n_drop=t["drop"], temperature=zero)
            assert t["served"].item() == S and t["slots"].min().item() >= 0
            for s, (n, v) in enumerate(zip(n_accept.tolist(), nxt.tolist())):
                texts[s] += toks[s * (1 + k) + 1:s * (1 + k) + 1 + n] + [v]
                cur[s] = v
        # all pages are in a table or in the list, once
        torch.cuda.synchronize()
        held = [p for r in t["table"].tolist() for p in r if p >= 0] + t["free"].tolist()[:t["n_free"].item()]
        assert sorted(held) == list(range(P))
        return [x[:most] for x in texts]
    want = server(0)
    for k in (1, drafts):
        assert server(k, want) == want


def test_a_step_in_one_graph():
    """Tables, append, attention and verification, whose drops the next tables take, captured once and replayed, against the
    same calls made eagerly; the pages' bytes, the tables and the tokens of each step."""
    torch = _torch()
    S, NQ, NKV, D, V, page, P, k = 4, 8, 2, 64, 5000, 16, 48, 3
    rows, rope = S * (1 + k), paged.rope(64, 1e4)

    def server():
        s = dict(kv_len=ints([0] * S), table=ints([[-1] * 10] * S), free=ints(list(range(P))), n_free=ints([P]), drop=ints([0] * S),
                 new=ints([1 + k] * S), q_start=ints([0] * (S + 1)), slots=ints([0] * rows), accept=ints([0] * S), next=ints([0] * S),
                 tok=ints([0] * rows), served=ints([0]))
        s["K"], s["V"] = (torch.full((1, P, NKV, paged.kv_head_bytes(page, D)), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
        s["x"], s["q"], s["out"] = (torch.zeros(rows, n, D, device="cuda", dtype=torch.float16) for n in (NQ + 2 * NKV, NQ, NQ))
        s["logits"], s["draft"] = (torch.zeros(rows, V, device="cuda") for _ in range(2))
        s["ua"], s["un"] = torch.zeros(rows, device="cuda"), torch.zeros(S, device="cuda")
        h = paged.kv_tables(page, s["kv_len"], s["new"], s["table"], s["free"], s["n_free"], q_start=s["q_start"], n_drop=s["drop"],
                            slots=s["slots"], served=s["served"])
        c = paged.kv_cache(s["K"], s["V"], head_dim=D)
        b = paged.kv_batch(s["q_start"], s["kv_len"], s["table"], rows, max_q=1 + k, max_kv=160)
        ws = [torch.empty(max(n, 16), dtype=torch.uint8, device="cuda") for n in
              (paged.attn_workspace_size(c, b, NQ, torch.float16), paged.draft_verify_workspace_size(S, rows, V, torch.float32, True))]

        def step():
            paged.kv_build_tables(h)
            x = s["x"]
            paged.kv_append(c, 0, b, x[:, :NQ], x[:, NQ:NQ + NKV], x[:, NQ + NKV:], s["q"], rope=rope)
            paged.attn_paged(c, 0, b, s["q"], s["out"], workspace=ws[0])
            paged.draft_verify(s["q_start"], s["tok"], s["logits"], s["ua"], s["un"], s["accept"], s["next"], n_drop=s["drop"],
                               draft_logits=s["draft"], workspace=ws[1])
        return s, step
    (a, replayed), (e, eager) = server(), server()
    start = {n: t.clone() for n, t in a.items()}
    graph = torch.cuda.CUDAGraph()
    replayed()   # (what a first call sets up)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        replayed()
    for n, t in a.items():
        t.copy_(start[n])
    for r in range(8):
        g = torch.Generator().manual_seed(r)
        l = 3 * torch.randn(rows, V, generator=g)
        new = dict(x=torch.randn(rows, NQ + 2 * NKV, D, generator=g), logits=l, draft=l + 0.4 * torch.randn(rows, V, generator=g),
                   tok=torch.cat([torch.zeros(1), l.argmax(-1)[:-1].float()]), ua=torch.rand(rows, generator=g),
                   un=torch.rand(S, generator=g), new=torch.randint(1, 2 + k, (S,), generator=g))
        for s in (a, e):
            for n, t in new.items():
                s[n].copy_(t)
        graph.replay()
        eager()
        torch.cuda.synchronize()
        assert a["served"].item() == S
        for n in a:
            assert torch.equal(a[n], e[n]), (r, n)
