"""GPU parity of tbq_dense_step (the dense model's forward over a paged
cache for several sequences, include/tbq_kv.h) against the float64 oracle of
oracle/dense.py with a cache of its own per sequence: prompts, chunks and
single tokens in one call, forks, compaction, defragmentation, windows and
rotations, as a server would use them together.

Tolerances.  STEP_TOL: the matvecs' path with keys and values rounded to fp16
(half a step is 2^-11): values change the attention's output by at most
2^-11 of their size, keys the scores by 2^-11 |s|, |s| of 1 to 3 here, so a
layer's output by below 4 * 2^-11 = 2e-3 of the attention's share, two layers
4e-3.  BATCH_TOL: the fp16 products of the batched prefill (the same 1e-2 as
tbq_dense_prefill's)."""
import numpy as np
import pytest

import trailblaze_amd as tb
from conftest import rel_l2
from gpu_util import host
from trailblaze_amd import formats as fm
from trailblaze_amd import paged

pytestmark = pytest.mark.gpu
STEP_TOL, BATCH_TOL = 5e-3, 1e-2


@pytest.fixture(scope="module", autouse=True)
def _init():
    print("device:", tb.init(), flush=True)


def _model(oracle, seed=1, **kw):
    from oracle.dense import DenseOracle
    from trailblaze_amd.dense import DenseConfig, SyntheticDense
    base = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=512, max_ctx=512)
    base.update(kw)
    cfg = DenseConfig(**base)
    m = SyntheticDense(cfg, seed, keep_host=True)
    return m, Model(DenseOracle(oracle, cfg, m.host))


class Model:
    """DenseOracle's forward over a cache handed to it, with a rotation and a window."""

    def __init__(self, ref):
        self.ref, self.cfg = ref, ref.cfg
        self.freq, self.mscale, self.interleaved = None, 1.0, False
        self.window = self.sinks = 0

    def rope(self, x, pos):
        D = x.shape[-1]
        f = self.cfg.rope_theta ** (-2.0 * np.arange(D // 2) / D) if self.freq is None else self.freq
        j, n = np.arange(len(f)), len(f)
        u, w = (2 * j, 2 * j + 1) if self.interleaved else (j, j + n)
        c, s = np.cos(pos * f) * self.mscale, np.sin(pos * f) * self.mscale
        y = x.copy()
        y[..., u], y[..., w] = x[..., u] * c - x[..., w] * s, x[..., u] * s + x[..., w] * c
        return y

    def decode(self, cache, token, rng=None):
        """Appends the token to cache = [K, V], each [layers][positions] of [kv heads][D].  rng: every
        operand that the batched path holds in fp16 is off by half a step, 2^-11, up or down at
        random: weights by that of the largest of their 32 (the GEMM's Q4_K form of them), others by
        that of themselves."""
        off = lambda x: x if rng is None else x * (1 + 2.0 ** -11 * rng.choice([-1.0, 1.0], x.shape))   # noqa: E731

        def mul(W, h):
            if rng is not None:
                big = np.abs(W).reshape(len(W), -1, 32).max(-1, keepdims=True)
                W = W + (2.0 ** -11 * big * rng.choice([-1.0, 1.0], (len(W), W.shape[1] // 32, 32))).reshape(W.shape)
            return W @ off(h)
        from oracle.dense import attention, rmsnorm, silu_mul
        c, r = self.cfg, self.ref
        D, NQ, NKV = c.head_dim, c.n_heads, c.n_kv_heads
        x, pos = r.lm[token].copy(), len(cache[0][0])
        seen = [p for p in range(pos + 1) if not self.window or p > pos - self.window or p < self.sinks]
        for l, L in enumerate(r.layers):
            qkv = mul(L["wqkv"], rmsnorm(x, L["attn_norm"], c.norm_eps)).reshape(NQ + 2 * NKV, D)
            q = off(self.rope(np.stack([rmsnorm(v, L["q_norm"], c.norm_eps) for v in qkv[:NQ]]), pos))
            k = off(self.rope(np.stack([rmsnorm(v, L["k_norm"], c.norm_eps) for v in qkv[NQ:NQ + NKV]]), pos))
            cache[0][l].append(k)
            cache[1][l].append(off(qkv[NQ + NKV:].copy()))
            K, V = (np.stack([t[l][p] for p in seen], 1) for t in cache)
            x = x + mul(L["wo"], attention(q, K, V, len(seen)).reshape(-1))
            gu = mul(L["wgu"], rmsnorm(x, L["ffn_norm"], c.norm_eps))
            x = x + mul(L["wdown"], silu_mul(gu[:c.ffn], gu[c.ffn:]))
        return r.lm @ rmsnorm(x, r.output_norm, c.norm_eps)

    def magnified(self, tokens, want):
        """How far half a step in every fp16 operand takes this prompt's logits: the largest of 8 random
        ways.  Roundings are half a step at most and 0.58 of one on average, so theirs is below twice
        that."""
        err = 0.0
        for i in range(8):
            cache, rng = self.empty(), np.random.default_rng(i)
            for t in tokens:
                got = self.decode(cache, t, rng)
            err = max(err, rel_l2(got, want))
        return 2 * err

    def empty(self):
        return [[[] for _ in range(self.cfg.n_layers)] for _ in range(2)]


class Server:
    """Sequences over one paged cache and the oracle's caches beside them."""

    def __init__(self, m, model, n_pages=40, page=16):
        self.m, self.model, self.page = m, model, page
        self.cache, self.pool = m.paged_cache(n_pages, page), paged.PagePool(n_pages)
        for t in self.cache._keep:
            t.fill_(float("nan"))   # what nobody has written must not show
        self.pages, self.len, self.ref = [], [], []

    def add(self):
        self.pages.append([])
        self.len.append(0)
        self.ref.append(self.model.empty())
        return len(self.len) - 1

    def table(self, seqs, width=None):
        width = width or max(len(self.pages[s]) for s in seqs)
        return [self.pages[s] + [-1] * (width - len(self.pages[s])) for s in seqs]

    def step(self, work, tol, **kw):
        """work: {sequence: its new tokens}."""
        import torch
        seqs = list(work)
        for s in seqs:
            self.len[s] += len(work[s])
            need = -(-self.len[s] // self.page) - len(self.pages[s])
            if need > 0:
                self.pages[s] += self.pool.alloc(need)
        logits = torch.full((len(seqs), self.m.cfg.vocab), float("nan"), device="cuda")
        print("step", {s: (len(work[s]), self.len[s]) for s in seqs}, flush=True)
        self.m.step(self.cache, [len(work[s]) for s in seqs], [self.len[s] for s in seqs], self.table(seqs),
                    [t for s in seqs for t in work[s]], logits, **kw)
        got = host(logits)
        for i, s in enumerate(seqs):
            for t in work[s]:
                want = self.model.decode(self.ref[s], t)
            err = rel_l2(got[i], want)
            assert err <= tol, (s, err)
        self.check_rows(seqs, tol)

    def check_rows(self, seqs, tol):
        k, v = (host(t) for t in self.cache._keep)
        for s in seqs:
            for t, r in ((k, 0), (v, 1)):
                rows = [p for p in range(self.len[s]) if self.pages[s][p // self.page] >= 0]
                got = np.stack([t[:, self.pages[s][p // self.page], :, p % self.page] for p in rows])
                want = np.stack([np.stack([self.ref[s][r][l][p] for l in range(self.m.cfg.n_layers)]) for p in rows])
                assert rel_l2(got, want) <= tol


def _tokens(rng, n):
    return [int(t) for t in rng.integers(0, 512, n)]


def test_single_sequence_decode(oracle):
    m, model = _model(oracle)
    s, rng = Server(m, model), np.random.default_rng(1)
    a = s.add()
    for t in _tokens(rng, 20):
        s.step({a: [t]}, STEP_TOL)


@pytest.mark.parametrize("kw", [dict(head_dim=128, n_heads=8, n_kv_heads=2, hidden=512), dict(qtype_layers=fm.Q6_K),
                                dict(n_heads=8, n_kv_heads=1, qtype_layers=fm.GGML | fm.Q4_K)])
def test_prompts_and_tokens_in_one_call(oracle, kw):
    m, model = _model(oracle, seed=3, **kw)
    s, rng = Server(m, model), np.random.default_rng(2)
    a, b, c = s.add(), s.add(), s.add()
    s.step({a: _tokens(rng, 40), b: _tokens(rng, 1)}, BATCH_TOL)
    s.step({b: _tokens(rng, 17), c: _tokens(rng, 100), a: _tokens(rng, 1)}, BATCH_TOL)
    s.step({a: _tokens(rng, 1), b: _tokens(rng, 1), c: _tokens(rng, 1)}, BATCH_TOL)
    s.step({c: _tokens(rng, 1)}, BATCH_TOL)   # earlier rows came from the fp16 products


def test_fork_compact_and_defragment(oracle):
    """A served run: two prompts, a fork with its copied page, drafted tokens
    of which one branch stays, a sequence that ends, pages moved together."""
    import torch
    m, model = _model(oracle, seed=4)
    s, rng = Server(m, model), np.random.default_rng(3)
    a, b = s.add(), s.add()
    s.step({a: _tokens(rng, 37), b: _tokens(rng, 20)}, BATCH_TOL)
    c = s.add()
    s.pages[c], copy = s.pool.fork(s.len[a], s.page, s.pages[a])
    assert copy is not None
    paged.kv_copy_pages(s.cache, [copy[0]], [copy[1]])
    s.len[c], s.ref[c] = s.len[a], [[list(rows) for rows in t] for t in s.ref[a]]
    s.step({a: _tokens(rng, 1), b: _tokens(rng, 1), c: _tokens(rng, 1)}, BATCH_TOL)
    s.step({a: _tokens(rng, 6), c: _tokens(rng, 4)}, BATCH_TOL)          # drafts
    keep = [list(range(39)) + [40, 43], list(range(38)) + [41]]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    paged.kv_compact(s.cache, ints(s.table([a, c])), ints([0, 41, 80]), ints(keep[0] + keep[1]))
    for q, rows in zip((a, c), keep):
        s.len[q] = len(rows)
        s.ref[q] = [[[t[p] for p in rows] for t in side] for side in s.ref[q]]
        n = -(-s.len[q] // s.page)
        s.pool.release(s.pages[q][n:])
        s.pages[q] = s.pages[q][:n]
    s.check_rows([a, c], BATCH_TOL)
    s.pool.release(s.pages[b])
    moves = s.pool.defrag(40)
    assert moves
    paged.kv_copy_pages(s.cache, [x for x, _ in moves], [y for _, y in moves])
    to = dict(moves)
    for q in (a, c):
        s.pages[q] = [to.get(p, p) for p in s.pages[q]]
    s.step({c: _tokens(rng, 3), a: _tokens(rng, 2)}, BATCH_TOL)
    s.step({a: _tokens(rng, 1), c: _tokens(rng, 1)}, BATCH_TOL)


def test_window_with_freed_pages(oracle):
    m, model = _model(oracle, seed=5)
    model.window, model.sinks = 20, 3
    s, rng = Server(m, model), np.random.default_rng(4)
    a, b = s.add(), s.add()
    s.step({a: _tokens(rng, 70), b: _tokens(rng, 9)}, BATCH_TOL, window=20, sinks=3)
    s.pages[a][1] = s.pages[a][2] = -1    # positions 16..47: behind the window of 71 and on
    s.step({a: _tokens(rng, 1), b: _tokens(rng, 30)}, BATCH_TOL, window=20, sinks=3)
    s.step({a: _tokens(rng, 1)}, BATCH_TOL, window=20, sinks=3)
    with pytest.raises(tb.TbqError, match="page -1"):
        s.step({a: _tokens(rng, 1)}, BATCH_TOL)   # without a window it would see them


@pytest.mark.parametrize("layout,rot,scaling", [("interleaved", 64, "none"), ("half", 32, "yarn")])
def test_rotations(oracle, layout, rot, scaling):
    from paged_ref import frequencies
    m, model = _model(oracle, seed=6)
    kw = dict(factor=4.0, orig_ctx=64) if scaling == "yarn" else {}
    f, model.mscale = frequencies(rot, 1e4, scaling, **kw)
    model.freq, model.interleaved = f.numpy(), layout == "interleaved"
    s, rng = Server(m, model), np.random.default_rng(5)
    a, b = s.add(), s.add()
    rope = paged.rope(rot, 1e4, layout=layout, scaling=scaling, **kw)
    for t in _tokens(rng, 4):
        s.step({a: [t]}, STEP_TOL, rope=rope)
    s.step({a: _tokens(rng, 5), b: _tokens(rng, 33)}, BATCH_TOL, rope=rope)


def test_models_beyond_the_batched_rows(oracle):
    """hidden 8448: one token after the other on the decode step's matvecs."""
    m, model = _model(oracle, seed=7, n_layers=1, hidden=8448, ffn=256, vocab=512)
    assert not m.prefill_batched()
    s, rng = Server(m, model), np.random.default_rng(6)
    a, b = s.add(), s.add()
    s.step({a: _tokens(rng, 18), b: _tokens(rng, 2)}, STEP_TOL)
    s.step({a: _tokens(rng, 1), b: _tokens(rng, 1)}, STEP_TOL)


@pytest.mark.parametrize("n,vocab", [(300, 512), (9, 2064), (9, 514)])
def test_many_sequences(oracle, n, vocab):
    """More sequences than the 256 whose starts travel in one launch; an lm_head of several of the
    weight buffer's 1024 rows, the last part of 16; one that the product does not take (rows not a
    multiple of 4)."""
    m, model = _model(oracle, seed=8, n_layers=1, vocab=vocab)
    import torch
    cache = m.paged_cache(n)
    rng = np.random.default_rng(7)
    n_new = [1 + i % 3 for i in range(n)]
    toks = _tokens(rng, sum(n_new))
    logits = torch.empty(n, vocab, device="cuda")
    m.step(cache, n_new, n_new, [[i] for i in range(n)], toks, logits)
    got, at = host(logits), 0
    for i in range(n):
        ref = model.empty()
        mine = toks[at:at + n_new[i]]
        for t in mine:
            want = model.decode(ref, t)
        at += n_new[i]
        err = rel_l2(got[i], want)
        # a few of these prompts of two or three tokens magnify the roundings of their products
        # (synthetic weights whose rows have a mean: sums that nearly cancel)
        assert err <= BATCH_TOL or err <= model.magnified(mine, want), (i, err)


def test_step_is_reproducible_and_takes_other_streams(oracle):
    import torch
    m, _ = _model(oracle, seed=9)
    rng = np.random.default_rng(8)
    toks = _tokens(rng, 50)
    out = []
    for i in range(3):
        cache = m.paged_cache(8, 16)
        logits = torch.empty(2, 512, device="cuda")
        st = torch.cuda.Stream() if i == 2 else torch.cuda.current_stream()
        st.wait_stream(torch.cuda.current_stream())
        m.step(cache, [45, 5], [45, 5], [[4, 1, 7], [2, -1, -1]], toks, logits, stream=st)
        st.synchronize()
        out.append((host(logits), host(cache._keep[0]), host(cache._keep[1])))
    for o in out[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(out[0], o))


def test_step_refusals(oracle):
    """What the Python entry checks: logits on the cache's device, no capture (a replay would take the
    tokens and lengths of the captured call)."""
    import torch
    m, _ = _model(oracle)
    c = m.paged_cache(4, 16)
    logits = torch.empty(1, m.cfg.vocab, device="cuda")
    a = (c, [1], [1], [[0]], [3])
    with pytest.raises(ValueError, match="cpu"):
        m.step(*a, logits.cpu())
    m.step(*a, logits)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        try:
            with pytest.raises(ValueError, match="capture"):
                m.step(*a, logits)
        finally:
            g.capture_end()


def test_a_larger_workspace_changes_nothing():
    """The logits' product of eight and more sequences splits its sums by the call's shape alone: with the
    workspace that a call asks for and with one left from a longer prompt, the same bits.  Rows of 2048, 2048
    of them at a time, in 8 slices, where the layers' products take 4 or fewer rows."""
    import ctypes as C
    import torch
    from trailblaze_amd.dense import DenseConfig, SyntheticDense
    m = SyntheticDense(DenseConfig(n_layers=1, hidden=2048, n_heads=4, n_kv_heads=2, head_dim=64, ffn=1024, vocab=4128,
                                   max_ctx=16), 11)
    for n in (8, 16):
        cache = m.paged_cache(n, 16)
        logits = [torch.empty(n, m.cfg.vocab, device="cuda") for _ in range(2)]
        size = int(tb.lib().tbq_dense_step_workspace_size(C.byref(m.model), C.byref(cache), n, n, 1))
        for spare, o in zip((0, 64 << 20), logits):
            m._step_ws = torch.empty(size + spare, dtype=torch.uint8, device="cuda")
            m.step(cache, [1] * n, [1] * n, [[i] for i in range(n)], list(range(3, 3 + n)), o)
        assert torch.equal(*logits), n


def test_small_values_over_many_positions(oracle):
    """Values near the end of fp16: the attention's rows, averages of 500 of them, are an order of magnitude
    smaller and reach the o product scaled, as the contiguous prefill's do.  attn_norm of 2^-21 leaves values
    of 16 * 2^-21 = 7.6e-6 (rows of 256, weights N(0, 1); q and k are normalised), which the cache rounds to
    steps of 2^-24: off by 2.2e-3 (rms), and so are their averages.  Averages in steps of 2^-24 would be off
    by 3e-2 of themselves.  wo and the embedding are scaled so that the logits are what the attention adds."""
    import torch
    m, model = _model(oracle, seed=12, n_layers=1, qtype_layers=fm.F32, qtype_embd=fm.F32, norm_eps=1e-14, max_ctx=16)
    L, dev = model.ref.layers[0], m._keep[0]
    for name, f in (("attn_norm", 2.0 ** -21), ("wo", 2.0 ** 10), ("wdown", 2.0 ** -30)):
        L[name] = L[name] * f
        dev[name].view(torch.float32).mul_(f)
    model.ref.lm = model.ref.lm * 2.0 ** -20
    m.lm_head.view(torch.float32).mul_(2.0 ** -20)
    rng = np.random.default_rng(12)
    toks = _tokens(rng, 500)
    cache, logits, ref = m.paged_cache(8), torch.empty(1, 512, device="cuda"), model.empty()
    m.step(cache, [500], [500], [list(range(8))], toks, logits)
    for t in toks:
        want = model.decode(ref, t)
    err = rel_l2(host(logits)[0], want)
    print("error", err, flush=True)
    assert err <= BATCH_TOL


@pytest.mark.parametrize("qt", [fm.Q6_K, fm.Q4_K, fm.GGML | fm.Q4_K, fm.Q8_0, fm.F32])
@pytest.mark.parametrize("n,hidden", [(33, 256), (64, 2048)])
def test_logits_of_many_sequences_are_as_exact_as_of_few(n, hidden, qt):
    """The product that forms the logits of many sequences, against the matvecs on the same rows (what a
    vocabulary that is no multiple of 4 takes): each within the matvecs' 1e-5 of the formula."""
    import dataclasses
    import torch
    from trailblaze_amd.dense import DenseConfig, SyntheticDense
    m = SyntheticDense(DenseConfig(n_layers=1, hidden=hidden, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=2068,
                                   max_ctx=16, qtype_embd=qt), 13)
    cache, got = m.paged_cache(n, 16), []
    for vocab in (2068, 2066):
        m.model.vocab, m.cfg = vocab, dataclasses.replace(m.cfg, vocab=vocab)
        logits = torch.full((n, vocab), float("nan"), device="cuda")
        m.step(cache, [1] * n, [1] * n, [[i] for i in range(n)], list(range(5, 5 + n)), logits)
        got.append(host(logits))
    for i in range(n):
        assert rel_l2(got[0][i, :2066], got[1][i]) <= 2e-5, i


def test_logits_do_not_depend_on_their_address():
    """logits 4 bytes into an allocation: the same product, the same bits."""
    import torch
    from trailblaze_amd.dense import DenseConfig, SyntheticDense
    m = SyntheticDense(DenseConfig(n_layers=1, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=512,
                                   max_ctx=16), 14)
    cache, buf = m.paged_cache(40, 16), torch.empty(40 * 512 + 1, device="cuda")
    got = []
    for off in (0, 1):
        logits = buf[off:off + 40 * 512].view(40, 512)
        m.step(cache, [1] * 40, [1] * 40, [[i] for i in range(40)], list(range(40)), logits)
        got.append(host(logits))
    assert np.array_equal(*got)


@pytest.mark.parametrize("n,vocab,qt", [(300, 2068, fm.Q8_0), (40, 2068, fm.Q6_K), (9, 2068, fm.Q8_0), (9, 514, fm.Q6_K)])
def test_many_sequences_within_the_stated_bound(oracle, n, vocab, qt):
    """Weights without a mean (Q8_0 and Q6_K quants are symmetric), whose sums do not cancel against each
    other: the stated 1e-2 without exception; an lm_head in five parts of 512 rows, the last of 20."""
    import torch
    m, model = _model(oracle, seed=15, n_layers=1, vocab=vocab, qtype_layers=qt)
    cache, rng = m.paged_cache(n), np.random.default_rng(15)
    n_new = [1 + i % 3 for i in range(n)]
    toks = _tokens(rng, sum(n_new))
    logits = torch.empty(n, vocab, device="cuda")
    m.step(cache, n_new, n_new, [[i] for i in range(n)], toks, logits)
    got, at, errs = host(logits), 0, []
    for i in range(n):
        ref = model.empty()
        for t in toks[at:at + n_new[i]]:
            want = model.decode(ref, t)
        at += n_new[i]
        errs.append(rel_l2(got[i], want))
    print("errors", n, vocab, max(errs), float(np.mean(errs)), flush=True)
    assert max(errs) <= BATCH_TOL
