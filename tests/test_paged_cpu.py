"""CPU checks of include/tbq_kv.h: rotation plans against 64-bit formulas,
the page pool, and what the calls refuse (fake, aligned device pointers:
every check comes before the first HIP call, so nothing is dereferenced)."""
import ctypes as C
import random

import pytest

import trailblaze_amd as tb
from paged_ref import frequencies
from trailblaze_amd import paged

FAKE = 1 << 20


@pytest.mark.parametrize("rot", [8, 64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(scaling="linear", factor=4.0),
                                dict(scaling="yarn", factor=4.0, orig_ctx=32768),
                                dict(scaling="yarn", factor=32.0, orig_ctx=4096, beta_fast=16.0, beta_slow=2.0)])
def test_rope_plan(rot, kw):
    r = paged.rope(rot, 1e6, **kw)
    f, m = frequencies(rot, 1e6, **kw)
    assert r.rot_dim == rot and r.mscale == pytest.approx(m, rel=1e-15)
    assert list(r.freq)[:rot // 2] == pytest.approx(f.tolist(), rel=1e-13)   # a few 64-bit roundings


def test_rope_plan_factors():
    fac = [1.0 + 0.5 * j for j in range(32)]
    r = paged.rope(64, 5e5, layout="interleaved", factors=fac)
    assert list(r.freq)[:32] == pytest.approx(frequencies(64, 5e5, factors=fac)[0].tolist(), rel=1e-13)


@pytest.mark.parametrize("a", [(0, 0, 1e4, 0, 1.0, 0), (12, 0, 1e4, 0, 1.0, 0), (136, 0, 1e4, 0, 1.0, 0),
                               (64, 2, 1e4, 0, 1.0, 0), (64, 0, 1.0, 0, 1.0, 0), (64, 0, float("inf"), 0, 1.0, 0),
                               (64, 0, 1e4, 3, 1.0, 0), (64, 0, 1e4, 1, 0.5, 0), (64, 0, 1e4, 2, 4.0, 0),
                               (64, 0, 1e4, 1, float("nan"), 0)])
def test_rope_plan_refusals(a):
    r = paged.Rope()
    assert tb.lib().tbq_rope_init(C.byref(r), *a, 0.0, 0.0, None) == 0
    assert b"tbq_rope_init" in tb.lib().tbq_last_error()


# ---- pool --------------------------------------------------------------------
def test_pool_against_a_model():
    """Random calls against a plain list of holders."""
    rng = random.Random(4)
    n = 40
    pool, model = paged.PagePool(n), [0] * n
    for _ in range(2000):
        op, used = rng.randrange(4), [i for i in range(n) if model[i]]
        if op == 0:
            m = rng.randrange(0, 8)
            free = [i for i in range(n) if not model[i]]
            if m > len(free):
                with pytest.raises(tb.TbqError):
                    pool.alloc(m)
            else:
                got = pool.alloc(m)
                assert got == free[:m]
                for i in got:
                    model[i] = 1
        elif op == 1 and used:
            some = [rng.choice(used) for _ in range(3)]
            pool.share(some)
            for i in some:
                model[i] += 1
        elif op == 2 and used:
            some = [rng.choice(used) for _ in range(rng.randrange(1, 5))]
            if all(some.count(i) <= model[i] for i in some):
                pool.release(some)
                for i in some:
                    model[i] -= 1
            else:
                with pytest.raises(tb.TbqError):
                    pool.release(some)
        elif op == 3 and rng.random() < 0.2:
            most = rng.choice([0, 3, n])
            moves = pool.defrag(most)
            assert len(moves) <= most
            for s, d in moves:
                assert model[s] and not model[d] and d < s
                model[d], model[s] = model[s], 0
            if len(moves) < most:
                assert all(model[:sum(m > 0 for m in model)])
        assert pool.free_pages() == model.count(0)
        assert [pool.holders(i) for i in range(n)] == model
    pool.close()


@pytest.mark.parametrize("positions,page", [(0, 16), (1, 16), (16, 16), (40, 16), (48, 16)])
def test_pool_fork(positions, page):
    pool = paged.PagePool(8)
    n = -(-positions // page)
    mine = pool.alloc(n)
    child, copy = pool.fork(positions, page, mine)
    if positions % page:
        assert copy == (mine[-1], n) and child == mine[:-1] + [n]
        assert pool.holders(mine[-1]) == 1 and pool.holders(n) == 1
    else:
        assert copy is None and child == mine
    assert all(pool.holders(p) == 2 for p in mine[:positions // page])
    pool.release(child)
    pool.release(mine)
    assert pool.free_pages() == 8


@pytest.mark.parametrize("positions,page", [(-1, 16), (3, 0), (17, 16)])
def test_pool_fork_sizes(positions, page):
    with pytest.raises(ValueError):
        paged.PagePool(4).fork(positions, page, [0])


def test_pool_refusals():
    with pytest.raises(tb.TbqError):
        paged.PagePool(0)
    pool = paged.PagePool(2)
    mine = pool.alloc(2)
    with pytest.raises(tb.TbqError):        # no page for the partly filled one, and nothing shared
        pool.fork(17, 16, mine)
    assert [pool.holders(p) for p in (0, 1, 2, -1)] == [1, 1, -1, -1]
    for bad in ([2], [-1], [0, 0]):
        with pytest.raises(tb.TbqError):
            pool.release(bad)
    with pytest.raises(tb.TbqError):
        pool.share([5])
    assert pool.defrag(4) == [] and pool.free_pages() == 0


# ---- refusals ------------------------------------------------------------------
def cache(**kw):
    d = dict(n_layers=2, n_pages=8, n_kv_heads=2, page_size=16, head_dim=128, type=1, k=FAKE, v=FAKE)
    d.update(kw)
    return paged.KvCache(*[d[n] for n, _ in paged.KvCache._fields_])


def batch(**kw):
    d = dict(n_seqs=2, n_tokens=3, max_pages=4, max_q=0, max_kv=0, q_start=FAKE, kv_len=FAKE, page_table=FAKE)
    d.update(kw)
    return paged.KvBatch(*[d[n] for n, _ in paged.KvBatch._fields_])


def refused(ok, words):
    assert ok == 0
    msg = tb.lib().tbq_last_error().decode()
    assert words in msg, msg


CACHES = [(dict(type=0), "cache type"), (dict(type=12), "cache type"), (dict(head_dim=96), "head_dim"),
          (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(n_layers=0), "layers"),
          (dict(n_pages=0), "pages"), (dict(n_kv_heads=0), "kv heads"), (dict(k=None), "null or misaligned"),
          (dict(v=FAKE + 8), "null or misaligned")]
BATCHES = [(dict(n_seqs=-1), "sequences"), (dict(n_tokens=-1), "tokens"), (dict(max_pages=0), "pages"),
           (dict(max_q=-1), "max_q"), (dict(q_start=None), "null batch"), (dict(page_table=None), "null batch")]


def append(c, b, layer=0, heads=4, rope=None, in_type=1, q=FAKE, qs=512, k=FAKE, ks=256, v=FAKE, vs=256, q_type=1,
           q_out=2 * FAKE, qn=None):
    return tb.lib().tbq_kv_append(C.byref(c), layer, C.byref(b), heads, None if rope is None else C.byref(rope), qn, None,
                                  1e-6, None, in_type, q, qs, k, ks, v, vs, q_type, q_out, None)


def attn(c, b, layer=0, heads=4, q_type=1, q=FAKE, qs=512, out=FAKE, window=0, sinks=0, scale=0.0, ws=FAKE,
         wsb=1 << 40):
    return tb.lib().tbq_attn_paged(C.byref(c), layer, C.byref(b), heads, q_type, q, qs, out, window, sinks, scale, ws,
                                   wsb, None)


@pytest.mark.parametrize("kw,words", CACHES)
def test_cache_refusals(kw, words):
    c, b = cache(**kw), batch()
    refused(append(c, b), words)
    refused(attn(c, b), words)
    one = (C.c_int * 1)(0)
    refused(tb.lib().tbq_kv_copy_pages(C.byref(c), one, one, 1, None), words)
    refused(tb.lib().tbq_kv_compact(C.byref(c), 1, FAKE, 4, FAKE, FAKE, None), words)
    assert tb.lib().tbq_attn_paged_workspace_size(C.byref(c), C.byref(b), 4, 1) == 0


@pytest.mark.parametrize("kw,words", BATCHES)
def test_batch_refusals(kw, words):
    refused(append(cache(), batch(**kw)), words)
    refused(attn(cache(), batch(**kw)), words)


@pytest.mark.parametrize("kw,words", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(in_type=30), "in_type"), (dict(in_type=12), "in_type"),
    (dict(q_type=0), "q_type"), (dict(q_type=30), "q_type"), (dict(q=None), "go together"), (dict(q_out=None), "go together"),
    (dict(heads=0), "n_heads"), (dict(k=None), "null k or v"), (dict(v=FAKE + 2), "misaligned"), (dict(q=FAKE + 8), "misaligned"),
    (dict(qn=FAKE + 4), "misaligned"), (dict(ks=260), "strides"), (dict(vs=128), "shorter"), (dict(qs=504), "shorter"),
    (dict(q_out=FAKE, qs=1024), "q_out is q"), (dict(in_type=0, q_out=FAKE), "q_out is q"),
    (dict(rope=paged.Rope(12, 0, 1.0)), "rot_dim"), (dict(rope=paged.Rope(136, 0, 1.0)), "rot_dim"),
    (dict(rope=paged.Rope(64, 7, 1.0)), "rope layout")])
def test_append_refusals(kw, words):
    refused(append(cache(), batch(), **kw), words)


def test_append_rotation_longer_than_the_head():
    refused(append(cache(head_dim=64), batch(), rope=paged.rope(128, 1e4)), "rot_dim")


@pytest.mark.parametrize("kw,words", [
    (dict(layer=2), "layer"), (dict(heads=3), "n_heads"), (dict(heads=0), "n_heads"), (dict(q_type=30), "q_type"),
    (dict(window=-1), "window"), (dict(sinks=-1), "sinks"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(q=None), "null"), (dict(out=FAKE + 8), "misaligned"), (dict(qs=500), "q_stride"),
    (dict(qs=256), "q_stride")])
def test_attention_refusals(kw, words):
    refused(attn(cache(), batch(), **kw), words)


def test_attention_f32_needs_an_f16_cache():
    refused(attn(cache(type=30), batch(), q_type=0), "q_type")


@pytest.mark.parametrize("src,dst,words", [([0], [8], "pair 0"), ([-1], [1], "pair 0"), ([0, 1], [2, 2], "written twice"),
                                           ([0, 1], [1, 2], "read and written"), ([3], [3], "read and written")])
def test_copy_refusals(src, dst, words):
    a = lambda v: (C.c_int * len(v))(*v)   # noqa: E731
    refused(tb.lib().tbq_kv_copy_pages(C.byref(cache()), a(src), a(dst), len(src), None), words)


def test_compact_refusals():
    c = cache()
    refused(tb.lib().tbq_kv_compact(C.byref(c), -1, FAKE, 4, FAKE, FAKE, None), "sequences")
    refused(tb.lib().tbq_kv_compact(C.byref(c), 1, FAKE, 0, FAKE, FAKE, None), "pages")
    refused(tb.lib().tbq_kv_compact(C.byref(c), 1, None, 4, FAKE, FAKE, None), "null")


def test_nothing_to_do_is_done():
    """Empty batches and lists, without a device."""
    c = cache()
    for b in (batch(n_seqs=0), batch(n_tokens=0)):
        assert append(c, b) == 1 and attn(c, b) == 1
    assert tb.lib().tbq_kv_copy_pages(C.byref(c), None, None, 0, None) == 1
    assert tb.lib().tbq_kv_compact(C.byref(c), 0, None, 4, None, None, None) == 1


# ---- the dense step ----------------------------------------------------------------
def _dense():
    from trailblaze_amd import formats as fm
    from trailblaze_amd.dense import DenseLayer, DenseModel
    layers = (DenseLayer * 2)()
    for L in layers:
        for name in ("attn_norm", "q_norm", "k_norm", "ffn_norm", "wqkv", "wo", "wgu", "wdown"):
            setattr(L, name, FAKE)
    m = DenseModel(2, 512, 8, 2, 128, 512, 1000, 0, 1e-6, 1e6, fm.Q4_K, fm.Q6_K, FAKE, FAKE, FAKE, layers, None, None)
    m._layers = layers
    return m


def step(m, c, n_new=(3, 1), kv_len=(20, 1), table=((0, 1), (2, -1)), tokens=(1, 2, 3, 4), rope=None, window=0, sinks=0,
         logits=FAKE, ws=FAKE, wsb=1 << 40, n=None):
    a = lambda v: (C.c_int * len(v))(*v)   # noqa: E731
    return tb.lib().tbq_dense_step(C.byref(m), C.byref(c), len(n_new) if n is None else n, a(n_new), a(kv_len),
                                   a([p for r in table for p in r]), len(table[0]), a(tokens),
                                   None if rope is None else C.byref(rope), window, sinks, logits, ws, wsb, None)


@pytest.mark.parametrize("kw,words", [
    (dict(n=0), "sequences"), (dict(n=1025), "sequences"), (dict(n_new=(0, 1)), "new tokens"), (dict(kv_len=(2, 1)), "new tokens"),
    (dict(kv_len=(33, 1)), "new tokens"), (dict(table=((0, 8), (2, -1))), "page 8"), (dict(table=((-1, 1), (2, -1))), "page -1"),
    (dict(table=((-1, 1), (2, -1)), window=4, sinks=1), "page -1"), (dict(tokens=(1, 2, 3, 1000)), "token 1000"),
    (dict(tokens=(-1, 2, 3, 4)), "token -1"), (dict(window=-1), "window"), (dict(sinks=-2), "sinks"), (dict(logits=None), "null"),
    (dict(ws=FAKE + 8), "misaligned"), (dict(wsb=100), "workspace"), (dict(rope=paged.Rope(4, 0, 1.0)), "rope")])
def test_dense_step_refusals(kw, words):
    refused(step(_dense(), cache(), **kw), words)


@pytest.mark.parametrize("kw", [
    dict(table=((0, 1), (1, -1)), n_new=(17, 3), kv_len=(32, 3)),      # 15..31 and 0..2 of pages 0, 1 and 1
    dict(table=((0, 0), (1, -1)), n_new=(18, 1), kv_len=(32, 1)),      # 14 of a page and 14 of it again
    dict(table=((0, 1), (0, 1)), n_new=(1, 1), kv_len=(20, 20))])
def test_dense_step_refuses_two_tokens_in_one_row(kw):
    refused(step(_dense(), cache(page_size=16), tokens=(1,) * 20, **kw), "share row")


@pytest.mark.parametrize("kw", [
    dict(table=((0, 1), (0, 2)), n_new=(1, 1), kv_len=(20, 20)),       # a shared page that is read only
    dict(table=((0, 1), (0, 1)), n_new=(2, 1), kv_len=(20, 21))])      # rows 2, 3 and 4 of one page
def test_dense_step_takes_shared_pages(kw):
    refused(step(_dense(), cache(page_size=16), wsb=100, **kw), "workspace")   # what is checked last


@pytest.mark.parametrize("kw,words", [(dict(type=30), "cache type"), (dict(n_layers=3), "a cache of"), (dict(n_kv_heads=4), "a cache of"),
                                      (dict(head_dim=64), "a cache of"), (dict(page_size=48), "page_size")])
def test_dense_step_cache_refusals(kw, words):
    refused(step(_dense(), cache(**kw)), words)


def test_dense_step_workspace_serves_every_smaller_call():
    m, c = _dense(), cache(page_size=64)
    size = lambda *a: tb.lib().tbq_dense_step_workspace_size(C.byref(m), C.byref(c), *a)   # noqa: E731
    assert size(2, 1, 4) == 0 and size(1, 65537, 4) == 0 and size(1025, 2000, 4) == 0 and size(1, 1, 0) == 0
    rng = random.Random(3)
    for _ in range(2000):
        n = rng.randrange(1, 200)
        a = (n, rng.randrange(n, 3000), rng.randrange(1, 300))
        s = rng.randrange(1, a[0] + 1)
        b = (s, rng.randrange(s, a[1] + 1), rng.randrange(1, a[2] + 1))
        assert 0 < size(*b) <= size(*a), (a, b)


def test_attention_workspace_is_within_the_steps():
    """What tbq_attn_paged asks for a batch never exceeds the room that the step sets aside
    for one of that size: the step's size less that of the same step with hardly any room."""
    m = _dense()
    rng = random.Random(5)
    for _ in range(500):
        page, pages, n = 64, rng.randrange(1, 400), rng.randrange(1, 300)
        T = n if rng.random() < 0.5 else rng.randrange(n, 5000)
        c = cache(page_size=page)
        b = batch(n_seqs=n, n_tokens=T, max_pages=pages, max_q=0 if T > n else 1)
        need = tb.lib().tbq_attn_paged_workspace_size(C.byref(c), C.byref(b), 8, 1)
        assert need <= tb.lib().tbq_dense_step_workspace_size(C.byref(m), C.byref(c), n, max(T, 2), pages)


# ---- the built code ------------------------------------------------------------------
def test_built_copies_wait_for_lds_reads(tmp_path):
    """The chunk kernel's direct copies are issued with no LDS read outstanding (the walk of
    test_lds_copies.py over this kernel)."""
    import os
    import shutil
    import subprocess
    from test_lds_copies import OBJDUMP, _copies
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(tb.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    seen = {}
    for f in sorted(os.listdir(tmp_path)):
        if "amdgcn" in f and b"k_pg_attn_chunk" in (tmp_path / f).read_bytes():
            r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], cwd=tmp_path, check=True, capture_output=True, text=True)
            seen.update(_copies(r.stdout.splitlines()))
    assert any("k_pg_attn_chunk" in k for k in seen)
    assert {k: c for k, c in seen.items() if c[1]} == {}


# ---- workspaces made for a call ------------------------------------------------------
class _Allocations:
    """torch.empty and torch.cuda.stream on the CPU: the stream that each workspace is made on."""

    def __init__(self, monkeypatch):
        import torch
        self.current, self.made = [], []
        empty = torch.empty

        class on:
            def __init__(this, stream):
                this.stream = stream

            def __enter__(this):
                self.current.append(this.stream)

            def __exit__(this, *e):
                self.current.pop()

        def make(*a, device=None, **kw):
            self.made.append(self.current[-1] if self.current else None)
            return empty(*a, **kw)
        paged._init_torch()
        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(torch, "empty", make)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: None)
        monkeypatch.setattr(paged, "_device", lambda: -1)
        monkeypatch.setattr(paged, "_raw", lambda dev: 0)


class _Stream:
    device_index, cuda_stream = -1, 7


class _Lib:
    """Every call succeeds; workspace sizes are 1000 bytes."""

    def __getattr__(self, name):
        return (lambda *a: 1000) if name.endswith("workspace_size") else (lambda *a: 1)


@pytest.mark.parametrize("stream", [None, _Stream()])
def test_attention_makes_its_workspace_on_the_calls_stream(monkeypatch, stream):
    """The workspace comes from the pool of the stream that the kernels run on: a block of another
    stream's pool may still be in use there by what was freed before."""
    import torch
    q, out = torch.zeros(3, 4, 128).half(), torch.zeros(3, 4, 128).half()
    c, b = cache(), batch()
    c._dev = b._dev = -1
    allocations = _Allocations(monkeypatch)
    monkeypatch.setattr(paged, "lib", _Lib)
    paged.attn_paged(c, 0, b, q, out, stream=stream)
    assert allocations.made == [stream]


@pytest.mark.parametrize("stream", [None, _Stream()])
def test_step_grows_its_workspace_on_the_calls_stream(monkeypatch, stream):
    import torch
    from types import SimpleNamespace
    from trailblaze_amd import dense
    m = object.__new__(dense.SyntheticDense)
    m.cfg, m.model = SimpleNamespace(vocab=1000), _dense()
    c, logits = cache(), torch.zeros(1, 1000)
    c._dev = -1
    allocations = _Allocations(monkeypatch)
    monkeypatch.setattr(dense, "lib", _Lib)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: None)
    m.step(c, [1], [1], [[0]], [3], logits, stream=stream)
    m.step(c, [1], [2], [[0]], [4], logits)   # large enough: kept
    assert allocations.made == [stream]


@pytest.mark.parametrize("stream", [None, _Stream()])
def test_older_calls_make_their_workspaces_on_their_streams(monkeypatch, stream):
    """gemm, SyntheticDense.prefill and gguf.dense_prefill, as the paged calls."""
    import torch
    from trailblaze_amd import dense, gguf
    x = torch.zeros(4)
    allocations = _Allocations(monkeypatch)
    for mod in (tb, dense, gguf):
        monkeypatch.setattr(mod, "lib", _Lib)
        monkeypatch.setattr(mod, "_stream", lambda s=None: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: None)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    tb.gemm(x, 1, x, 2, 4, 256, x, stream=stream)
    m = object.__new__(dense.SyntheticDense)
    m.model = _dense()
    m.prefill([1, 2, 3], 0, x, stream=stream)
    gguf.dense_prefill(_dense(), [1, 2, 3], 0, x, stream=stream)
    assert allocations.made == [stream] * 3


def test_step_refuses_capture_on_a_named_stream(monkeypatch):
    """The stream that the step runs on is asked, not the current one."""
    import torch
    from types import SimpleNamespace
    from trailblaze_amd import dense
    m = object.__new__(dense.SyntheticDense)
    m.cfg, m.model = SimpleNamespace(vocab=1000), _dense()
    c, logits, stream = cache(), torch.zeros(1, 1000), _Stream()
    c._dev = -1
    allocations = _Allocations(monkeypatch)
    monkeypatch.setattr(dense, "lib", _Lib)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: allocations.current[-1:] == [stream])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: None)
    with pytest.raises(ValueError, match="capture"):
        m.step(c, [1], [1], [[0]], [3], logits, stream=stream)
    m.step(c, [1], [1], [[0]], [3], logits)


def test_steps_attention_has_its_room():
    """The bound that sets aside the attention's part of a step's workspace, whatever the batch: the call
    compares it with what the batch's plan writes before it looks at the whole workspace's size."""
    import numpy as np
    from trailblaze_amd import formats as fm
    from trailblaze_amd.dense import DenseModel
    rng = random.Random(6)
    ptr = lambda a: a.ctypes.data_as(C.c_void_p)   # noqa: E731
    m = _dense()
    for i in range(400):
        D, G = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        NKV = rng.choice([n for n in (1, 2, 4, 8, 16, 32) if n * G * D % 256 == 0])
        hidden = 8448 if i % 10 == 0 else 512    # beyond the batched rows: one token after the other
        mod = DenseModel(2, hidden, NKV * G, NKV, D, 512, 1000, 0, 1e-6, 1e6, fm.Q4_K, fm.Q6_K, FAKE, FAKE, FAKE,
                         m._layers, None, None)
        n = 1 if rng.random() < 0.2 else int(2 ** rng.uniform(0, 9))
        page = rng.choice([16, 64, 256])
        most = max(1, int(2 ** rng.uniform(0, min(14, 20 - np.log2(n)))))   # pages of a sequence
        q = rng.choice([1, rng.randrange(1, 40), rng.randrange(1, 1 + 6000 // n)])
        q = min(q, most * page)
        n_new = np.array([rng.randrange(1, q + 1) for _ in range(n)], np.int32)
        kv_len = np.array([rng.randrange(k, most * page + 1) for k in n_new], np.int32)
        kv_len[0] = most * page
        table = np.arange(n * most, dtype=np.int32).reshape(n, most)
        c = cache(n_pages=n * most, n_kv_heads=NKV, page_size=page, head_dim=D)
        if n * most * NKV * page > 0x7FFFFFFF:
            continue
        tokens = np.zeros(int(n_new.sum()), np.int32)
        ok = tb.lib().tbq_dense_step(C.byref(mod), C.byref(c), n, ptr(n_new), ptr(kv_len), ptr(table), most, ptr(tokens),
                                     None, rng.choice([0, 100]), 0, FAKE, FAKE, 100, None)
        refused(ok, "workspace 100 <")


# ---- numbers that a C int does not hold --------------------------------------------------
@pytest.mark.parametrize("bad", [2 ** 32, 2 ** 31, -2 ** 32, 1.0])
def test_numbers_beyond_an_int_are_refused(monkeypatch, bad):
    """None of them is taken as the number that its low 32 bits are."""
    import torch
    allocations = _Allocations(monkeypatch)
    monkeypatch.setattr(paged, "_device", lambda: -1)
    c, b = cache(), batch()
    c._dev = b._dev = -1
    pool = paged.PagePool(4)
    pool.alloc(2)
    monkeypatch.setattr(paged, "lib", _Lib)
    q, out = torch.zeros(3, 4, 128).half(), torch.zeros(3, 4, 128).half()
    kv = torch.zeros(3, 2, 128).half()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)   # noqa: E731
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for call in (lambda: paged.kv_copy_pages(c, [bad], [1]), lambda: paged.kv_copy_pages(c, [0, 1], [2, bad]),
                 lambda: paged.kv_batch(i32(0, 1), i32(1), i32(0)[None], bad),
                 lambda: paged.kv_batch(i32(0, 1), i32(1), i32(0)[None], 1, max_q=bad),
                 lambda: paged.kv_batch(i32(0, 1), i32(1), i32(0)[None], 1, max_kv=bad)):
        with pytest.raises((ValueError, TypeError)):
            call()
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: -1)
    if bad != 1.0:   # (an argument of a call: ctypes refuses a float itself)
        for call in (lambda: paged.attn_paged(c, bad, b, q, out), lambda: paged.attn_paged(c, 0, b, q, out, window=bad),
                     lambda: paged.attn_paged(c, 0, b, q, out, window=4, sinks=bad),
                     lambda: paged.kv_append(c, bad, b, q, kv, kv, out)):
            with pytest.raises(ValueError):
                call()
    monkeypatch.undo()
    for call in (lambda: pool.share([0, bad]), lambda: pool.release([bad]), lambda: pool.fork(16, 16, [bad]),
                 lambda: pool.alloc(bad), lambda: pool.defrag(bad), lambda: pool.holders(bad)):
        with pytest.raises((ValueError, TypeError)):
            call()
    assert [pool.holders(p) for p in range(4)] == [1, 1, 0, 0]


@pytest.mark.parametrize("kw", [dict(n_new=[2 ** 32 + 1]), dict(kv_len=[2 ** 32 + 1]), dict(page_table=[[2 ** 32]]),
                                dict(tokens=[2 ** 32 + 3]), dict(tokens=[3.5])])
def test_step_refuses_numbers_beyond_an_int(monkeypatch, kw):
    import numpy as np
    import torch
    from types import SimpleNamespace
    from trailblaze_amd import dense
    m = object.__new__(dense.SyntheticDense)
    m.cfg, m.model = SimpleNamespace(vocab=1000), _dense()
    c, logits = cache(), torch.zeros(1, 1000)
    c._dev = -1
    _Allocations(monkeypatch)
    monkeypatch.setattr(dense, "lib", _Lib)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: None)
    a = dict(n_new=[1], kv_len=[1], page_table=[[0]], tokens=[3])
    m.step(c, *a.values(), logits)
    for form in (lambda v: v, np.array):
        with pytest.raises(ValueError):
            m.step(c, *{**a, **{k: form(v) for k, v in kw.items()}}.values(), logits)
