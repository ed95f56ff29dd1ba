"""CPU checks of a serving step's calls: what they refuse (fake, aligned device
pointers: every check comes before the first HIP call), workspace sizes, and the
reference's draws against the distribution that they are to have."""
import ctypes as C

import numpy as np
import pytest
import torch

import serve_ref
import trailblaze_amd as tb
from trailblaze_amd import paged

FAKE = 1 << 20


def refused(ok, words):
    assert ok == 0
    assert words in tb.lib().tbq_last_error().decode(), tb.lib().tbq_last_error()


def tables(**kw):
    d = dict(n_seqs=2, max_pages=8, page_size=16, n_pages=40, n_tokens=9, kv_len=FAKE, n_drop=FAKE, n_new=FAKE, page_table=FAKE,
             free_pages=FAKE, n_free=FAKE, kv_len_out=FAKE, page_table_out=FAKE, free_out=FAKE, n_free_out=FAKE, q_start=FAKE,
             slots=FAKE, positions=FAKE, served=FAKE)
    d.update(kw)
    return tb.lib().tbq_kv_build_tables(C.byref(paged.KvTables(**d)), None)


@pytest.mark.parametrize("kw,words", [
    (dict(page_size=24), "page_size"), (dict(page_size=0), "page_size"), (dict(n_seqs=-1), "sequences"),
    (dict(n_seqs=65536), "sequences"), (dict(max_pages=0), "pages"), (dict(n_pages=0), "pages"), (dict(n_tokens=-1), "tokens"),
    (dict(n_tokens=(1 << 30) + 1), "tokens"), (dict(max_pages=(1 << 26) + 1), "pages"),
    (dict(n_seqs=65535, max_pages=1 << 16), "pages"), (dict(n_pages=1 << 27), "pages"), (dict(q_start=None), "null"),
    (dict(kv_len=None), "null"), (dict(n_new=None), "null"), (dict(page_table=None), "null"), (dict(free_pages=None), "null"),
    (dict(n_free=None), "null"), (dict(kv_len_out=None), "null"), (dict(page_table_out=None), "null"),
    (dict(free_out=2 * FAKE), "go together"), (dict(n_free_out=2 * FAKE), "go together")])
def test_tables_refusals(kw, words):
    refused(tables(**kw), words)


def test_null_tables():
    refused(tb.lib().tbq_kv_build_tables(None, None), "null")


def verify(n_seqs=2, n_rows=5, vocab=100, type=0, q_start=FAKE, tokens=FAKE, logits=FAKE, stride=100, draft=FAKE, dstride=100,
           temperature=None, u_accept=FAKE, u_next=FAKE, n_accept=FAKE, next=FAKE, n_drop=None, ws=FAKE, ws_bytes=1 << 30):
    return tb.lib().tbq_draft_verify(n_seqs, n_rows, vocab, type, q_start, tokens, logits, stride, draft, dstride, temperature,
                                     u_accept, u_next, n_accept, next, n_drop, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,words", [
    (dict(n_seqs=-1), "sequences"), (dict(n_seqs=65536), "sequences"), (dict(n_rows=-1), "rows"), (dict(vocab=0), "rows"),
    (dict(vocab=(1 << 28) + 1), "rows"), (dict(type=39), "type"), (dict(type=12), "type"), (dict(n_rows=1 << 24), "rows"),
    (dict(q_start=None), "null"), (dict(tokens=None), "null"), (dict(logits=None), "null"), (dict(u_accept=None), "null"),
    (dict(u_next=None), "null"), (dict(n_accept=None), "null"), (dict(next=None), "null"), (dict(stride=99), "stride"),
    (dict(dstride=99), "stride"), (dict(logits=FAKE + 2), "misaligned"), (dict(draft=FAKE + 1, type=1), "misaligned"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=100), "workspace"), (dict(ws=FAKE + 8), "workspace")])
def test_verify_refusals(kw, words):
    refused(verify(**kw), words)


def test_verify_of_nothing_and_sizes():
    assert verify(n_seqs=0, q_start=None, ws=None) == 1
    size = tb.lib().tbq_draft_verify_workspace_size
    assert 0 < size(2, 5, 8192, 0, 0) < size(2, 6, 8192, 0, 0) < size(2, 6, 90000, 0, 0) < size(2, 6, 90000, 0, 1)
    assert size(1, 1, 1, 30, 0) >= 16
    assert size(2, 5, 0, 0, 0) == 0 and size(2, 5, 10, 39, 0) == 0


def test_python_refusals():
    i = lambda *n: torch.zeros(n, dtype=torch.int32)   # noqa: E731
    good = dict(kv_len=i(3), n_new=i(3), page_table=i(3, 4), free_pages=i(9), n_free=i(1), q_start=i(4))
    for kw, words in ((dict(), "one device"), (dict(kv_len=i(3).long()), "int32"), (dict(n_new=i(2)), "n_new"),
                      (dict(page_table=i(12)), "page_table"), (dict(q_start=i(3)), "q_start"), (dict(n_free=i(2)), "n_free"),
                      (dict(slots=i(5), positions=i(6)), "positions"), (dict(page_table=i(4, 3).t()), "page_table"),
                      (dict(free_out=i(8)), "free_out")):
        with pytest.raises(ValueError, match=words):
            paged.kv_tables(16, **{**good, **kw})


@pytest.mark.parametrize("certain", [False, True])
def test_reference_draws_the_targets_distribution(certain):
    """Two drafts of three tokens and the token behind, over all ways the random numbers can fall: the first
    token out has the target's probabilities.  (Acceptance and draw integrated on a fine grid of numbers.)"""
    rng = np.random.default_rng(0)
    logits, draft = rng.standard_normal((2, 3)), rng.standard_normal((2, 3))
    p, q = serve_ref.law(logits[0], 1.0), serve_ref.law(draft[0], 1.0)
    n, out = 200, np.zeros(3)
    grid = (np.arange(n) + 0.5) / n
    for x in range(3):
        for ua in grid:
            a, nxt, _ = serve_ref.verify([0, 2], [0, x], logits, None if certain else draft, None, [ua, 0.0], [0.0])
            chance = (p[x] if certain else q[x]) / n   # (a certain draft: any rule for choosing it will do)
            if a[0]:
                out[x] += chance
                continue
            for un in grid[::4]:
                out[serve_ref.verify([0, 2], [0, x], logits, None if certain else draft, None, [ua, 0.0], [un])[1][0]] += \
                    chance / (n / 4)
    # each of the grid's sums is off by at most a cell a border: 1 / n for acceptance, 4 / n for the draw, 3 tokens
    assert np.abs(out - p).max() <= 3 * (1 + 4) / n
