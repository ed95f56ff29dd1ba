"""CPU checks of the MXFP4 cache: the reference blocks against the format's
definition, and what the calls refuse (fake, aligned device pointers: every check
comes before the first HIP call)."""
import ctypes as C

import pytest
import torch

import mx_ref
import trailblaze_amd as tb
from trailblaze_amd import paged

FAKE = 1 << 20


def test_blocks_are_the_nearest_values():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 64, generator=g).double() * 10.0 ** torch.randint(-6, 5, (500, 1), generator=g)
    code, scale = mx_ref.blocks(x)
    assert int(code.max()) <= 15 and int(scale.min()) >= 104 and int(scale.max()) <= 140
    y, s = mx_ref.unblock(code, scale), 2.0 ** (scale.double() - 127).repeat_interleave(32, -1)
    a = x.abs().unflatten(-1, (2, 32)).amax(-1).repeat_interleave(32, -1)
    inside = (a <= 7 * 2.0 ** 13)
    assert bool((a <= 7 * s)[inside].all()) and bool((a > 3.5 * s)[inside & (scale.repeat_interleave(32, -1) > 104)].all())
    err = (y - x).abs() / s
    assert bool((err <= torch.where(x.abs() / s > 4, 1.0, 0.5))[inside].all())
    for v in torch.unbind(mx_ref.GRID):   # no other value of the grid is nearer
        for sign in (1, -1):
            assert bool((err <= (sign * v - x / s).abs() + 1e-12).all())
    assert torch.equal(mx_ref.rounded(y), y)   # what is held is held again


def test_pack_and_unpack():
    g = torch.Generator().manual_seed(1)
    for page, D in ((16, 64), (32, 128)):
        for is_v in (False, True):
            code, scale = torch.randint(0, 16, (3, page, D), generator=g), torch.randint(0, 256, (3, page, D // 32), generator=g)
            pages = mx_ref.pack(code, scale, is_v)
            assert pages.shape[-1] == paged.kv_head_bytes(page, D)
            c, s = mx_ref.unpack(pages, page, D, is_v)
            assert torch.equal(c, code) and torch.equal(s, scale)


def test_head_bytes():
    f = tb.lib().tbq_kv_head_bytes
    assert f(39, 16, 64) == 16 * 34 and f(39, 256, 128) == 256 * 68 and f(1, 64, 128) == 64 * 256 and f(30, 16, 64) == 2048
    for bad in ((0, 16, 64), (38, 16, 64), (39, 8, 64), (39, 16, 96), (39, 0, 64), (39, 16, -64)):
        assert f(*bad) == 0
    with pytest.raises(ValueError):
        paged.kv_head_bytes(24, 128)
    with pytest.raises(ValueError):
        paged.kv_head_bytes(1 << 40, 128)


def cache(**kw):
    d = dict(n_layers=2, n_pages=8, n_kv_heads=2, page_size=16, head_dim=128, type=39, k=FAKE, v=FAKE)
    d.update(kw)
    return paged.KvCache(**d)


def batch(**kw):
    d = dict(n_seqs=1, n_tokens=1, max_pages=4, max_q=0, max_kv=0, q_start=FAKE, kv_len=FAKE, page_table=FAKE)
    d.update(kw)
    return paged.KvBatch(**d)


def refused(ok, words):
    assert ok == 0
    assert words in tb.lib().tbq_last_error().decode(), tb.lib().tbq_last_error()


@pytest.mark.parametrize("types,words", [((12, 1), "in_type"), ((39, 39), "in_type"), ((1, 0), "q_type"), ((1, 30), "q_type"),
                                         ((30, 1), "q_type"), ((0, 39), "q_type"), ((0, 12), "q_type")])
def test_append_refusals(types, words):
    in_type, q_type = types
    refused(tb.lib().tbq_kv_append(C.byref(cache()), 0, C.byref(batch()), 4, None, None, None, 1e-6, None, in_type, FAKE, 512,
                                   FAKE, 256, FAKE, 256, q_type, FAKE, None), words)


@pytest.mark.parametrize("q_type", [2, 12, 39, -1])
def test_attention_refusals(q_type):
    refused(tb.lib().tbq_attn_paged(C.byref(cache()), 0, C.byref(batch()), 4, q_type, FAKE, 512, FAKE, 0, 0, 0.0, FAKE, 1 << 30,
                                    None), "q_type")
    assert tb.lib().tbq_attn_paged_workspace_size(C.byref(cache()), C.byref(batch()), 4, q_type) == 0


def dequant(c, layer=0, pages=FAKE, n=3, out_type=1, k=FAKE, v=FAKE):
    return tb.lib().tbq_kv_dequant(C.byref(c), layer, pages, n, out_type, k, v, None)


@pytest.mark.parametrize("kw,words", [(dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(n=-1), "pages"),
                                      (dict(n=9, pages=None), "pages"), (dict(n=(1 << 20) + 1), "pages"),
                                      (dict(out_type=39), "out_type"), (dict(out_type=12), "out_type"), (dict(k=None), "null"),
                                      (dict(v=FAKE + 8), "misaligned")])
def test_dequant_refusals(kw, words):
    refused(dequant(cache(), **kw), words)


def test_dequant_of_other_caches_and_of_nothing():
    refused(dequant(cache(type=1)), "cache type")
    refused(dequant(cache(head_dim=96)), "head_dim")
    assert dequant(cache(), n=0, k=None, v=None) == 1


def test_python_cache_refusals():
    t = torch.zeros(1, 2, 1, 16 * 68, dtype=torch.uint8)
    for k, v, kw, words in ((t, t, dict(head_dim=128), "device"), (t[0], t[0], dict(head_dim=128), "alike"),
                            (t, t[:, :1], dict(head_dim=128), "alike"), (t[..., :500], t[..., :500], dict(head_dim=128), "alike")):
        with pytest.raises(ValueError, match=words):
            paged.kv_cache(k, v, **kw)


def test_steps_attention_has_its_room_over_mxfp4():
    """The bound that sets aside the attention's part of a step's workspace, whatever the batch: the call compares it with
    what the batch's plan writes before it looks at the whole workspace's size."""
    import random
    import numpy as np
    from test_paged_cpu import _dense
    from trailblaze_amd import formats as fm
    from trailblaze_amd.dense import DenseModel
    rng, m = random.Random(7), _dense()
    ptr = lambda a: a.ctypes.data_as(C.c_void_p)   # noqa: E731
    for i in range(400):
        D, G = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        NKV = rng.choice([n for n in (1, 2, 4, 8, 16, 32) if n * G * D % 256 == 0])
        hidden = 8448 if i % 10 == 0 else 512    # beyond the batched rows: one token after the other
        mod = DenseModel(2, hidden, NKV * G, NKV, D, 512, 1000, 0, 1e-6, 1e6, fm.Q4_K, fm.Q6_K, FAKE, FAKE, FAKE,
                         m._layers, None, None)
        n = 1 if rng.random() < 0.2 else int(2 ** rng.uniform(0, 10))
        page = rng.choice([16, 64, 256])
        most = max(1, int(2 ** rng.uniform(0, min(14, 20 - np.log2(n)))))   # pages of a sequence
        q = min(rng.choice([1, rng.randrange(1, 65), rng.randrange(1, 2 + 6000 // n)]), most * page)
        n_new = np.array([rng.randrange(1, q + 1) for _ in range(n)], np.int32)
        kv_len = np.array([rng.randrange(k, most * page + 1) for k in n_new], np.int32)
        kv_len[0] = most * page
        table = np.arange(n * most, dtype=np.int32).reshape(n, most)
        if n * most * NKV * page > 0x7FFFFFFF:
            continue
        c = cache(n_pages=n * most, n_kv_heads=NKV, page_size=page, head_dim=D)
        tokens = np.zeros(int(n_new.sum()), np.int32)
        ok = tb.lib().tbq_dense_step(C.byref(mod), C.byref(c), n, ptr(n_new), ptr(kv_len), ptr(table), most, ptr(tokens),
                                     None, rng.choice([0, 100]), 0, FAKE, FAKE, 100, None)
        refused(ok, "workspace 100 <")
