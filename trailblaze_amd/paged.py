"""The paged key/value cache of include/tbq_kv.h over torch tensors: append
with rotary positions, attention over the pages, page copies, compaction and
the host-side page pool.

A cache is two tensors [layers][pages][kv heads][page size][head dim] of
float16 or bfloat16, or [layers][pages][kv heads][bytes] of uint8 (MXFP4, 4.25
bits a value); a batch is int32 tensors on the same device.  Every call
checks its tensors (device, type, shape, strides) and raises TbqError or
ValueError before anything is launched; work goes to torch's current stream
unless ``stream`` names one.
"""
from __future__ import annotations

import ctypes as C
from array import array
from operator import index

from . import TbqError, _check, _stream, _workspace, lib

F32, F16, BF16, MXFP4 = 0, 1, 30, 39
ROPE_HALF, ROPE_INTERLEAVED = 0, 1
_LAYOUTS = {"half": ROPE_HALF, "interleaved": ROPE_INTERLEAVED}
_SCALINGS = {"none": 0, "linear": 1, "yarn": 2}


class KvCache(C.Structure):
    """Mirror of ``tbq_kv_cache``."""
    _fields_ = [("n_layers", C.c_int), ("n_pages", C.c_int), ("n_kv_heads", C.c_int), ("page_size", C.c_int),
                ("head_dim", C.c_int), ("type", C.c_int), ("k", C.c_void_p), ("v", C.c_void_p)]


class KvBatch(C.Structure):
    """Mirror of ``tbq_kv_batch``."""
    _fields_ = [("n_seqs", C.c_int), ("n_tokens", C.c_int), ("max_pages", C.c_int), ("max_q", C.c_int),
                ("max_kv", C.c_int), ("q_start", C.c_void_p), ("kv_len", C.c_void_p), ("page_table", C.c_void_p)]


class Rope(C.Structure):
    """Mirror of ``tbq_rope``."""
    _fields_ = [("rot_dim", C.c_int), ("layout", C.c_int), ("mscale", C.c_double), ("freq", C.c_double * 64)]


class KvTables(C.Structure):
    """Mirror of ``tbq_kv_tables``."""
    _fields_ = [(n, C.c_int) for n in ("n_seqs", "max_pages", "page_size", "n_pages", "n_tokens")] + \
        [(n, C.c_void_p) for n in ("kv_len", "n_drop", "n_new", "page_table", "free_pages", "n_free", "kv_len_out",
                                   "page_table_out", "free_out", "n_free_out", "q_start", "slots", "positions", "served")]


_torch, _raw, _device, _ids = None, None, None, {}
_INT = 1 << 31


def _init_torch():
    """torch, imported at the first use as everywhere in this package."""
    global _torch, _raw, _device
    if _torch is None:
        import torch
        _torch = torch
        # (torch's own functions behind current_stream and current_device, 3 and 0.3 us a call less)
        _raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _ids.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    return _torch


def _type_id(dtype):
    _init_torch()
    if dtype not in _ids:
        raise ValueError(f"{dtype}: float32, float16 or bfloat16")
    return _ids[dtype]


def _int(name, v):
    """v, where a C int holds it (ctypes would pass on its low 32 bits)."""
    v = index(v)
    if not -_INT <= v < _INT:
        raise ValueError(f"{name}: {v} is no 32-bit int")
    return v


def _c_ints(name, values):
    """A C array of a list of ints."""
    try:
        a = array("i", values)
    except OverflowError:
        raise ValueError(f"{name}: a number that is no 32-bit int") from None
    return (C.c_int * len(a)).from_buffer(a) if a else (C.c_int * 0)()


def _here(*owners):
    """The current device, whose stream the call takes: that of the cache and the batch."""
    _init_torch()
    cur = _device()
    for o in owners:
        if o._dev != cur:
            raise ValueError(f"tensors on device {o._dev}, current device is cuda:{cur}")
    return cur


def _to(stream, dev):
    """_stream, of the current device, which the tensors are on."""
    if stream is None:
        return _stream() if _raw is None else _raw(dev)
    if stream.device_index != dev:
        raise ValueError(f"stream on cuda:{stream.device_index}, tensors on cuda:{dev}")
    return _stream(stream)


def _on(name, t, dev):
    if t.get_device() != dev:
        raise ValueError(f"{name}: tensor on {t.device}, current device is cuda:{dev}")


def _ints(name, t, shape):
    if t.dtype != _init_torch().int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}")


def _heads(name, t, rows, n_heads, D, dev):
    """Elements between the rows of [rows][heads][D], whose heads lie side by side."""
    if t.shape != (rows, n_heads, D):
        raise ValueError(f"{name}: {(rows, n_heads, D)} expected, got {tuple(t.shape)}")
    if t.get_device() != dev:
        _on(name, t, dev)
    row, head, one = t.stride()
    if one != 1 or (n_heads > 1 and head != D):
        raise ValueError(f"{name}: the heads of a row must lie side by side")
    return row if rows > 1 else n_heads * D


def _flat(name, t, shape, dtype, dev):
    """The address of a contiguous tensor."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous {dtype} {shape} expected, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != dev:
        _on(name, t, dev)
    return t.data_ptr()


def _vec(name, t, n, dtype, dev):
    """_flat of n elements, or nothing (t None)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != n or t.dim() != 1 or not t.is_contiguous() or t.get_device() != dev:
        _flat(name, t, (n,), dtype, dev)
    return t.data_ptr()


def kv_head_bytes(page_size: int, head_dim: int, type_id: int = MXFP4) -> int:
    """Bytes of one kv head in a page of K (or of V): the last size of an MXFP4 cache's tensors."""
    n = int(lib().tbq_kv_head_bytes(type_id, _int("page_size", page_size), _int("head_dim", head_dim)))
    if n == 0:
        raise ValueError(f"no cache of type {type_id} has pages of {page_size} positions of {head_dim}")
    return n


def kv_cache(k, v, head_dim: int = 0) -> KvCache:
    """A ``tbq_kv_cache`` over two device tensors.  uint8 tensors [layers][pages]
    [kv heads][kv_head_bytes(page size, head_dim)] are an MXFP4 cache of head_dim."""
    _init_torch()
    mx = k.dtype == _torch.uint8
    if k.dim() != (4 if mx else 5) or k.shape != v.shape or k.dtype != v.dtype or not k.is_contiguous() or \
            not v.is_contiguous():
        raise ValueError("k and v: contiguous [layers][pages][kv heads][page size][head dim] "
                         "(MXFP4: [layers][pages][kv heads][bytes]), alike")
    if not mx and _type_id(k.dtype) == F32:
        raise ValueError("k and v: float16 or bfloat16 (or uint8, MXFP4)")
    if k.get_device() < 0 or k.get_device() != v.get_device():
        raise ValueError(f"k and v: on one device, got {k.device} and {v.device}")
    if mx:
        L, P, H, n = k.shape
        D = _int("head_dim", head_dim)
        S = next((p for p in (16, 32, 64, 128, 256) if D in (64, 128) and kv_head_bytes(p, D) == n), 0)
        if not S:
            raise ValueError(f"k and v: {n} bytes a kv head are no page of MXFP4 rows of head_dim {head_dim}")
    else:
        L, P, H, S, D = k.shape
        if head_dim not in (0, D):
            raise ValueError(f"head_dim {head_dim}, but k and v have {D}")
    c = KvCache(L, P, H, S, D, MXFP4 if mx else _type_id(k.dtype), k.data_ptr(), v.data_ptr())
    c._keep, c._dev = (k, v), k.get_device()
    return c


def kv_batch(q_start, kv_len, page_table, n_tokens: int, max_q: int = 0, max_kv: int = 0) -> KvBatch:
    """A ``tbq_kv_batch`` over int32 device tensors: q_start [sequences + 1],
    kv_len [sequences], page_table [sequences][pages]."""
    n = kv_len.numel()
    _ints("kv_len", kv_len, (n,))
    _ints("q_start", q_start, (n + 1,))
    if page_table.dim() != 2:
        raise ValueError("page_table: [sequences][pages]")
    _ints("page_table", page_table, (n, page_table.shape[1]))
    dev = kv_len.get_device()
    if dev < 0 or q_start.get_device() != dev or page_table.get_device() != dev:
        raise ValueError("q_start, kv_len and page_table: on one device")
    for name, v in (("n_tokens", n_tokens), ("max_q", max_q), ("max_kv", max_kv)):
        _int(name, v)
    b = KvBatch(n, n_tokens, page_table.shape[1], max_q, max_kv, q_start.data_ptr(), kv_len.data_ptr(),
                page_table.data_ptr())
    b._keep, b._dev = (q_start, kv_len, page_table), dev
    return b


def rope(rot_dim: int, theta: float, layout: str = "half", scaling: str = "none", factor: float = 1.0,
         orig_ctx: int = 0, beta_fast: float = 0.0, beta_slow: float = 0.0, factors=None) -> Rope:
    """A rotation plan (tbq_rope_init).  factors: rot_dim / 2 numbers that the
    frequencies are divided by."""
    r = Rope()
    arr = None
    if factors is not None:
        arr = (C.c_float * len(factors))(*[float(f) for f in factors])
        if len(arr) != rot_dim // 2:
            raise ValueError(f"factors: {rot_dim // 2} expected, got {len(arr)}")
    if layout not in _LAYOUTS or scaling not in _SCALINGS:
        raise ValueError(f"layout {layout!r}, scaling {scaling!r}: one of {sorted(_LAYOUTS)}, of {sorted(_SCALINGS)}")
    _check(lib().tbq_rope_init(C.byref(r), rot_dim, _LAYOUTS[layout], theta, _SCALINGS[scaling], factor, orig_ctx,
                               beta_fast, beta_slow, arr), "tbq_rope_init")
    return r


def kv_append(cache: KvCache, layer: int, batch: KvBatch, q, k, v, q_out, rope: Rope = None, q_norm=None, k_norm=None,
              eps: float = 1e-6, positions=None, stream=None):
    """Rotate and append the batch's new rows: q [tokens][heads][D] to q_out
    (both may be None), k and v [tokens][kv heads][D] to their pages."""
    dev = _here(cache, batch)
    if not -_INT <= layer < _INT:
        _int("layer", layer)
    T, D, nkv = batch.n_tokens, cache.head_dim, cache.n_kv_heads
    in_type = _type_id(k.dtype)
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("q, k and v: one type")
    ks, vs = _heads("k", k, T, nkv, D, dev), _heads("v", v, T, nkv, D, dev)
    nq, qs, q_type, qp, qo = 0, 0, cache.type, None, None
    if (q is None) != (q_out is None):
        raise ValueError("q and q_out go together")
    if q is not None:
        nq = q.shape[1]
        qs = _heads("q", q, T, nq, D, dev)
        q_type = _type_id(q_out.dtype)
        qp, qo = q.data_ptr(), _flat("q_out", q_out, (T, nq, D), q_out.dtype, dev)
    f32 = _torch.float32
    qn, kn = _vec("q_norm", q_norm, D, f32, dev), _vec("k_norm", k_norm, D, f32, dev)
    if positions is not None:
        _ints("positions", positions, (T,))
        _on("positions", positions, dev)
    _check(lib().tbq_kv_append(C.byref(cache), layer, C.byref(batch), nq, None if rope is None else C.byref(rope),
                               qn, kn, eps, None if positions is None else positions.data_ptr(), in_type, qp, qs, k.data_ptr(), ks,
                               v.data_ptr(), vs, q_type, qo, _to(stream, dev)), "tbq_kv_append")
    return q_out


def attn_workspace_size(cache: KvCache, batch: KvBatch, n_heads: int, dtype) -> int:
    return int(lib().tbq_attn_paged_workspace_size(C.byref(cache), C.byref(batch), n_heads, _type_id(dtype)))


def attn_paged(cache: KvCache, layer: int, batch: KvBatch, q, out, window: int = 0, sinks: int = 0,
               scale: float = 0.0, workspace=None, stream=None):
    """out[token][head] = attention of q over the pages the token sees."""
    dev = _here(cache, batch)
    if not (-_INT <= layer < _INT and -_INT <= window < _INT and -_INT <= sinks < _INT):
        for name, v in (("layer", layer), ("window", window), ("sinks", sinks)):
            _int(name, v)
    T, D = batch.n_tokens, cache.head_dim
    if q.dim() != 3:
        raise ValueError("q: [tokens][heads][head dim]")
    nq = q.shape[1]
    qs = _heads("q", q, T, nq, D, dev)
    _flat("out", out, (T, nq, D), q.dtype, dev)
    to = _to(stream, dev)
    if workspace is None:
        n = attn_workspace_size(cache, batch, nq, q.dtype)
        if n:
            workspace = _workspace(n, stream)
    else:
        _on("workspace", workspace, dev)
        if not workspace.is_contiguous():
            raise ValueError("workspace: contiguous")
    wp, wb = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _check(lib().tbq_attn_paged(C.byref(cache), layer, C.byref(batch), nq, _type_id(q.dtype), q.data_ptr(), qs,
                                out.data_ptr(), window, sinks, scale, wp, wb, to), "tbq_attn_paged")
    return out


def kv_dequant(cache: KvCache, layer: int, k_out, v_out, pages=None, stream=None):
    """The values of an MXFP4 cache's pages of `layer`: k_out, v_out [n][kv heads]
    [page size][head dim] of one floating type.  pages: int32 device tensor [n]
    (None: the first n pages)."""
    dev = _here(cache)
    if not -_INT <= layer < _INT:
        _int("layer", layer)
    shape = (k_out.shape[0] if k_out.dim() else 0, cache.n_kv_heads, cache.page_size, cache.head_dim)
    out_type = _type_id(k_out.dtype)
    kp, vp = _flat("k_out", k_out, shape, k_out.dtype, dev), _flat("v_out", v_out, shape, k_out.dtype, dev)
    if pages is not None:
        _ints("pages", pages, (shape[0],))
        _on("pages", pages, dev)
    _check(lib().tbq_kv_dequant(C.byref(cache), layer, None if pages is None else pages.data_ptr(), shape[0], out_type,
                                kp, vp, _to(stream, dev)), "tbq_kv_dequant")
    return k_out, v_out


def kv_copy_pages(cache: KvCache, src, dst, stream=None):
    """Pages src[i] -> dst[i] of every layer (lists of int)."""
    n = len(src)
    if len(dst) != n:
        raise ValueError(f"{n} sources, {len(dst)} destinations")
    dev = _here(cache)
    _check(lib().tbq_kv_copy_pages(C.byref(cache), _c_ints("src", src), _c_ints("dst", dst), n, _to(stream, dev)),
           "tbq_kv_copy_pages")


def kv_compact(cache: KvCache, page_table, keep_start, keep, stream=None):
    """Row j of sequence s becomes its row keep[keep_start[s] + j] (int32
    device tensors: page_table [sequences][pages], keep_start [sequences + 1])."""
    dev = _here(cache)
    if page_table.dim() != 2:
        raise ValueError("page_table: [sequences][pages]")
    n = page_table.shape[0]
    _ints("page_table", page_table, page_table.shape)
    _ints("keep_start", keep_start, (n + 1,))
    _ints("keep", keep, (keep.numel(),))
    for name, t in (("page_table", page_table), ("keep_start", keep_start), ("keep", keep)):
        _on(name, t, dev)
    if keep.numel() == 0:   # no row is kept, so none moves
        return
    _check(lib().tbq_kv_compact(C.byref(cache), n, page_table.data_ptr(), page_table.shape[1], keep_start.data_ptr(),
                                keep.data_ptr(), _to(stream, dev)), "tbq_kv_compact")


def kv_tables(page_size: int, kv_len, n_new, page_table, free_pages, n_free, *, q_start, n_drop=None, kv_len_out=None,
              table_out=None, free_out=None, n_free_out=None, slots=None, positions=None, served=None) -> KvTables:
    """A ``tbq_kv_tables`` over int32 device tensors, for ``kv_build_tables``: kv_len,
    n_new, n_drop [sequences], page_table [sequences][pages], free_pages [pages of the
    cache], n_free [1]; outputs that are not given are the inputs of the same meaning.
    slots and positions have a row a token of the batch."""
    _init_torch()
    kv_len_out, table_out = kv_len if kv_len_out is None else kv_len_out, page_table if table_out is None else table_out
    free_out, n_free_out = free_pages if free_out is None else free_out, n_free if n_free_out is None else n_free_out
    n = kv_len.numel()
    if page_table.dim() != 2:
        raise ValueError("page_table: [sequences][pages]")
    rows = next((t.numel() for t in (slots, positions) if t is not None), None)
    if rows is None:
        rows = 1 << 30   # no rows to fill, so no bound on them
    one, table, pages = (1,), (n, page_table.shape[1]), (free_pages.numel(),)
    given = dict(kv_len=(kv_len, (n,)), n_drop=(n_drop, (n,)), n_new=(n_new, (n,)), page_table=(page_table, table),
                 free_pages=(free_pages, pages), n_free=(n_free, one), kv_len_out=(kv_len_out, (n,)),
                 page_table_out=(table_out, table), free_out=(free_out, pages), n_free_out=(n_free_out, one),
                 q_start=(q_start, (n + 1,)), slots=(slots, (rows,)), positions=(positions, (rows,)), served=(served, one))
    dev = kv_len.get_device()
    for name, (t, shape) in given.items():
        if t is not None:
            _ints(name, t, shape)
    for name, (t, _) in given.items():
        if dev < 0 or (t is not None and t.get_device() != dev):
            raise ValueError(f"{name}: tensors on one device, got {kv_len.device if t is None else t.device}")
    t = KvTables(n, page_table.shape[1], _int("page_size", page_size), free_pages.numel(), rows,
                 *(None if t is None else t.data_ptr() for t, _ in given.values()))
    t._keep, t._dev = tuple(t for t, _ in given.values()), dev
    return t


def kv_build_tables(tables: KvTables, stream=None):
    """Pages of dropped positions go back, pages for new ones are taken; the batch's q_start, lengths, page
    table, slots and positions (tbq_kv_build_tables).  Pages that several sequences hold (PagePool.share, fork) must
    not be dropped here: they would be free while the others read them."""
    dev = _here(tables)
    _check(lib().tbq_kv_build_tables(C.byref(tables), _to(stream, dev)), "tbq_kv_build_tables")


def draft_verify_workspace_size(n_seqs: int, n_rows: int, vocab: int, dtype, with_draft: bool) -> int:
    return int(lib().tbq_draft_verify_workspace_size(_int("n_seqs", n_seqs), _int("n_rows", n_rows), _int("vocab", vocab),
                                                     _type_id(dtype), bool(with_draft)))


def _rows_of(name, t, rows, vocab, dev):
    """Elements between the rows of logits [rows][vocab]."""
    if t.dim() != 2 or t.shape != (rows, vocab) or (vocab > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: {(rows, vocab)} with the elements of a row side by side expected, got {tuple(t.shape)}")
    _on(name, t, dev)
    return t.stride(0) if rows > 1 else vocab


def draft_verify(q_start, tokens, logits, u_accept, u_next, n_accept, next_token, n_drop=None, draft_logits=None,
                 temperature=None, workspace=None, stream=None):
    """Which drafts stay, and the token behind them (tbq_draft_verify).  q_start [sequences + 1], tokens [rows],
    n_accept, next_token, n_drop [sequences]: int32; logits, draft_logits [rows][vocab] of one type; u_accept
    [rows], u_next, temperature [sequences]: float32."""
    _init_torch()
    dev, n = _device(), next_token.numel()
    if logits.dim() != 2:
        raise ValueError("logits: [rows][vocab]")
    rows, vocab = logits.shape
    type_id = _type_id(logits.dtype)
    stride = _rows_of("logits", logits, rows, vocab, dev)
    dstride = 0
    if draft_logits is not None:
        if draft_logits.dtype != logits.dtype:
            raise ValueError("logits and draft_logits: one type")
        dstride = _rows_of("draft_logits", draft_logits, rows, vocab, dev)
    i32, f32 = _torch.int32, _torch.float32
    starts, toks = _vec("q_start", q_start, n + 1, i32, dev), _vec("tokens", tokens, rows, i32, dev)
    outs = _vec("n_accept", n_accept, n, i32, dev), _vec("next_token", next_token, n, i32, dev), _vec("n_drop", n_drop, n, i32, dev)
    temp = _vec("temperature", temperature, n, f32, dev)
    us = _vec("u_accept", u_accept, rows, f32, dev), _vec("u_next", u_next, n, f32, dev)
    to = _to(stream, dev)
    if workspace is None:
        size = draft_verify_workspace_size(n, rows, vocab, logits.dtype, draft_logits is not None)
        if size:
            workspace = _workspace(size, stream)
    else:
        _on("workspace", workspace, dev)
        if not workspace.is_contiguous():
            raise ValueError("workspace: contiguous")
    wp, wb = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _check(lib().tbq_draft_verify(n, rows, vocab, type_id, starts, toks, logits.data_ptr(), stride,
                                  None if draft_logits is None else draft_logits.data_ptr(), dstride, temp, *us, *outs, wp, wb,
                                  to), "tbq_draft_verify")
    return next_token


class PagePool:
    """Which pages of a cache are held, and how often (tbq_kv_pool_*)."""

    def __init__(self, n_pages: int):
        self._p = lib().tbq_kv_pool_create(_int("n_pages", n_pages))
        _check(self._p, "tbq_kv_pool_create")

    def close(self):
        if getattr(self, "_p", None):
            lib().tbq_kv_pool_destroy(self._p)
            self._p = None

    __del__ = close

    def free_pages(self) -> int:
        return lib().tbq_kv_pool_free_pages(self._p)

    def holders(self, page: int) -> int:
        return lib().tbq_kv_pool_holders(self._p, _int("page", page))

    def alloc(self, n: int) -> list:
        a = (C.c_int * max(_int("n", n), 1))()
        _check(lib().tbq_kv_pool_alloc(self._p, n, a), "tbq_kv_pool_alloc")
        return list(a[:n])

    def share(self, pages):
        _check(lib().tbq_kv_pool_share(self._p, len(pages), _c_ints("pages", pages)), "tbq_kv_pool_share")

    def release(self, pages):
        _check(lib().tbq_kv_pool_release(self._p, len(pages), _c_ints("pages", pages)), "tbq_kv_pool_release")

    def fork(self, positions: int, page_size: int, pages):
        """The child's pages, and (source, destination) of the page that is to
        be copied, or None."""
        if _int("positions", positions) < 0 or _int("page_size", page_size) < 1:
            raise ValueError(f"{positions} positions in pages of {page_size}")
        n = -(-positions // page_size)
        if len(pages) < n:
            raise ValueError(f"{positions} positions need {n} pages, got {len(pages)}")
        child, copy = (C.c_int * max(n, 1))(), (C.c_int * 2)()
        _check(lib().tbq_kv_pool_fork(self._p, positions, page_size, _c_ints("pages", pages), child, copy),
               "tbq_kv_pool_fork")
        return list(child[:n]), (copy[0], copy[1]) if copy[0] >= 0 else None

    def defrag(self, most: int):
        """[(source, destination)] of the moves that bring the held pages to
        the lowest numbers, at most `most`."""
        src, dst = ((C.c_int * max(_int("most", most), 1))() for _ in range(2))
        n = lib().tbq_kv_pool_defrag(self._p, most, src, dst)
        if n < 0:
            raise TbqError(f"tbq_kv_pool_defrag failed: {lib().tbq_last_error().decode()}")
        return list(zip(src[:n], dst[:n]))


__all__ = ["KvCache", "KvBatch", "KvTables", "Rope", "PagePool", "kv_tables", "kv_build_tables", "draft_verify",
           "draft_verify_workspace_size", "kv_cache", "kv_head_bytes", "kv_batch", "rope", "kv_append", "attn_paged",
           "attn_workspace_size", "kv_dequant", "kv_copy_pages", "kv_compact"]
