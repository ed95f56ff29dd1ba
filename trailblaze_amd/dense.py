"""Dense Qwen3-style decode on libtbq (tbq_dense_decode, include/tbq.h).

``DenseModel``/``DenseLayer`` mirror the C structs; ``SyntheticDense`` builds a
random-init model of a given shape on the device (the seeded recipe of
``synth``: K-quant blocks with fp16(U(1e-3, 1e-2)) scale fields, fp32 norm
weights around 1) and keeps the host copies of small models for the tests.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _check, _ptr, _stream, _workspace, formats as fm, lib, synth

_vp, _i, _f = C.c_void_p, C.c_int, C.c_float


class DenseLayer(C.Structure):
    _fields_ = [("attn_norm", _vp), ("q_norm", _vp), ("k_norm", _vp), ("ffn_norm", _vp),
                ("wqkv", _vp), ("wo", _vp), ("wgu", _vp), ("wdown", _vp),
                ("wq", _vp), ("wk", _vp), ("wv", _vp), ("wgate", _vp), ("wup", _vp),
                ("qt_qkv", _i), ("qt_o", _i), ("qt_gu", _i), ("qt_down", _i), ("qt_q", _i), ("qt_k", _i),
                ("qt_v", _i), ("qt_gate", _i), ("qt_up", _i)]


class DenseModel(C.Structure):
    _fields_ = [("n_layers", _i), ("hidden", _i), ("n_heads", _i), ("n_kv_heads", _i), ("head_dim", _i),
                ("ffn", _i), ("vocab", _i), ("max_ctx", _i), ("norm_eps", _f), ("rope_theta", _f),
                ("qtype_layers", _i), ("qtype_embd", _i), ("tok_embd", _vp), ("lm_head", _vp),
                ("output_norm", _vp), ("layers", C.POINTER(DenseLayer)), ("k_cache", _vp), ("v_cache", _vp)]


@dataclass
class DenseConfig:
    n_layers: int
    hidden: int
    n_heads: int
    n_kv_heads: int
    head_dim: int
    ffn: int
    vocab: int
    max_ctx: int
    norm_eps: float = 1e-6
    rope_theta: float = 1e6
    qtype_layers: int = fm.Q4_K
    qtype_embd: int = fm.Q6_K


# Qwen3-4B shape, context 4096
QWEN3_4B = DenseConfig(n_layers=36, hidden=2560, n_heads=32, n_kv_heads=8, head_dim=128, ffn=9728,
                       vocab=151936, max_ctx=4096)


class SyntheticDense:
    """A random-init model on the device.  keep_host=True also keeps every
    tensor on the host (``self.host``) for the oracle."""

    def __init__(self, cfg: DenseConfig, seed: int, keep_host: bool = False):
        import torch
        self.cfg = c = cfg
        rng = np.random.default_rng(seed)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        QR = (c.n_heads + 2 * c.n_kv_heads) * c.head_dim
        norm = lambda n: (1.0 + 0.1 * rng.standard_normal(n)).astype(np.float32)
        self.host = {"layers": []} if keep_host else None
        self._keep = []
        layers = (DenseLayer * c.n_layers)()
        for l in range(c.n_layers):
            t = {"attn_norm": norm(c.hidden), "q_norm": norm(c.head_dim), "k_norm": norm(c.head_dim),
                 "ffn_norm": norm(c.hidden),
                 "wqkv": synth.kquant_matrix(c.qtype_layers, QR, c.hidden, rng),
                 "wo": synth.kquant_matrix(c.qtype_layers, c.hidden, c.n_heads * c.head_dim, rng),
                 "wgu": synth.kquant_matrix(c.qtype_layers, 2 * c.ffn, c.hidden, rng),
                 "wdown": synth.kquant_matrix(c.qtype_layers, c.hidden, c.ffn, rng)}
            d = {k: dev(v) for k, v in t.items()}
            self._keep.append(d)
            for k, v in d.items():
                setattr(layers[l], k, v.data_ptr())
            if keep_host:
                self.host["layers"].append(t)
        lm = synth.kquant_matrix(c.qtype_embd, c.vocab, c.hidden, rng)
        on = norm(c.hidden)
        self.lm_head = dev(lm)
        self.output_norm = dev(on)
        if keep_host:
            self.host["lm_head"] = lm
            self.host["output_norm"] = on
        del lm
        kv = (c.n_layers, c.n_kv_heads, c.max_ctx, c.head_dim)
        self.k_cache = torch.zeros(kv, dtype=torch.float32, device="cuda")
        self.v_cache = torch.zeros(kv, dtype=torch.float32, device="cuda")
        self.layers = layers
        self.model = DenseModel(c.n_layers, c.hidden, c.n_heads, c.n_kv_heads, c.head_dim, c.ffn, c.vocab,
                                c.max_ctx, c.norm_eps, c.rope_theta, c.qtype_layers, c.qtype_embd,
                                self.lm_head.data_ptr(), self.lm_head.data_ptr(), self.output_norm.data_ptr(),
                                layers, self.k_cache.data_ptr(), self.v_cache.data_ptr())
        ws = int(lib().tbq_dense_workspace_size(C.byref(self.model)))
        _check(ws > 0, "tbq_dense_workspace_size")
        self.workspace = torch.empty(ws, dtype=torch.uint8, device="cuda")

    def decode(self, token: int, pos: int, logits, stream=None):
        """logits[vocab] (device fp32) for `token` at `pos`; appends K/V at pos."""
        _check(lib().tbq_dense_decode(C.byref(self.model), token, pos, _ptr(logits), _ptr(self.workspace),
                                      self.workspace.numel(), _stream(stream)), "tbq_dense_decode")
        return logits

    def prefill(self, tokens, pos0: int, logits, stream=None):
        """tbq_dense_prefill of `tokens` at positions pos0.. : the last
        token's logits into `logits`, K/V of every position appended."""
        import torch
        toks = np.ascontiguousarray(tokens, dtype=np.int32)
        ws = getattr(self, "_pf_ws", None)
        if ws is None or len(toks) > self._pf_len:   # a workspace serves every shorter prompt
            n = int(lib().tbq_dense_prefill_workspace_size(C.byref(self.model), len(toks)))
            if n > 0:
                ws = self._pf_ws = _workspace(n, stream)
                self._pf_len = len(toks)
        if ws is not None:   # used on this stream, whichever it was made on
            ws.record_stream(torch.cuda.current_stream() if stream is None else stream)
        self._pf_tokens = toks   # read by an asynchronous copy on the stream
        # (n == 0: bad arguments, which the call itself reports)
        _check(lib().tbq_dense_prefill(C.byref(self.model), toks.ctypes.data, len(toks), pos0, _ptr(logits),
                                       _ptr(ws), 0 if ws is None else ws.numel(), _stream(stream)),
               "tbq_dense_prefill")
        return logits

    def prefill_batched(self) -> bool:
        return bool(lib().tbq_dense_prefill_batched(C.byref(self.model)))

    def paged_cache(self, n_pages: int, page_size: int = 64, mxfp4: bool = False):
        """An F16 (or MXFP4) ``paged.KvCache`` of this model's shape, for ``step``."""
        import torch
        from . import paged
        c = self.cfg
        if mxfp4:
            shape = (c.n_layers, n_pages, c.n_kv_heads, paged.kv_head_bytes(page_size, c.head_dim))
            return paged.kv_cache(*(torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2)), head_dim=c.head_dim)
        shape = (c.n_layers, n_pages, c.n_kv_heads, page_size, c.head_dim)
        return paged.kv_cache(*(torch.zeros(shape, dtype=torch.float16, device="cuda") for _ in range(2)))

    def step(self, cache, n_new, kv_len, page_table, tokens, logits, rope=None, window: int = 0, sinks: int = 0,
             stream=None):
        """tbq_dense_step: n_new[s] tokens of every sequence s (side by side in
        `tokens`), kv_len[s] its positions with them, page_table
        [sequences][pages] (host ints); logits [sequences][vocab] (device fp32)
        of each one's last token.  The model has one workspace: steps on
        several streams must wait for each other."""
        import torch
        from . import paged

        def ints(name, v):
            v = np.asarray(v)
            if v.size and (v.dtype.kind not in "iu" or v.min() < -0x80000000 or v.max() > 0x7FFFFFFF):
                raise ValueError(f"{name}: 32-bit ints")
            return np.ascontiguousarray(v, dtype=np.int32)
        n_new, kv_len, page_table = ints("n_new", n_new), ints("kv_len", kv_len), ints("page_table", page_table)
        toks = ints("tokens", tokens)
        n = len(n_new)
        if page_table.ndim != 2 or kv_len.shape != (n,) or len(page_table) != n or len(toks) != n_new.sum():
            raise ValueError("n_new, kv_len and page_table: one row a sequence; tokens: the sum of n_new")
        if logits.numel() != n * self.cfg.vocab or logits.dtype != torch.float32 or not logits.is_contiguous():
            raise ValueError("logits: contiguous float32 [sequences][vocab]")
        dev = paged._here(cache)
        paged._on("logits", logits, dev)
        to, window, sinks = paged._to(stream, dev), paged._int("window", window), paged._int("sinks", sinks)
        with torch.cuda.stream(stream):   # (None: the current one)
            capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            raise ValueError("step is not for capture: a replay would repeat this call's tokens and lengths")
        need = int(lib().tbq_dense_step_workspace_size(C.byref(self.model), C.byref(cache), n, len(toks),
                                                       page_table.shape[1]))
        ws = getattr(self, "_step_ws", None)
        if need > (0 if ws is None else ws.numel()):
            ws = self._step_ws = _workspace(need, stream)
        if ws is not None:   # used on this stream, whichever it was made on
            ws.record_stream(torch.cuda.current_stream() if stream is None else stream)
        # (need == 0: bad arguments, which the call itself reports)
        _check(lib().tbq_dense_step(C.byref(self.model), C.byref(cache), n, n_new.ctypes.data, kv_len.ctypes.data,
                                    page_table.ctypes.data, page_table.shape[1], toks.ctypes.data,
                                    None if rope is None else C.byref(rope), window, sinks, _ptr(logits), _ptr(ws),
                                    0 if ws is None else ws.numel(), to), "tbq_dense_step")
        return logits

    def matvec_shapes(self):
        """(qtype, M, K, weight tensor) of every matvec one decode step runs."""
        c = self.cfg
        QR = (c.n_heads + 2 * c.n_kv_heads) * c.head_dim
        out = []
        for d in self._keep:
            out += [(c.qtype_layers, QR, c.hidden, d["wqkv"]),
                    (c.qtype_layers, c.hidden, c.n_heads * c.head_dim, d["wo"]),
                    (c.qtype_layers, 2 * c.ffn, c.hidden, d["wgu"]),
                    (c.qtype_layers, c.hidden, c.ffn, d["wdown"])]
        out.append((c.qtype_embd, c.vocab, c.hidden, self.lm_head))
        return out
