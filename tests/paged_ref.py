"""The paged key/value cache's operators in 64 bits on the CPU (torch), and
the setting up of small caches, for the tests of include/tbq_kv.h.  Parity
unpinned against the reference, which has no paged cache; the formulas are
those of include/tbq_kv.h."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    """Largest relative error of one rounding to type t."""
    return torch.finfo(t).eps / 2


def least(t):
    """Half the distance between type t's smallest numbers: what a rounding near zero can lose besides."""
    return float(torch.finfo(t).tiny) * torch.finfo(t).eps / 2


def frequencies(rot, theta, scaling="none", factor=1.0, orig_ctx=0, beta_fast=32.0, beta_slow=1.0, factors=None):
    f, m = [], 1.0
    lo = hi = 0.0
    if scaling == "yarn":
        pair = lambda b: rot * math.log(orig_ctx / (b * 2 * math.pi)) / (2 * math.log(theta))   # noqa: E731
        lo, hi = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot - 1)
        m = 0.1 * math.log(factor) + 1
    for j in range(rot // 2):
        x = theta ** (-2 * j / rot) / (factors[j] if factors is not None else 1)
        if scaling == "linear":
            x /= factor
        if scaling == "yarn":
            r = min(max((j - lo) / max(hi - lo, 0.001), 0), 1)
            x = x / factor * r + x * (1 - r)
        f.append(x)
    return torch.tensor(f, dtype=torch.float64), m


def rotate(x, pos, freq, mscale, layout):
    """x [T][heads][D] (64 bits), pos [T]."""
    R = 2 * len(freq)
    a = pos.double()[:, None, None] * freq
    c, s = torch.cos(a) * mscale, torch.sin(a) * mscale
    y = x.clone()
    i = torch.arange(R // 2)
    u, w = (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y[..., u] = x[..., u] * c - x[..., w] * s
    y[..., w] = x[..., u] * s + x[..., w] * c
    return y


def rmsnorm(x, w, eps):
    return x if w is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


def tokens(q_start, kv_len):
    """(row, sequence, position) of every token row of a sequence."""
    out = []
    for s in range(len(kv_len)):
        n = q_start[s + 1] - q_start[s]
        out += [(q_start[s] + i, s, kv_len[s] - n + i) for i in range(n)]
    return out


def page_of(table, s, pos, page, n_pages):
    e = pos // page
    if e >= len(table[s]):
        return -1
    p = table[s][e]
    return p if 0 <= p < n_pages else -1


def visible(pos, window, sinks):
    """Positions that a token at `pos` sees."""
    return [p for p in range(pos + 1) if window == 0 or p > pos - window or p < sinks]


def attention(k, v, layer, q_start, kv_len, table, q, window=0, sinks=0, scale=0.0):
    """(rows' attention, and sum p |v| and the largest |q|.|k| scale of each, for tolerances), 64 bits:
    {row: (out [heads][D], spread [heads][D], size [heads])}."""
    _, P, NKV, page, D = k.shape
    NQ = q.shape[1]
    scale = scale or 1 / math.sqrt(D)
    res = {}
    for t, s, pos in tokens(q_start, kv_len):
        at = [(page_of(table, s, p, page, P), p % page) for p in visible(pos, window, sinks)]
        at = [x for x in at if x[0] >= 0]
        out, spread, size = torch.zeros(NQ, D).double(), torch.zeros(NQ, D).double(), torch.zeros(NQ).double()
        if at:
            pg, row = torch.tensor([x[0] for x in at]), torch.tensor([x[1] for x in at])
            K = k[layer, pg, :, row].double().repeat_interleave(NQ // NKV, 1)   # [keys][NQ][D]
            V = v[layer, pg, :, row].double().repeat_interleave(NQ // NKV, 1)
            Q = q[t].double()
            sc = (K * Q).sum(-1) * scale
            p = torch.softmax(sc, 0)
            out = (p[..., None] * V).sum(0)
            spread = (p[..., None] * V.abs()).sum(0)
            size = ((K * Q).abs().sum(-1) * scale).amax(0)
        res[t] = (out, spread, size)
    return res


def attention_tolerance(out, spread, size, q_type, c_type):
    """A score's error: F32 rows as pairs of halves (2^-21 of their largest
    element times the keys', taken as 2^-20 of the products' sum with the fp32
    accumulation of up to 128 of them; 16-bit rows: the accumulation alone) and
    a few fp32 roundings of the score itself; p = e^score has that, absolute,
    as its relative error, twice (numerator and sum), and 2^-20 from exp and
    the sums.  16-bit rows round p once (half a step) and the output once."""
    ds = size[:, None] * 2 ** -20
    tol = (2 * ds + 2 ** -20) * spread
    if q_type != torch.float32:
        tol = tol + half_step(c_type) * spread + half_step(q_type) * out.abs() + least(q_type)
    return tol


def make_table(lens, page, gen, spare=0):
    """Table (lists) with every sequence's pages in random order, -1 behind them; number of pages."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    ids = torch.randperm(max(total, 1), generator=gen).tolist()
    width = max(1, max(need, default=1))
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return table, max(total, 1)
