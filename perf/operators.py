"""The operators of the paged key/value cache as a server's program calls them:
new tokens' keys and values rotated and appended to pages, attention of a chunk
of new tokens over the pages (one token or many, full or with a sliding window
and sinks), copies of whole pages, and compaction of a sequence's kept rows.

Cache: K and V [layers][pages][kv heads][page size][head dim] in 16 bits; page
p of a sequence holds its positions p * page size and on.  Activations N(0, 1),
norm weights around 1; pages of a sequence lie in random order.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False   # True: run() makes the framework's calls instead of the plain forms

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
PAD = 3       # rows behind the last sequence, as a batch padded for a graph has them


# ---- the cases ---------------------------------------------------------------
def listed():
    qwen4b = dict(heads=32, kv=8, dim=128)    # Qwen3-4B's attention
    moe30b = dict(heads=32, kv=4, dim=128)    # Qwen3-30B-A3B's
    small = dict(heads=16, kv=8, dim=64)
    plain = dict(layout="half", scaling="none", factor=1.0, theta=1e6)
    return [
        # one token of one sequence in a decode step: latency
        dict(name="append-1-f32-f16", op="append", act="f32", qact="f32", cache="f16", seqs=1, q=1, past=4095,
             even=True, page=64, layers=2, rot=128, norm=True, **qwen4b, **plain),
        # a decode step of 61 ragged sequences; part of the head rotated, interleaved pairs, without norms
        dict(name="append-61-bf16-partial", op="append", act="bf16", qact="bf16", cache="bf16", seqs=61, q=1,
             past=8000, even=False, page=16, layers=1, rot=64, norm=False, heads=16, kv=4, dim=128,
             layout="interleaved", scaling="linear", factor=4.0, theta=1e4),
        # a long prompt far behind the trained context, as the prefill's 32-bit products give it
        dict(name="append-8192-yarn-f16", op="append", act="f32", qact="f16", cache="f16", seqs=1, q=8192,
             past=122880, even=True, page=64, layers=1, rot=128, norm=True, layout="half", scaling="yarn",
             factor=4.0, theta=1e6, **qwen4b),
        # one token of one sequence over the benchmark's context, 32-bit activations as the decode step has them
        dict(name="attn-1x4096-f32-f16", op="attn", act="f32", cache="f16", seqs=1, q=1, past=4095, even=True,
             page=64, layers=2, window=0, sinks=0, **qwen4b),
        # a decode step of 64 ragged sequences
        dict(name="attn-64x8192-f16", op="attn", act="f16", cache="f16", seqs=64, q=1, past=8191, even=False,
             page=64, layers=1, window=0, sinks=0, **qwen4b),
        # one token over a very long context
        dict(name="attn-1x131072-bf16", op="attn", act="bf16", cache="bf16", seqs=1, q=1, past=131071, even=True,
             page=128, layers=1, window=0, sinks=0, **moe30b),
        # chunks of several prompts and single tokens in one batch, sliding window with sinks, heads of 64
        dict(name="attn-mixed-window-bf16", op="attn", act="bf16", cache="bf16", seqs=9, q=700, past=5000,
             even=False, page=16, layers=1, window=1024, sinks=4, **small),
        # a chunk of a long prompt: matrix products
        dict(name="attn-2048-after-8192-f16", op="attn", act="f16", cache="f16", seqs=1, q=2048, past=8192,
             even=True, page=64, layers=1, window=0, sinks=0, **qwen4b),
        # a fork: the partly filled page of 4 samples
        dict(name="copy-4", op="copy", cache="f16", pages=64, copies=4, page=64, layers=36, kv=8, dim=128),
        # defragmentation of a pool
        dict(name="copy-100", op="copy", cache="bf16", pages=256, copies=100, page=64, layers=36, kv=8, dim=128),
        # rejected speculative tokens leave 16 sequences' ends
        dict(name="compact-16x24", op="compact", cache="f16", seqs=16, rows=24, kept=9, page=16, layers=36, kv=8,
             dim=128),
        # a long context evicted to a bit more than half
        dict(name="compact-16000-to-9001", op="compact", cache="bf16", seqs=1, rows=16000, kept=9001, page=64,
             layers=36, kv=4, dim=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "append", "attn", "attn", "attn", "copy", "compact"])
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    act, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(op=op, act=act, qact=rng.choice([act, cache]), cache=cache, seqs=seqs, q=_log(rng, 1, 8000 // seqs),
                    past=_log(rng, 1, 100000 // seqs), even=rng.random() < 0.3, page=page, layers=rng.choice([1, 2]),
                    rot=rng.choice([dim, dim // 2, dim // 4]), norm=rng.random() < 0.5, heads=heads, kv=kv, dim=dim,
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 8.0]), theta=rng.choice([1e4, 5e5, 1e6]))
    if op == "attn":
        q = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 1500)])
        seqs = _log(rng, 1, 64) if q == 1 else _log(rng, 1, max(1, min(32, 3000 // q)))
        past = _log(rng, 1, min(100000, 300000 // seqs, 12000000 // (q * seqs)))
        window = rng.choice([0, 0, _log(rng, 1, 4000)])
        return dict(op=op, act=act, cache=cache, seqs=seqs, q=q, past=past, even=rng.random() < 0.3, page=page,
                    layers=rng.choice([1, 2]), window=window, sinks=rng.choice([0, 1, 4, 70]) if window else 0,
                    heads=heads, kv=kv, dim=dim)
    layers = _log(rng, 1, 36)
    if op == "copy":
        pages = _log(rng, 4, 200)
        return dict(op=op, cache=cache, pages=pages, copies=_log(rng, 1, pages // 2), page=page, layers=layers, kv=kv,
                    dim=dim)
    seqs = _log(rng, 1, 16)
    rows = _log(rng, 2, 16000 // seqs)
    return dict(op=op, cache=cache, seqs=seqs, rows=rows, kept=_log(rng, 1, rows), page=page, layers=layers, kv=kv,
                dim=dim)


def _lengths(c):
    """(new tokens, cached positions before them) of each sequence; ragged
    batches are the same for every seed."""
    if c["even"]:
        return [(c["q"], c["past"])] * c["seqs"]
    r = random.Random(c["q"] * 1000003 + c["past"] * 101 + c["seqs"])
    out = [(c["q"], c["past"])]
    while len(out) < c["seqs"]:
        n = 1 if c["q"] == 1 or r.random() < 0.3 else r.randint(0, c["q"])
        out.append((n, r.randint(0, c["past"])))
    r.shuffle(out)
    return out


# ---- inputs ------------------------------------------------------------------
def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _pool(c, pages, g):
    shape = (c["layers"], pages, c["kv"], c["page"], c["dim"])
    k, v = (torch.empty(shape, device="cuda", dtype=DTYPES[c["cache"]]) for _ in range(2))
    for l in range(c["layers"]):
        k[l], v[l] = _randn(shape[1:], g), _randn(shape[1:], g)
    return k, v


def _table(lens, page, g):
    """Page table [sequences][most pages of one] and the number of pages: every
    sequence's pages in random order, -1 behind its last."""
    need = [-(-n // page) for n in lens]
    total = max(1, sum(need))
    ids = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    c, s = case, SimpleNamespace(case=case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    if c["op"] in ("append", "attn"):
        lens = _lengths(c)
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        s.tokens, s.rows = starts[-1], starts[-1] + (PAD if not c["even"] else 0)
        s.max_q, s.max_kv = max(n for n, _ in lens), max(n + p for n, p in lens)
        s.q_start, s.kv_len = ints(starts), ints([n + p for n, p in lens])
        s.table, pages = _table([n + p for n, p in lens], c["page"], g)
        s.k, s.v = _pool(c, pages, g)
        s.layer = c["layers"] - 1
        act = DTYPES[c["act"]]
        D, NQ, NKV = c["dim"], c["heads"], c["kv"]
        if c["op"] == "append":
            # q, k and v of a token side by side, as one product with the three matrices gives them
            s.qkv = _randn((s.rows, (NQ + 2 * NKV) * D), g, act)
            s.q_norm, s.k_norm = (1 + 0.1 * _randn((D,), g) if c["norm"] else None for _ in range(2))
            s.q_out = torch.zeros((s.rows, NQ, D), device="cuda", dtype=DTYPES[c["qact"]])
        else:
            s.q = (1.5 * _randn((s.rows, NQ, D), g)).to(act)
            s.out = torch.zeros((s.rows, NQ, D), device="cuda", dtype=act)
    elif c["op"] == "copy":
        s.k, s.v = _pool(c, c["pages"], g)
        ids = torch.randperm(c["pages"], device="cuda", generator=g).tolist()
        s.src, s.dst = ids[:c["copies"]], ids[c["copies"]:2 * c["copies"]]
    else:
        lens = [c["rows"]] * c["seqs"]
        s.table, pages = _table(lens, c["page"], g)
        s.k, s.v = _pool(c, pages, g)
        keep = [torch.randperm(c["rows"], device="cuda", generator=g)[:c["kept"]].sort().values for _ in lens]
        s.keep = torch.cat(keep).to(torch.int32)
        s.keep_start = ints([i * c["kept"] for i in range(c["seqs"] + 1)])
    if own:   # the handles that a server keeps
        from trailblaze_amd import paged
        s.cache = paged.kv_cache(s.k, s.v)
        if c["op"] in ("append", "attn"):
            s.batch = paged.kv_batch(s.q_start, s.kv_len, s.table, s.rows, max_q=s.max_q, max_kv=s.max_kv)
        if c["op"] == "append":
            s.rope = paged.rope(c["rot"], c["theta"], layout=c["layout"], scaling=c["scaling"], factor=c["factor"],
                                orig_ctx=ORIG_CTX)
        if c["op"] == "attn":
            size = paged.attn_workspace_size(s.cache, s.batch, c["heads"], s.q.dtype)
            s.ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------
def run(s):
    c = s.case
    if own:
        return _own(s, c)
    return {"append": _append, "attn": _attn, "copy": _copy, "compact": _compact}[c["op"]](s, c)


def _own(s, c):
    from trailblaze_amd import paged
    if c["op"] == "append":
        NQ, NKV, D = c["heads"], c["kv"], c["dim"]
        q, k, v = s.qkv.view(s.rows, NQ + 2 * NKV, D).split((NQ, NKV, NKV), 1)
        paged.kv_append(s.cache, s.layer, s.batch, q, k, v, s.q_out, rope=s.rope, q_norm=s.q_norm, k_norm=s.k_norm,
                        eps=EPS)
        return {"q": s.q_out, "k": s.k, "v": s.v}
    if c["op"] == "attn":
        return paged.attn_paged(s.cache, s.layer, s.batch, s.q, s.out, window=c["window"], sinks=c["sinks"],
                                workspace=s.ws)
    if c["op"] == "copy":
        paged.kv_copy_pages(s.cache, s.src, s.dst)
    else:
        paged.kv_compact(s.cache, s.table, s.keep_start, s.keep)
    return {"k": s.k, "v": s.v}


# rotation frequencies in 64 bits: theta^(-2j/rot), divided by the factor
# (linear), or by a share of it that grows from the pairs that turn often
# within the trained context to those that turn seldom (YaRN, arXiv 2309.00071)
ORIG_CTX = 32768
BETA_FAST, BETA_SLOW = 32.0, 1.0


def _frequencies(c):
    j = torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64)
    f = c["theta"] ** (-2 * j / c["rot"])
    if c["scaling"] == "none":
        return f, 1.0
    if c["scaling"] == "linear":
        return f / c["factor"], 1.0
    turns = lambda beta: c["rot"] * math.log(ORIG_CTX / (beta * 2 * math.pi)) / (2 * math.log(c["theta"]))   # noqa: E731
    lo, hi = max(math.floor(turns(BETA_FAST)), 0), min(math.ceil(turns(BETA_SLOW)), c["rot"] - 1)
    share = ((j - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f / c["factor"] * share + f * (1 - share), 0.1 * math.log(c["factor"]) + 1


def _places(s, c):
    """Sequence, cache position, page and row in the page of every token."""
    n = (s.q_start[1:] - s.q_start[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), n, output_size=s.tokens)
    pos = torch.arange(s.tokens, device="cuda") - s.q_start[seq] + (s.kv_len[seq].long() - n[seq])
    return seq, pos, s.table[seq, pos // c["page"]].long(), pos % c["page"]


def _append(s, c):
    NQ, NKV, D, rot, T = c["heads"], c["kv"], c["dim"], c["rot"], s.tokens
    seq, pos, pg, row = _places(s, c)
    x = s.qkv[:T].view(T, NQ + 2 * NKV, D).float()
    qk = x[:, :NQ + NKV]
    if c["norm"]:
        w = torch.cat([s.q_norm.expand(NQ, D), s.k_norm.expand(NKV, D)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    f, m = _frequencies(c)
    ang = pos.double()[:, None] * f
    cos, sin = (ang.cos() * m).float()[:, None], (ang.sin() * m).float()[:, None]
    if c["layout"] == "half":
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    qk = torch.cat([turned, qk[..., rot:]], -1)
    s.q_out[:T] = qk[:, :NQ].to(s.q_out.dtype)
    s.k[s.layer][pg, :, row] = qk[:, NQ:].to(s.k.dtype)
    s.v[s.layer][pg, :, row] = x[:, NQ + NKV:].to(s.v.dtype)
    return {"q": s.q_out, "k": s.k, "v": s.v}


def _attn(s, c):
    NQ, NKV, D, S = c["heads"], c["kv"], c["dim"], c["seqs"]
    G, n_pages = NQ // NKV, -(-s.max_kv // c["page"])
    seq, pos, _, _ = _places(s, c)
    at = torch.arange(s.tokens, device="cuda") - s.q_start[seq]
    ids = s.table[:, :n_pages].clamp(min=0).long()
    rows = lambda t: t[s.layer][ids].transpose(1, 2).reshape(S, NKV, n_pages * c["page"], D).float()   # noqa: E731
    q = torch.zeros((S, s.max_q, NQ, D), device="cuda")
    q[seq, at] = s.q[:s.tokens].float()
    qpos = torch.full((S, s.max_q), -1, dtype=torch.int64, device="cuda")
    qpos[seq, at] = pos
    q = q.view(S, s.max_q, NKV, G, D).permute(0, 2, 1, 3, 4).reshape(S, NKV, s.max_q * G, D)
    score = torch.matmul(q, rows(s.k).transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(D))
    key, qp = torch.arange(n_pages * c["page"], device="cuda"), qpos[..., None]
    seen = key <= qp
    if c["window"]:
        seen &= (key > qp - c["window"]) | (key < c["sinks"])
    hidden = ~seen.repeat_interleave(G, 1)[:, None]
    score.masked_fill_(hidden, -1e30)
    score.sub_(score.amax(-1, keepdim=True)).exp_().masked_fill_(hidden, 0)
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score, rows(s.v)) / total.clamp(min=1e-30)
    o = o.view(S, NKV, s.max_q, G, D).permute(0, 2, 1, 3, 4).reshape(S, s.max_q, NQ, D)
    s.out[:s.tokens] = o[seq, at].to(s.out.dtype)
    return s.out


def _copy(s, c):
    src, dst = (torch.tensor(x, device="cuda") for x in (s.src, s.dst))
    for t in (s.k, s.v):
        t[:, dst] = t[:, src]
    return {"k": s.k, "v": s.v}


def _compact(s, c):
    n = (s.keep_start[1:] - s.keep_start[:-1]).long()
    total = s.keep.numel()
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), n, output_size=total)
    to = torch.arange(total, device="cuda") - s.keep_start[seq]
    src, dst = (s.table[seq, p // c["page"]].long() * c["page"] + p % c["page"] for p in (s.keep.long(), to))
    for t in (s.k, s.v):
        r = t.transpose(2, 3)   # [layers][pages][rows][heads][dims]
        r[:, dst // c["page"], dst % c["page"]] = r[:, src // c["page"], src % c["page"]]
    return {"k": s.k, "v": s.v}


# ---- what a pass cannot do without --------------------------------------------
def work(case):
    c = case
    size = lambda name: 4 if name == "f32" else 2   # noqa: E731
    if c["op"] == "copy":
        return {"bytes": 2 * c["copies"] * c["layers"] * c["kv"] * c["page"] * c["dim"] * 2 * 2, "flops": 0}
    if c["op"] == "compact":
        return {"bytes": 2 * c["seqs"] * c["kept"] * c["layers"] * c["kv"] * c["dim"] * 2 * 2, "flops": 0}
    lens, D, NQ, NKV = _lengths(c), c["dim"], c["heads"], c["kv"]
    T = sum(n for n, _ in lens)
    if c["op"] == "append":
        inp, out = T * (NQ + 2 * NKV) * D * size(c["act"]), T * (NQ * size(c["qact"]) + 2 * NKV * 2) * D
        return {"bytes": inp + out, "flops": T * (NQ + NKV) * (3 * c["rot"] + (4 * D if c["norm"] else 0))}
    W, keys, pairs = c["window"], 0, 0
    for n, past in lens:
        if n == 0:
            continue
        far = lambda p: max(0, p - W + 1) if W else 0   # noqa: E731   first position of the window of a token at p
        first = far(past)
        keys += past + n - first + min(first, c["sinks"])
        pairs += sum(p + 1 - far(p) + min(far(p), c["sinks"]) for p in range(past, past + n))
    return {"bytes": keys * NKV * D * 2 * 2 + 2 * T * NQ * D * size(c["act"]), "flops": 4 * pairs * NQ * D}


# ---- the same in 64 bits -------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] in ("copy", "compact"):
        return _moved64(s, c)
    starts, lens, table = s.q_start.tolist(), s.kv_len.tolist(), s.table.tolist()
    return _append64(s, c, starts, lens, table) if c["op"] == "append" else _attn64(s, c, starts, lens)


def _moved64(s, c):
    """Values are moved, not computed: page by page, and row by row of a sequence."""
    out = {}
    for name in ("k", "v"):
        old = getattr(s, name)
        new = old.clone()
        if c["op"] == "copy":
            for a, b in zip(s.src, s.dst):
                new[:, b] = old[:, a]
        else:
            for q in range(c["seqs"]):
                i, j = int(s.keep_start[q]), int(s.keep_start[q + 1])
                pages = [p for p in s.table[q].tolist() if p >= 0]
                flat = old[:, pages].permute(0, 2, 1, 3, 4).reshape(c["layers"], c["kv"], -1, c["dim"])
                moved = flat.clone()
                moved[:, :, :j - i] = flat[:, :, s.keep[i:j].long()]
                new[:, pages] = moved.view(c["layers"], c["kv"], len(pages), c["page"], c["dim"]).permute(0, 2, 1, 3, 4)
        out[name] = new
    return out


def _append64(s, c, starts, lens, table):
    NQ, NKV, D, R, page = c["heads"], c["kv"], c["dim"], c["rot"], c["page"]
    place = torch.full((s.rows,), -1, dtype=torch.int64)
    pos = torch.zeros(s.rows, dtype=torch.float64)
    for i in range(c["seqs"]):
        a, b = starts[i], starts[i + 1]
        for t in range(a, b):
            p = lens[i] - (b - a) + t - a
            pos[t], place[t] = p, table[i][p // page] * page + p % page
    # complex rotation: pair (u, w) as u + iw times m e^(ia)
    j = torch.arange(R // 2, dtype=torch.float64)
    f, m = torch.exp(-2 * j / R * math.log(c["theta"])), 1.0
    if c["scaling"] == "linear":
        f = f / c["factor"]
    elif c["scaling"] == "yarn":
        edge = lambda b: R * math.log(ORIG_CTX / (2 * math.pi * b)) / (2 * math.log(c["theta"]))   # noqa: E731
        lo, hi = max(math.floor(edge(BETA_FAST)), 0), min(math.ceil(edge(BETA_SLOW)), R - 1)
        ramp = torch.clamp((j - lo) / max(hi - lo, 0.001), 0, 1)
        f, m = f * (1 - ramp) + f * ramp / c["factor"], 1 + 0.1 * math.log(c["factor"])
    turn = torch.polar(torch.full((s.rows, R // 2), m, dtype=torch.float64), pos[:, None] * f).cuda()
    x = s.qkv.double().view(s.rows, NQ + 2 * NKV, D)

    def heads(y, w):
        if w is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
        r = y[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2) if c["layout"] == "half" else \
            y[..., :R].unflatten(-1, (R // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(r.contiguous()) * turn[:, None])
        z = z.transpose(-1, -2).flatten(-2) if c["layout"] == "half" else z.flatten(-2)
        return torch.cat([z, y[..., R:]], -1)

    q = s.q_out.double()
    q[:s.tokens] = heads(x[:, :NQ], s.q_norm)[:s.tokens]
    out = {"q": q}
    at = place[:s.tokens].cuda()
    new = {"k": heads(x[:, NQ:NQ + NKV], s.k_norm)[:s.tokens], "v": x[:s.tokens, NQ + NKV:]}
    for name in ("k", "v"):
        pool = getattr(s, name).double()
        pool[s.layer].transpose(1, 2)[at // page, at % page] = new[name]
        out[name] = pool
    return out


def _attn64(s, c, starts, lens):
    NQ, NKV, D = c["heads"], c["kv"], c["dim"]
    G = NQ // NKV
    out = s.out.double()
    for i in range(c["seqs"]):
        a, b, n = starts[i], starts[i + 1], lens[i]
        if a == b:
            continue
        ids = s.table[i, :-(-n // c["page"])].long()
        K, V = (t[s.layer][ids].transpose(0, 1).flatten(1, 2)[:, :n].double() for t in (s.k, s.v))
        pos = torch.arange(n - (b - a), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        off = key > pos
        if c["window"]:
            off |= (pos - key >= c["window"]) & (key >= c["sinks"])
        for h in range(NQ):
            sc = s.q[a:b, h].double() @ K[h // G].t().contiguous() / math.sqrt(D)
            out[a:b, h] = torch.softmax(sc.masked_fill_(off, -math.inf), -1) @ V[h // G].contiguous()
    return out
