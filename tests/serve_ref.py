"""A serving step's tables and the verification of drafts as include/tbq_kv.h
words them, on the host: lists, and numpy in 64 bits."""
import numpy as np


def tables(page, n_tokens, kv_len, n_drop, n_new, table, free, n_free):
    """dict of the outputs, as lists.  free has an entry a page of the cache."""
    W, P = len(table[0]) if table else 1, len(free)
    up = lambda n: -(-n // page)   # noqa: E731
    table, stack = [list(r) for r in table], list(free[:min(max(n_free, 0), P)])
    lens = [min(max(n, 0), W * page) for n in kv_len]
    for s, row in enumerate(table):
        base = lens[s] - min(max(n_drop[s] if n_drop else 0, 0), lens[s])
        for e in range(up(base), up(lens[s])):
            if 0 <= row[e] < P and len(stack) < P:
                stack.append(row[e])
        row[up(base):] = [-1] * (W - up(base))
        lens[s] = base
    q_start, slots, positions, served, going = [0], [], [], 0, True
    for s, row in enumerate(table):
        new, kept = max(n_new[s], 0), up(lens[s])
        need = up(lens[s] + new)
        going = going and need <= W and need - kept <= len(stack) and q_start[-1] + new <= n_tokens
        if going:
            served += 1
            for e in range(kept, need):
                row[e] = stack.pop()
            for p in range(lens[s], lens[s] + new):
                at = row[p // page]
                positions.append(p)
                slots.append(at * page + p % page if 0 <= at < P else -1)
            lens[s] += new
        q_start.append(len(positions))
    rest = [-1] * (n_tokens - len(positions))
    return dict(kv_len=lens, table=table, free=stack + [-1] * (P - len(stack)), n_free=[len(stack)], q_start=q_start,
                slots=slots + rest, positions=positions + rest, served=[served])


def law(row, T):
    """Probabilities of a row of logits at temperature T (zeros for a row without weight)."""
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return np.zeros(len(x))
    if not T > 0:
        return (np.arange(len(x)) == x.argmax()).astype(np.float64)
    if m == np.inf:
        e = (x == np.inf).astype(np.float64)
    else:
        with np.errstate(invalid="ignore"):
            z = (x - m) / T
        e = np.where(x == -np.inf, 0.0, np.exp(np.where(np.isnan(z), -np.inf, z)))
    return e / e.sum()


def verify(q_start, tokens, logits, draft, T, u_accept, u_next):
    """(n_accept, next, n_drop) of each sequence; logits and draft (or None): 64-bit arrays [rows][vocab]."""
    n_rows, V = logits.shape
    out = []
    u_accept, u_next = (np.clip(np.nan_to_num(u, nan=0.0), 0.0, 1 - 2.0 ** -24) for u in (u_accept, u_next))
    for s in range(len(q_start) - 1):
        a, b = q_start[s], q_start[s + 1]
        if a < 0 or b <= a or b > n_rows:
            out.append((0, -1, 0))
            continue
        t = 1.0 if T is None else T[s]
        for r in range(a, b):
            w = p = law(logits[r], t)
            if r + 1 == b:
                break
            x = tokens[r + 1]
            q = (np.arange(V) == x).astype(np.float64) if draft is None else law(draft[r], t)
            px, qx = (p[x], q[x]) if 0 <= x < V else (0.0, 0.0)
            if not u_accept[r] * qx < px:
                w = np.maximum(p - q, 0)
                w = w if w.sum() > 0 else p
                break
        run = np.cumsum(w)
        at = -1
        if run[-1] > 0:
            over = np.nonzero((run > u_next[s] * run[-1]) & (w > 0))[0]
            at = int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])
        out.append((r - a, at, b - a - 1 - (r - a)))
    return tuple(list(c) for c in zip(*out)) if out else ([], [], [])
