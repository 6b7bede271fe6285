"""Plain 64-bit restatements of the cache in pages and of beam selection, and a
small pool to run them on (helpers of the tests, not a test module)."""
import numpy as np


def slot(table_row, pos, page, n_pages):
    """(page, row) of a position, or None where no page holds it."""
    col = pos // page
    if col >= len(table_row):
        return None
    p = int(table_row[col])
    return (p, pos % page) if 0 <= p < n_pages else None


def turned(x, pos, cos, sin):
    """Rotate-half RoPE of x [..., hd] in 64 bits."""
    half = x.shape[-1] // 2
    c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def attention(q, k, v, table, lens, n_tok, mask, page, heads, layer=0):
    """q [n, T, H, hd] turned already; k, v [layers, pages, rows, kvh, hd].  Returns the
    result and sum_j p_j |v_j| (what rounding errors are relative to); rows past
    n_tok are NaN in both."""
    n, T, H, hd = q.shape
    g = H // k.shape[3]
    out = np.full((n, T, H, hd), np.nan)
    size = np.full((n, T, H, hd), np.nan)
    for s in range(n):
        for i in range(n_tok[s]):
            rows = []
            for j in range(lens[s] + n_tok[s]):
                own = j - int(lens[s])
                if own >= 0 and not (int(mask[s][i]) >> own) & 1:
                    continue
                at = slot(table[s], j, page, k.shape[1])
                if at is not None:
                    rows.append(at)
            out[s, i], size[s, i] = 0, 0
            if not rows:
                continue
            p, r = np.array([x[0] for x in rows]), np.array([x[1] for x in rows])
            kk, vv = k[layer, p, r].astype(np.float64), v[layer, p, r].astype(np.float64)
            for h in range(H):
                sc = kk[:, h // g] @ q[s, i, h].astype(np.float64) / np.sqrt(hd)
                w = np.exp(sc - sc.max()) if sc.max() > -np.inf else np.zeros_like(sc)
                if w.sum() == 0:
                    continue
                w /= w.sum()
                used = w > 0  # a weight of 0 gives a value no part, whatever the value
                out[s, i, h] = w[used] @ vv[used, h // g]
                size[s, i, h] = w[used] @ np.abs(vv[used, h // g])
    return out, size


def fork(table, refs, parent, lens, page, extra, table_ld):
    """(table_out, refs_out, info, copies [(src, dst, rows)]) by the rules, one step after
    the other."""
    n_pages, pr = len(refs), page
    refs = refs.astype(np.int64).copy()
    ok = lambda p: 0 <= p < n_pages  # noqa: E731
    for p in table.reshape(-1):
        if ok(p):
            refs[p] -= 1
    n = len(parent)
    new = np.full((n, table_ld), -1, np.int32)
    plan = []
    for i in range(n):
        s, L = int(parent[i]), int(lens[i])
        if not (0 <= s < len(table)) or L < 0:
            plan.append(None)
            continue
        L = min(L, table_ld * pr)
        full = L // pr if extra > 0 else -(-L // pr)
        tail = L % pr if extra > 0 else 0
        need = min(table_ld, -(-(L + extra) // pr))
        plan.append((s, full, tail, need))
        for c in range(full):
            if ok(table[s, c]):
                new[i, c] = table[s, c]
                refs[table[s, c]] += 1
    seen, keeps = set(), []
    for i, f in enumerate(plan):
        if f and f[2] and ok(table[f[0], f[1]]):
            p = int(table[f[0], f[1]])
            if p not in seen and refs[p] == 0:
                keeps.append((i, p))
            seen.add(p)
    for i, p in keeps:
        new[i, plan[i][1]] = p
        refs[p] += 1
    free = [p for p in range(n_pages) if refs[p] == 0]
    taken, copies, missing = 0, [], 0
    for i, f in enumerate(plan):
        if not f:
            continue
        s, full, tail, need = f
        for c in range(full, need):
            if new[i, c] >= 0:
                continue
            if taken == len(free):
                missing += 1
                continue
            new[i, c] = free[taken]
            taken += 1
            refs[new[i, c]] += 1
            if c == full and tail and ok(table[s, c]):
                copies.append((int(table[s, c]), int(new[i, c]), tail))
    info = np.array([len(copies), missing, len(free) - taken], np.int32)
    return new, refs.astype(np.int32), info, copies


def select(logits, cum, done, eos, n_out):
    """logits [n, B, V]: (token, parent, score) [n, n_out] in 64 bits."""
    n, B, V = logits.shape
    token, parent = np.full((n, n_out), -1, np.int32), np.full((n, n_out), -1, np.int32)
    score = np.full((n, n_out), -np.inf)
    for s in range(n):
        best = []
        for b in range(B):
            c = float(cum[s, b])
            if done is not None and done[s, b]:
                if c > -np.inf:
                    best.append((-c, b, 0.0, eos))
                continue
            x = logits[s, b].astype(np.float64)
            if np.isnan(x).any() or (x == np.inf).any() or not np.isfinite(x.max()):
                continue
            lse = x.max() + np.log(np.exp(x - x.max()).sum())
            order = np.argsort(-x, kind="stable")[:n_out]
            best += [(-(c + (x[t] - lse)), b, -x[t], int(t)) for t in order
                     if c + (x[t] - lse) > -np.inf]
        for r, (a, b, _, t) in enumerate(sorted(best)[:n_out]):
            token[s, r], parent[s, r], score[s, r] = t, b, -a
    return token, parent, score


class Device:
    """Arrays on the device for one test, freed together."""

    def __init__(self, ctx):
        self.ctx, self.bufs = ctx, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.ctx.sync()
        for b in self.bufs:
            b.free()
            self.ctx._bufs.remove(b)

    def up(self, a):
        b = self.ctx.upload(np.ascontiguousarray(a))
        self.bufs.append(b)
        return b.ptr

    def get(self, ptr, like):
        return self.ctx.download(ptr, like.dtype, like.size).reshape(like.shape)


KV = {"f32": (0, np.float32), "f16": (1, np.float16)}


def tables(lens, page, ld, n_pages, rng):
    """Page tables of sequences of lens rows, pages shuffled, -1 past the end."""
    table = np.full((len(lens), ld), -1, np.int32)
    need = [min(ld, -(-x // page)) for x in lens]
    perm = rng.permutation(n_pages)[:sum(need)]
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = perm[at:at + k]
        at += k
    return table


def tree(n, rng):
    """Parents of a drafted tree's nodes."""
    return np.array([-1] + [i - 1 if rng.random() < 0.5 else int(rng.integers(-1, i))
                            for i in range(1, n)], np.int32)
