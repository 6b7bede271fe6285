"""Operators of decoding with several hypotheses at once, as measurable cases.

Beam search and drafted (speculated) token trees keep many continuations of a text
over one cache of K/V pages.  A case is one call of the entry point for one step of
that: the beams' selection over the vocabulary, the fork of their page tables, the
store of new K/V rows, the attention over the pages (one token a sequence, or a tree of
drafted ones) and the compaction after a tree was verified.  `own` False computes it in
elementary torch operations; True calls this library.

All inputs are made on the GPU from the seed.  exact() restates each case in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
KV_TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16)}

_ctx = None


def _context():
    """The program's one device context.  Its in-order stream is its own, not torch's: what
    torch still computes is waited for before the first call (prepare), and what the calls
    compute (Context.sync, or torch.cuda.synchronize) before torch reads or frees it."""
    global _ctx
    if _ctx is None:
        from llm_core_amd import hip

        _ctx = hip.Context(0)
    return _ctx


# --------------------------------------------------------------------------- cases


def listed():
    return [
        # one token of one sequence, 16/2 heads (a 2048-wide layer): the smallest attention call
        {"name": "attn 1x1 @1024 16/2", "op": "attn", "seqs": 1, "tok": 1, "heads": 16,
         "kv_heads": 2, "head_dim": 128, "len": 1024, "ragged": False, "share": 0, "kv": "f32",
         "page": 16, "rope": True},
        # 12 texts with 4 beams each at the 14/2-head, 64-wide shape, fp16 pages: the beams of a
        # text share all but their last pages
        {"name": "attn beams 48x1 14/2 f16", "op": "attn", "seqs": 48, "tok": 1, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "len": 3005, "ragged": True, "share": 4, "kv": "f16",
         "page": 32, "rope": True},
        # one sequence's tree of 32 drafted tokens
        {"name": "attn tree 1x32 @2048", "op": "attn", "seqs": 1, "tok": 32, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "len": 2048, "ragged": False, "share": 0, "kv": "f32",
         "page": 16, "rope": True},
        # 16 long sequences, each with a tree of up to 48 drafted tokens: the largest
        {"name": "attn tree 16x48 @8191", "op": "attn", "seqs": 16, "tok": 48, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "len": 8191, "ragged": True, "share": 0, "kv": "f32",
         "page": 32, "rope": True},
        # 4 beams over a 32000-token vocabulary
        {"name": "select 1x4 of 32000", "op": "select", "seqs": 1, "beams": 4, "vocab": 32000,
         "keep": 8, "done": False},
        # 8 texts with 8 beams each over the 151936-token vocabulary, some beams finished
        {"name": "select 8x8 of 151936", "op": "select", "seqs": 8, "beams": 8, "vocab": 151936,
         "keep": 16, "done": True},
        # beams of one text step on: the copies behind the survivors
        {"name": "fork 4 beams @1000", "op": "fork", "seqs": 1, "beams": 4, "len": 1000, "page": 16,
         "layers": 2, "kv_heads": 2, "head_dim": 128, "kv": "f32", "extra": 1},
        # 16 texts with 8 beams each, 24 layers of fp16 pages
        {"name": "fork 16x8 beams @1500", "op": "fork", "seqs": 16, "beams": 8, "len": 1500,
         "page": 32, "layers": 24, "kv_heads": 2, "head_dim": 64, "kv": "f16", "extra": 1},
        # new K/V rows of one decode step, and of 24 drafted trees into fp16 pages
        {"name": "store 8x1", "op": "store", "seqs": 8, "tok": 1, "kv_heads": 8, "head_dim": 128,
         "len": 3005, "kv": "f32", "page": 16, "bias": True},
        {"name": "store 24x48 f16", "op": "store", "seqs": 24, "tok": 48, "kv_heads": 8,
         "head_dim": 128, "len": 900, "kv": "f16", "page": 32, "bias": False},
        # one verified tree of a short model, and 16 of 32 layers: the accepted rows move together
        {"name": "compact 1x16 tree", "op": "compact", "seqs": 1, "tok": 16, "kv_heads": 2,
         "head_dim": 128, "len": 1024, "layers": 2, "kv": "f32", "page": 16},
        {"name": "compact 16x32 tree", "op": "compact", "seqs": 16, "tok": 32, "kv_heads": 8,
         "head_dim": 128, "len": 300, "layers": 32, "kv": "f32", "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "attn", "select", "select", "fork", "store",
                     "compact"])
    kv_heads, group = rng.choice([2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    head_dim = rng.choice([64, 128, 128, 256])
    kv, page = rng.choice(["f32", "f32", "f16"]), rng.choice([8, 16, 32, 64])
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = _log(rng, 1000, 152000)
        most = max(1, 8 * 8 * 151936 // (beams * vocab))
        return {"op": op, "seqs": min(_log(rng, 1, 32), most), "beams": beams, "vocab": vocab,
                "keep": rng.choice([beams, 2 * beams]), "done": rng.random() < 0.5}
    if op == "attn":
        tok = 1 if rng.random() < 0.4 else _log(rng, 2, 64)
        seqs = _log(rng, 1, 48)
        share = rng.choice([0, 0, 2, 4]) if tok == 1 else 0
        rows = seqs * kv_heads * head_dim
        most = min(16 * 8191 * 8 * 128 // rows, 16 * 8191 * 48 * 32 * 128 // (rows * group * tok))
        return {"op": op, "seqs": seqs, "tok": tok, "heads": kv_heads * group,
                "kv_heads": kv_heads, "head_dim": head_dim,
                "len": max(1, min(_log(rng, 1, 12000), most)), "ragged": rng.random() < 0.6,
                "share": share, "kv": kv, "page": page, "rope": rng.random() < 0.7}
    layers = _log(rng, 1, 32)
    if op == "fork":
        # page tables of some hundred sequences, the pool within a GiB
        row = layers * kv_heads * head_dim * 8
        beams = rng.randint(1, 16)
        seqs = max(1, min(_log(rng, 1, 24), (1 << 30) // (row * page * 3 * beams)))
        return {"op": op, "seqs": seqs, "beams": beams,
                "len": max(1, min(_log(rng, 1, 8000), (1 << 29) // (row * seqs))), "page": page,
                "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "kv": kv,
                "extra": rng.choice([1, 1, rng.randint(2, 70)])}
    tok = _log(rng, 1, 64)
    if op == "store":
        return {"op": op, "seqs": _log(rng, 1, 48), "tok": tok, "kv_heads": kv_heads,
                "head_dim": head_dim, "len": _log(rng, 1, 3000), "kv": kv, "page": page,
                "bias": rng.random() < 0.5}
    row = layers * kv_heads * head_dim * 8
    seqs = max(1, min(_log(rng, 1, 24), (1 << 29) // (row * 2 * (tok + page))))
    return {"op": op, "seqs": seqs, "tok": tok, "kv_heads": kv_heads, "head_dim": head_dim,
            "len": max(1, min(_log(rng, 1, 3000), (1 << 29) // (row * seqs) - tok)),
            "layers": layers, "kv": kv, "page": page}


# --------------------------------------------------------------------------- inputs


class _Made:
    """What prepare() keeps: plain attributes."""


def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values)).to(DEV)


def _lengths(case, r):
    n, most = case["seqs"], case["len"]
    if case.get("ragged") and n > 1:
        lens = [r.randint(max(0, most // 4), most) for _ in range(n)]
        lens[r.randrange(n)] = most
        return lens
    return [most] * n


def _tables(lens, page, r, share=0, spare=0):
    """Page tables of sequences of lens rows over a shuffled pool: int32 [n, ld], -1 past
    the end.  share: groups of that many sequences have all but their last pages in common."""
    need = [-(-x // page) for x in lens]
    ld = max(max(need), 1)
    table = np.full((len(lens), ld), -1, np.int32)
    n = 0
    for s, k in enumerate(need):
        common = 0
        if share and s % share:
            first = s - s % share
            common = max(0, min(k, need[first]) - 3)
            table[s, :common] = table[first, :common]
        table[s, common:k] = np.arange(n, n + k - common)
        n += k - common
    perm = np.array(r.sample(range(n + spare), n + spare), np.int32)
    return np.where(table >= 0, perm[table.clip(0)], -1).astype(np.int32), n + spare


def _pool(case, n_pages, g):
    kind, dtype = KV_TYPES[case["kv"]]
    shape = (case.get("layers", 1), n_pages, case["page"], case["kv_heads"], case["head_dim"])
    pools = []
    for _ in range(2):
        p = torch.empty(shape, dtype=dtype, device=DEV)
        for layer in range(shape[0]):
            p[layer] = torch.randn(shape[1:], generator=g, device=DEV)
        pools.append(p)
    return pools


def _tree(n, r):
    """Parents of n drafted tokens (-1: the text itself): a chain with side branches."""
    parent = [-1]
    for i in range(1, n):
        parent.append(i - 1 if r.random() < 0.5 else r.randint(-1, i - 1))
    return parent


def _tree_inputs(s, case, r):
    """Visibility masks, positions and counts of each sequence's drafted tokens."""
    n, t = case["seqs"], case["tok"]
    s.parents, mask = [], np.zeros((n, t), np.uint64)
    pos, count = np.zeros((n, t), np.int32), np.zeros(n, np.int32)
    for i in range(n):
        count[i] = t if i == 0 else r.randint(max(1, t // 2), t)
        p = _tree(t, r)
        s.parents.append(p)
        depth = [0] * t
        for j in range(t):
            mask[i, j] = np.uint64(1 << j) | (mask[i, p[j]] if p[j] >= 0 else np.uint64(0))
            depth[j] = depth[p[j]] + 1 if p[j] >= 0 else 0
        pos[i] = np.array(depth) + s.lens[i]
    s.mask, s.pos, s.n_tok = _ints(mask.view(np.int64)), _ints(pos), _ints(count)
    s.count = count


def _rope(s, head_dim, n_pos):
    p = torch.arange(n_pos, device=DEV, dtype=torch.float64)[:, None]
    f = 1e4 ** (-2.0 * torch.arange(head_dim // 2, device=DEV, dtype=torch.float64) / head_dim)
    s.cos, s.sin, s.n_pos = torch.cos(p * f).float(), torch.sin(p * f).float(), n_pos


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        torch.cuda.synchronize()  # the library's calls run on a stream of their own
    return s


def _inputs(case, seed):
    r = random.Random(int(seed) * 6007 + 5)
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    s = _Made()
    s.case = dict(case)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * std

    if case["op"] == "select":
        n, b, v = case["seqs"], case["beams"], case["vocab"]
        # a language model's logits: a few likely tokens above a broad rest
        s.logits = normal(n * b, v, std=2.0)
        hot = torch.randint(0, v, (n * b, 24), generator=g, device=DEV)
        s.logits.scatter_add_(1, hot, torch.rand(n * b, 24, generator=g, device=DEV) * 9)
        s.cum = -20 * torch.rand(n, b, generator=g, device=DEV)
        done = (torch.rand(n, b, generator=g, device=DEV) < 0.2).int()
        s.done = done if case["done"] else None
        s.eos = 2
        s.token = torch.zeros(n, case["keep"], dtype=torch.int32, device=DEV)
        s.parent = torch.zeros_like(s.token)
        s.score = torch.zeros(n, case["keep"], device=DEV)
        return s

    page = case["page"]
    if case["op"] == "fork":
        n, b = case["seqs"], case["beams"]
        lens = [max(1, r.randint(case["len"] * 3 // 4, case["len"])) for _ in range(n)]
        s.lens = [x for x in lens for _ in range(b)]  # beams of a text are equally long
        # enough free pages for every beam's copy and growth
        grow = -(-case["extra"] // page) + 1
        most = -(-case["len"] // page)
        n_pages = n * (most + (b - 1) * min(most, 3)) + n * b * grow
        ld = most + grow
        table = np.full((n * b, ld), -1, np.int32)
        held, used = _tables(s.lens, page, r, b)
        table[:, :held.shape[1]] = np.where(
            held >= 0, np.array(r.sample(range(n_pages), used), np.int32)[held.clip(0)], -1)
        refs = np.zeros(n_pages, np.int32)
        np.add.at(refs, table[table >= 0], 1)
        # each beam continues one of its text's, the better ones more often
        parent = [i * b + min(r.randrange(b), r.randrange(b)) for i in range(n) for _ in range(b)]
        s.k, s.v = _pool(case, n_pages, g)
        s.table, s.refs, s.parent = _ints(table), _ints(refs), _ints(np.array(parent, np.int32))
        s.len = _ints(np.array(s.lens, np.int32))
        s.table_out = torch.empty(n * b, ld, dtype=torch.int32, device=DEV)
        s.refs_out, s.info = torch.empty_like(s.refs), torch.zeros(3, dtype=torch.int32, device=DEV)
        return s

    n, t = case["seqs"], case["tok"]
    kvh, hd = case["kv_heads"], case["head_dim"]
    s.lens = _lengths(case, r)
    table, n_pages = _tables([x + t for x in s.lens], page, r, case.get("share", 0), 3)
    s.k, s.v = _pool(case, n_pages, g)
    s.table, s.len = _ints(table), _ints(np.array(s.lens, np.int32))
    if case["op"] == "compact":
        # accepted: one way down each tree, as a verified draft leaves it
        path, count = np.zeros((n, t), np.int32), np.zeros(n, np.int32)
        for i in range(n):
            way = sorted(r.sample(range(t), r.randint(max(1, t // 8), max(1, t // 2))))
            path[i, :len(way)], count[i] = way, len(way)
        s.path, s.n_path = _ints(path), _ints(count)
        s.len_out = torch.empty_like(s.len)
        return s
    _tree_inputs(s, case, r)
    _rope(s, hd, max(s.lens) + t)
    if case["op"] == "store":
        s.new_k, s.new_v = normal(n * t, kvh * hd), normal(n * t, kvh * hd)
        s.bk = normal(kvh * hd, std=0.3) if case["bias"] else None
        s.bv = normal(kvh * hd, std=0.3) if case["bias"] else None
        return s
    s.q = normal(n * t, case["heads"] * hd, std=1.5)
    s.out = torch.zeros(n * t, case["heads"] * hd, device=DEV)
    return s


# --------------------------------------------------------------------------- the passes


def run(state):
    op = state.case["op"]
    if own:
        return {"attn": _own_attn, "select": _own_select, "fork": _own_fork, "store": _own_store,
                "compact": _own_compact}[op](state)
    return {"attn": _plain_attn, "select": _plain_select, "fork": _plain_fork,
            "store": _plain_store, "compact": _plain_compact}[op](state)


def _handle(s):
    """The page pool as the library takes it, made once for a state."""
    if not hasattr(s, "pages"):
        from llm_core_amd import hip

        layers, n_pages, page, kvh, hd = s.k.shape
        s.pages = hip.KvPages(s.k.data_ptr(), s.v.data_ptr(), KV_TYPES[s.case["kv"]][0], layers,
                              n_pages, page, kvh, hd)
    return s.pages


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_attn(s):
    c = s.case
    rope = c["rope"]
    _context().attn_paged(
        s.out.data_ptr(), None, s.q.data_ptr(), _handle(s), 0, s.table.data_ptr(),
        s.table.shape[1], s.len.data_ptr(), c["seqs"], c["tok"], c["len"], c["heads"],
        n_tok=s.n_tok.data_ptr(), mask=s.mask.data_ptr() if c["tok"] > 1 else None,
        pos=s.pos.data_ptr() if rope else None, cos_t=s.cos.data_ptr(), sin_t=s.sin.data_ptr(),
        n_pos=s.n_pos)
    return s.out


def _own_select(s):
    c = s.case
    _context().beam_select(s.token.data_ptr(), s.parent.data_ptr(), s.score.data_ptr(),
                           s.logits.data_ptr(), c["vocab"], s.cum.data_ptr(), c["seqs"],
                           c["beams"], c["vocab"], c["keep"], done=_ptr(s.done), eos_id=s.eos)
    return s.token, s.parent, s.score


def _own_fork(s):
    n, ld = s.table.shape
    _context().kv_fork(_handle(s), s.table_out.data_ptr(), s.refs_out.data_ptr(),
                       s.info.data_ptr(), s.table.data_ptr(), s.refs.data_ptr(), n,
                       s.parent.data_ptr(), s.len.data_ptr(), n, ld, s.case["extra"])
    return s.table_out, s.refs_out, s.info, s.k, s.v


def _own_store(s):
    c = s.case
    _context().kv_store(_handle(s), 0, s.table.data_ptr(), s.table.shape[1], s.len.data_ptr(),
                        c["seqs"], c["tok"], s.new_k.data_ptr(), s.new_v.data_ptr(),
                        n_tok=s.n_tok.data_ptr(), bk=_ptr(s.bk), bv=_ptr(s.bv),
                        pos=s.pos.data_ptr(), cos_t=s.cos.data_ptr(), sin_t=s.sin.data_ptr(),
                        n_pos=s.n_pos)
    return s.k, s.v


def _own_compact(s):
    c = s.case
    _context().kv_compact(_handle(s), s.len_out.data_ptr(), s.table.data_ptr(), s.table.shape[1],
                          s.len.data_ptr(), s.path.data_ptr(), s.n_path.data_ptr(), c["seqs"],
                          c["tok"])
    return s.len_out, s.k, s.v


def _rotated(x, cos, sin):
    """Rotate-half RoPE of x [..., heads, hd] by cos/sin [..., 1, hd / 2]."""
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_attn(s):
    c = s.case
    n, t, kvh, hd = c["seqs"], c["tok"], c["kv_heads"], c["head_dim"]
    g = c["heads"] // kvh
    q = s.q.reshape(n, t, c["heads"], hd)
    if c["rope"]:
        p = s.pos.long()
        q = _rotated(q, s.cos[p][:, :, None], s.sin[p][:, :, None])
    q = (q / math.sqrt(hd)).reshape(n, t, kvh, g, hd).permute(0, 2, 1, 3, 4).reshape(
        n, kvh, t * g, hd)
    pages = s.table.clamp_min(0).long()
    k = s.k[0][pages].reshape(n, -1, kvh, hd).permute(0, 2, 3, 1).contiguous().float()
    sc = (q @ k).reshape(n, kvh, t, g, -1)
    at = torch.arange(sc.shape[-1], device=DEV)[None] - s.len[:, None]  # own tokens from 0
    drafted = (at >= 0) & (at < s.n_tok[:, None])
    bit = (s.mask[:, :, None] >> at.clamp(0, 63)[:, None]) & 1
    seen = (at < 0)[:, None] | (drafted[:, None] & (bit == 1))
    sc.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1)
    v = s.v[0][pages].reshape(n, -1, kvh, hd).permute(0, 2, 1, 3).contiguous().float()
    o = (p.reshape(n, kvh, t * g, -1) @ v).reshape(n, kvh, t, g, hd)
    o = o / torch.where(total == 0, 1.0, total)[..., None]
    o = o.permute(0, 2, 1, 3, 4).reshape(n, t, -1)
    live = torch.arange(t, device=DEV)[None] < s.n_tok[:, None]
    return torch.where(live[..., None], o, s.out.reshape(n, t, -1)).reshape(n * t, -1)


def _plain_select(s):
    c = s.case
    n, b, keep = c["seqs"], c["beams"], c["keep"]
    x, at = torch.sort(s.logits, dim=1, descending=True, stable=True)
    x = x.double()  # which continuation is better may hang on the last bits
    lse = x[:, :1] + torch.log(torch.exp(x - x[:, :1]).sum(1, keepdim=True))
    k = min(keep, c["vocab"])
    cum = s.cum.double().reshape(-1, 1)
    score, at = cum + (x[:, :k] - lse), at[:, :k]
    if s.done is not None:
        first = torch.arange(k, device=DEV)[None] == 0
        over = s.done.reshape(-1, 1) != 0
        score = torch.where(over, torch.where(first, cum, -math.inf), score)
        at = torch.where(over & first, s.eos, at)
    score, order = torch.sort(score.reshape(n, -1), dim=1, descending=True, stable=True)
    score, order = score[:, :keep], order[:, :keep]
    token, parent = at.reshape(n, -1).gather(1, order), order // k
    none = score == -math.inf
    token, parent = torch.where(none, -1, token), torch.where(none, -1, parent)
    short = keep - score.shape[1]
    if short:
        pad = lambda t, v: torch.cat([t, torch.full((n, short), v, device=DEV, dtype=t.dtype)], 1)  # noqa: E731
        token, parent, score = pad(token, -1), pad(parent, -1), pad(score, -math.inf)
    return token.int(), parent.int(), score.float()


def _plain_fork(s):
    """Pages as reference counts: what the old tables held is let go, what the new ones
    share is taken, then pages written to later are made their sequence's own."""
    page, extra, (n, ld) = s.case["page"], s.case["extra"], s.table.shape
    n_pages = s.refs.numel()
    col = torch.arange(ld, device=DEV)[None]
    one = torch.ones((), dtype=torch.int32, device=DEV)
    # one slot more takes what is no page
    refs = torch.cat([s.refs, one[None]])
    slot = lambda t: torch.where(t < 0, n_pages, t).long().reshape(-1)  # noqa: E731
    refs.index_put_((slot(s.table),), -one, accumulate=True)
    old = s.table[s.parent.long()]
    full = (s.len // page)[:, None]
    new = torch.where(col < full, old, -1)
    refs.index_put_((slot(new),), one, accumulate=True)
    # the page that is part full: its first continuation keeps it if nothing else holds it
    part = (s.len % page != 0)[:, None] & (col == full)
    mine = torch.where(part, old, -1).amax(1)
    who = torch.arange(n, device=DEV)
    first = torch.full((n_pages + 1,), n, device=DEV).scatter_reduce(0, slot(mine), who, "amin")
    keeps = (mine >= 0) & (first[slot(mine)] == who) & (refs[slot(mine)] == 0)
    new = torch.where(part & keeps[:, None], old, new)
    refs.index_put_((slot(torch.where(keeps, mine, -1)),), one, accumulate=True)
    # the rest comes from the free pages, the lowest first
    need = (s.len[:, None] + extra + page - 1) // page
    want = (col >= full) & (col < need) & (new < 0)
    rank = torch.cumsum(want.reshape(-1).int(), 0) - 1
    free = torch.sort(torch.where(refs[:n_pages] == 0, 0, 1), stable=True)[1].int()
    n_free = (refs[:n_pages] == 0).sum()
    got = torch.where(rank < n_free, free[rank.clamp(0, n_pages - 1)], -1).reshape(n, ld)
    new = torch.where(want, got, new)
    refs.index_put_((slot(torch.where(want, got, -1)),), one, accumulate=True)
    to = torch.where(part & want, new, -1).amax(1)
    copied = (mine >= 0) & (to >= 0)
    # rows of the kept part; the others stay what they are
    src, dst = torch.where(copied, mine, 0).long(), torch.where(copied, to, 0).long()
    src, dst, rows = src[copied], dst[copied], (s.len % page)[copied]
    live = (torch.arange(page, device=DEV)[None] < rows[:, None])[None, :, :, None, None]
    s.k[:, dst] = torch.where(live, s.k[:, src], s.k[:, dst])
    s.v[:, dst] = torch.where(live, s.v[:, src], s.v[:, dst])
    total = want.sum()
    info = torch.stack([copied.sum(), (total - n_free).clamp_min(0), (n_free - total).clamp_min(0)])
    return new, refs[:n_pages], info.int(), s.k, s.v


def _slots(s, at):
    """Pool rows (flat) of the cache positions at [n, ...]."""
    page = s.case["page"]
    return s.table.long().gather(1, at // page) * page + at % page


def _plain_store(s):
    c = s.case
    n, t, kvh, hd = c["seqs"], c["tok"], c["kv_heads"], c["head_dim"]
    k, v = s.new_k, s.new_v
    if s.bk is not None:
        k, v = k + s.bk, v + s.bv
    p = s.pos.long()
    k = _rotated(k.reshape(n, t, kvh, hd), s.cos[p][:, :, None], s.sin[p][:, :, None])
    idx = torch.arange(t, device=DEV)[None]
    to = _slots(s, s.len[:, None].long() + idx)[idx < s.n_tok[:, None]]
    live = (idx < s.n_tok[:, None]).reshape(-1)
    s.k[0].reshape(-1, kvh, hd)[to] = k.reshape(n * t, kvh, hd)[live].to(s.k.dtype)
    s.v[0].reshape(-1, kvh, hd)[to] = v.reshape(n * t, kvh, hd)[live].to(s.v.dtype)
    return s.k, s.v


def _plain_compact(s):
    layers, _, _, kvh, hd = s.k.shape
    idx = torch.arange(s.path.shape[1], device=DEV)[None]
    live = idx < s.n_path[:, None]
    base = s.len[:, None].long()
    src, dst = _slots(s, base + s.path.long())[live], _slots(s, base + idx)[live]
    k, v = s.k.reshape(layers, -1, kvh, hd), s.v.reshape(layers, -1, kvh, hd)
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    return s.len + s.n_path, s.k, s.v


# --------------------------------------------------------------------------- what it takes


def _moved(case):
    """Expected pages that a fork copies and rows in them."""
    b = case["beams"]
    return case["seqs"] * b * 0.5, case["page"] / 2


def work(case):
    size = 4 if case.get("kv") == "f32" else 2
    if case["op"] == "select":
        rows = case["seqs"] * case["beams"]
        return {"bytes": rows * case["vocab"] * 4 + case["seqs"] * case["keep"] * 12,
                "flops": 4 * rows * case["vocab"]}
    row = case["kv_heads"] * case["head_dim"]
    if case["op"] == "fork":
        pages, rows = _moved(case)
        n, ld = case["seqs"] * case["beams"], case["len"] // case["page"] + 1
        return {"bytes": pages * rows * row * size * 4 * case["layers"] + n * ld * 8, "flops": n * ld}
    n, t = case["seqs"], case["tok"]
    if case["op"] == "store":
        return {"bytes": n * t * row * 2 * (4 + size), "flops": n * t * row * 4}
    if case["op"] == "compact":
        moved = n * max(1, t * 0.3)
        return {"bytes": moved * row * size * 4 * case["layers"], "flops": moved * row}
    keys = case["len"] * (0.625 if case["ragged"] and n > 1 else 1.0) + t
    texts = n / case["share"] if case["share"] else n
    texts = max(1.0, texts)
    tail = (n - texts) * min(keys, 3.0 * case["page"])
    q = n * t * case["heads"] * case["head_dim"]
    return {"bytes": (texts * keys + tail) * row * size * 2 + q * 8,
            "flops": 4 * n * (0.75 * t if t > 1 and n > 1 else t) * case["heads"] * keys * case["head_dim"]}


# --------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "select": _exact_select, "fork": _exact_fork,
            "store": _exact_store, "compact": _exact_compact}[case["op"]](s)


def _turn64(s, x, pos):
    """x [heads, hd] at a position, rotated pair by pair."""
    half = x.shape[-1] // 2
    c, w = s.cos[pos].double(), s.sin[pos].double()
    out = torch.empty_like(x)
    out[:, :half] = x[:, :half] * c - x[:, half:] * w
    out[:, half:] = x[:, half:] * c + x[:, :half] * w
    return out


def _rows64(s, pool, i, count):
    pages = s.table[i, :-(-count // s.case["page"])].long()
    return torch.cat([pool[0, p] for p in pages.tolist()])[:count].double()


def _exact_attn(s):
    c = s.case
    t, hd, g = c["tok"], c["head_dim"], c["heads"] // c["kv_heads"]
    out = s.out.double().reshape(c["seqs"], t, c["heads"], hd).clone()
    for i in range(c["seqs"]):
        held, drafted = s.lens[i], int(s.count[i])
        k, v = (_rows64(s, x, i, held + drafted).permute(1, 0, 2) for x in (s.k, s.v))
        see = torch.zeros(drafted, held + drafted, dtype=torch.bool)
        see[:, :held] = True
        for j in range(drafted):
            a = j
            while a >= 0:
                see[j, held + a] = True
                a = s.parents[i][a]
        q = s.q.double().reshape(c["seqs"], t, c["heads"], hd)[i, :drafted]
        if c["rope"]:
            q = torch.stack([_turn64(s, q[j], int(s.pos[i, j])) for j in range(drafted)])
        see = see.to(DEV)
        for h in range(c["heads"]):
            w = q[:, h] @ k[h // g].T.contiguous() / hd ** 0.5
            w = torch.softmax(w.masked_fill(~see, -math.inf), 1)
            out[i, :drafted, h] = w @ v[h // g]
    return out.reshape(c["seqs"] * t, -1)


def _exact_select(s):
    c = s.case
    n, b, v, keep = c["seqs"], c["beams"], c["vocab"], c["keep"]
    x = s.logits.cpu().numpy().astype(np.float64).reshape(n, b, v)
    cum = s.cum.cpu().numpy().astype(np.float64)
    done = np.zeros((n, b)) if s.done is None else s.done.cpu().numpy()
    token, parent = np.full((n, keep), -1, np.int32), np.full((n, keep), -1, np.int32)
    score = np.full((n, keep), -np.inf)
    for i in range(n):
        cands = []
        for j in range(b):
            if done[i, j]:
                cands.append((-cum[i, j], j, 0.0, s.eos))
                continue
            most = x[i, j].max()
            lse = most + math.log(np.exp(x[i, j] - most).sum())
            edge = np.partition(x[i, j], max(0, v - keep))[max(0, v - keep)]
            for w in np.nonzero(x[i, j] >= edge)[0]:
                cands.append((-(cum[i, j] + (x[i, j, w] - lse)), j, -x[i, j, w], int(w)))
        for r, (a, j, _, w) in enumerate(sorted(cands)[:keep]):
            token[i, r], parent[i, r], score[i, r] = w, j, -a
    return torch.from_numpy(token), torch.from_numpy(parent), torch.from_numpy(score)


def _exact_fork(s):
    page, extra, (n, ld) = s.case["page"], s.case["extra"], s.table.shape
    old, parent, lens = s.table.cpu().numpy(), s.parent.tolist(), s.lens
    refs = s.refs.cpu().numpy().copy()
    for p in old[old >= 0]:
        refs[p] -= 1
    new = np.full((n, ld), -1, np.int32)
    for i in range(n):
        for j in range(lens[i] // page):
            new[i, j] = old[parent[i], j]
            refs[new[i, j]] += 1
    taken, copies, short = set(), [], 0
    for i in range(n):
        j = lens[i] // page
        p = old[parent[i], j] if lens[i] % page else -1
        if p >= 0 and p not in taken and refs[p] == 0:
            new[i, j] = p
        taken.add(p)
    for i in range(n):
        j = lens[i] // page
        if new[i, j] >= 0:
            refs[new[i, j]] += 1
    free = [p for p in range(len(refs)) if refs[p] == 0]
    for i in range(n):
        for j in range(lens[i] // page, -(-(lens[i] + extra) // page)):
            if new[i, j] >= 0:
                continue
            if not free:
                short += 1
                continue
            new[i, j] = free.pop(0)
            refs[new[i, j]] += 1
            if j == lens[i] // page and lens[i] % page:
                copies.append((old[parent[i], j], new[i, j], lens[i] % page))
    k, v = s.k.clone(), s.v.clone()
    for a, b, rows in copies:
        k[:, int(b), :rows], v[:, int(b), :rows] = s.k[:, int(a), :rows], s.v[:, int(a), :rows]
    info = torch.tensor([len(copies), short, len(free)], dtype=torch.int32)
    return torch.from_numpy(new), torch.from_numpy(refs), info, k.double(), v.double()


def _exact_store(s):
    c = s.case
    kvh, hd, page = c["kv_heads"], c["head_dim"], c["page"]
    table = s.table.cpu().numpy()
    k, v = s.k.double(), s.v.double()
    nk, nv = (x.double().reshape(c["seqs"], c["tok"], kvh, hd) for x in (s.new_k, s.new_v))
    bk, bv = (0 if x is None else x.double().reshape(kvh, hd) for x in (s.bk, s.bv))
    for i in range(c["seqs"]):
        for j in range(int(s.count[i])):
            at = s.lens[i] + j
            p, r = int(table[i, at // page]), at % page
            k[0, p, r] = _turn64(s, nk[i, j] + bk, int(s.pos[i, j]))
            v[0, p, r] = nv[i, j] + bv
    return k, v


def _exact_compact(s):
    page, table = s.case["page"], s.table.cpu().numpy()
    k, v = s.k.double(), s.v.double()
    lens = []
    for i, held in enumerate(s.lens):
        way = s.path[i, :int(s.n_path[i])].tolist()
        lens.append(held + len(way))
        for a, b in enumerate(way):
            to, at = held + a, held + b
            k[:, table[i, to // page], to % page] = s.k[:, table[i, at // page], at % page].double()
            v[:, table[i, to // page], to % page] = s.v[:, table[i, at // page], at % page].double()
    return torch.tensor(lens, dtype=torch.int32), k, v
