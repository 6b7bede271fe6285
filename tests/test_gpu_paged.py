"""The cache in pages on the device, against 64-bit restatements (paged_ref)."""
import numpy as np
import pytest

import paged_ref as R
from llm_core_amd import hip
from oracle import oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32


class Case:
    """Inputs of one attention call on the host."""

    def __init__(self, seed, heads, kvh, hd, kv, page, lens, n_tok, max_tok, mask="tree", rope=True,
                 bias=False, layers=2, layer=1, spare=2, q_std=1.5):
        r = self.rng = np.random.default_rng(seed)
        self.heads, self.kvh, self.hd, self.page, self.kv = heads, kvh, hd, page, kv
        self.lens, self.n_tok, self.max_tok = np.array(lens, np.int32), np.array(n_tok, np.int32), max_tok
        self.n, self.layer, self.layers = len(lens), layer, layers
        total = [a + b for a, b in zip(lens, n_tok)]
        self.ld = max(1, max(-(-t // page) for t in total)) + 1
        self.n_pages = sum(-(-t // page) for t in total) + spare
        self.table = R.tables(total, page, self.ld, self.n_pages, r)
        self.type, dt = R.KV[kv]
        shape = (layers, self.n_pages, page, kvh, hd)
        self.k = r.standard_normal(shape).astype(dt)
        self.v = r.standard_normal(shape).astype(dt)
        self.q = (r.standard_normal((self.n, max_tok, heads, hd)) * q_std).astype(np.float32)
        self.bq = (r.standard_normal((heads, hd)) * 0.3).astype(np.float32) if bias else None
        self.rope = rope
        self.pos = np.zeros((self.n, max_tok), np.int32)
        self.mask = np.zeros((self.n, max_tok), np.uint64)
        self.no_mask = mask is None
        for s in range(self.n):
            if mask == "tree":
                m, depth = hip.tree_masks(R.tree(max_tok, r))
            elif mask == "random":  # any set of the drafted rows, none at all too
                m = r.integers(0, 2 ** 63, max_tok, dtype=np.uint64) * (r.random(max_tok) < 0.7)
                depth = r.integers(0, max_tok, max_tok)
            else:
                m, depth = hip.tree_masks(np.arange(max_tok) - 1)
            self.mask[s], self.pos[s] = m, depth + lens[s]
        self.cos, self.sin = hip.rope_table(hd, 1e4, max(total) + max_tok + 1)
        self.n_pos = max(total) + max_tok + 1

    def turned_q(self):
        q = self.q.astype(np.float64)
        if self.bq is not None:
            q = q + self.bq
        if self.rope:
            c = self.cos.reshape(self.n_pos, -1)
            w = self.sin.reshape(self.n_pos, -1)
            for s in range(self.n):
                for i in range(self.max_tok):
                    q[s, i] = R.turned(q[s, i], int(self.pos[s, i]), c, w)
        return q

    def want(self):
        return R.attention(self.turned_q(), self.k, self.v, self.table, self.lens, self.n_tok,
                           self.mask, self.page, self.heads, self.layer)

    def run(self, ctx, max_len=None, q8=False, q_pad=0):
        row = self.heads * self.hd
        with R.Device(ctx) as d:
            q = np.full((self.n * self.max_tok, row + q_pad), 1e30, np.float32)
            q[:, :row] = self.q.reshape(-1, row)
            out0 = np.full((self.n * self.max_tok, row), 777.0, np.float32)
            q80 = np.full((self.n * self.max_tok, row // 32 * 36), 0xa5, np.uint8)
            out, oq = d.up(out0), d.up(q80) if q8 else None
            kv = hip.KvPages(d.up(self.k), d.up(self.v), self.type, self.layers, self.n_pages,
                             self.page, self.kvh, self.hd)
            ctx.attn_paged(out, oq, d.up(q), kv, self.layer, d.up(self.table), self.ld,
                           d.up(self.lens), self.n, self.max_tok,
                           int(self.lens.max()) if max_len is None else max_len, self.heads,
                           q_ld=row + q_pad, bq=None if self.bq is None else d.up(self.bq),
                           n_tok=d.up(self.n_tok),
                           mask=None if self.no_mask else d.up(self.mask),
                           pos=d.up(self.pos) if self.rope else None, cos_t=d.up(self.cos),
                           sin_t=d.up(self.sin), n_pos=self.n_pos)
            got = d.get(out, out0).reshape(self.n, self.max_tok, self.heads, self.hd)
            return (got, d.get(oq, q80).reshape(self.n, self.max_tok, -1)) if q8 else got

    def check(self, got, want, size):
        """Against the 64-bit result.  A score is a sum of hd products and its q a rotation
        of fp32 values, each rounded by at most U: off by (hd + 6) U sum|q k| / sqrt(hd) at
        the most, which changes a weight by that part of it; weights and the sum over n
        rows add n + 16 roundings.  Both numerator and denominator: twice."""
        live = np.arange(self.max_tok)[None] < self.n_tok[:, None]
        assert np.all(got[~live] == 777.0), "rows past n_tok were written"
        rows = int((self.lens + self.n_tok).max())
        kmax = np.abs(np.nan_to_num(self.k[self.layer].astype(np.float64), posinf=0, neginf=0)).sum(-1)
        qk = np.abs(self.turned_q()).max() * kmax.max() / np.sqrt(self.hd)
        per = 2 * ((self.hd + 6) * U * min(qk, 60.0) + (rows + 16) * U)
        a, b, size = got[live].astype(np.float64), want[live], size[live]
        fine = np.isfinite(b)
        assert np.array_equal(fine, np.isfinite(a))
        assert np.array_equal(b[~fine], a[~fine], equal_nan=True)
        assert np.all(np.abs(a - b)[fine] <= per * size[fine] + 1e-30), float(
            np.max(np.abs(a - b)[fine] / (size[fine] + 1e-30)))
        # the errors are independent, so norm-wise they stay far below their bound: scores up
        # to 16 off by 2 U of themselves make 2e-6
        if fine.all() and b.size and np.linalg.norm(b):
            rel = np.linalg.norm(a - b) / np.linalg.norm(b)
            print(f"  norm-wise {rel:.2e}", flush=True)
            assert rel <= 2e-6


SHAPES = [(4, 2, 64), (16, 2, 128), (8, 8, 64), (7, 1, 128), (16, 4, 256), (18, 2, 64), (32, 1, 128)]


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_attn_single_tokens(ctx, heads, kvh, hd, kv):
    """Decode steps: one token a sequence over 0, 1 and odd lengths."""
    c = Case(heads * hd, heads, kvh, hd, kv, 16, [0, 1, 15, 16, 17, 33, 255, 700],
             [1, 1, 1, 1, 1, 1, 1, 0], 1, mask=None)
    c.check(c.run(ctx), *c.want())


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("mask", ["tree", "random", None])
@pytest.mark.parametrize("heads,kvh,hd,tok,page", [
    (4, 2, 64, 2, 8), (8, 2, 128, 5, 16), (8, 1, 128, 16, 32), (6, 3, 64, 33, 64),
    (16, 2, 128, 64, 16), (4, 4, 256, 17, 1), (16, 2, 256, 31, 128), (14, 2, 64, 48, 2)])
def test_attn_trees(ctx, heads, kvh, hd, tok, page, mask, kv):
    c = Case(tok, heads, kvh, hd, kv, page, [0, 40, 129, 1], [tok, max(1, tok // 2), tok, 0], tok,
             mask=mask, bias=True)
    c.check(c.run(ctx, q_pad=12), *c.want())


@pytest.mark.parametrize("tok", [1, 3, 24])
@pytest.mark.parametrize("kv,hd", [("f32", 128), ("f16", 128), ("f32", 64), ("f32", 256)])
def test_attn_long(ctx, tok, kv, hd):
    """Lengths that the work is split over, whatever the caller's estimate of them."""
    c = Case(7, 8, 2, hd, kv, 16, [3001, 64, 1023], [tok, tok, max(1, tok - 1)], tok, rope=False)
    want = c.want()
    for max_len in (3001, 0, 100000, 700):
        c.check(c.run(ctx, max_len=max_len), *want)


@pytest.mark.parametrize("heads,kvh,hd,tok,kv", [
    (32, 8, 128, 48, "f32"), (16, 2, 64, 40, "f32"), (24, 4, 128, 43, "f16"),
    (8, 2, 256, 37, "f32"), (28, 4, 64, 64, "f16"), (32, 4, 128, 64, "f32")])
def test_attn_row_tiles(ctx, heads, kvh, hd, tok, kv):
    """Rows that fill their last tile by a little, by half, more and in full, in sequences
    of one call, with their keys split over many workgroups and over few."""
    c = Case(heads + tok, heads, kvh, hd, kv, 16, [2003, 701, 0, 95], [tok, tok - 17, 1, tok], tok,
             mask="tree")
    want = c.want()
    for max_len in (2003, 0):
        c.check(c.run(ctx, max_len=max_len), *want)


@pytest.mark.parametrize("tok", [1, 20])
def test_attn_q8(ctx, tok):
    """outq8 holds the Q8_0 blocks of out, bit for bit; rows past n_tok stay."""
    c = Case(3, 8, 2, 128, "f32", 16, [300, 5, 0], [tok, 1, max(1, tok // 2)], tok)
    got, q8 = c.run(ctx, q8=True)
    c.check(got, *c.want())
    for s in range(c.n):
        for i in range(c.max_tok):
            if i < c.n_tok[s]:
                assert np.array_equal(q8[s, i], O.quantize_q8_0(got[s, i].reshape(-1)))
            else:
                assert np.all(q8[s, i] == 0xa5)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads,kvh,hd", [(6, 3, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("tok", [1, 5, 40])
def test_attn_q8_of_all_heads(ctx, heads, kvh, hd, tok, kv):
    """Q8_0 blocks of every head dimension and page type; a row that sees nothing is blocks of
    zeros."""
    c = Case(hd + tok, heads, kvh, hd, kv, 16, [300, 0, 0], [tok, 1, max(1, tok // 2)], tok)
    c.mask[1, 0] = 0
    for max_len in (300, 0):
        got, q8 = c.run(ctx, q8=True, max_len=max_len)
        c.check(got, *c.want())
        assert not got[1, 0].any() and not q8[1, 0].any()
        for s in range(c.n):
            for i in range(c.max_tok):
                if i < c.n_tok[s]:
                    assert np.array_equal(q8[s, i], O.quantize_q8_0(got[s, i].reshape(-1)))
                else:
                    assert np.all(q8[s, i] == 0xa5)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("tok", [1, 7, 40])
def test_attn_masked_places_change_nothing(ctx, tok, kv):
    """NaN and infinities in unused rows of used pages, in unused pages, in other layers and in
    drafted rows that a token does not see."""
    c = Case(11, 8, 2, 128, kv, 16, [37, 5, 0], [tok, max(1, tok // 2), tok], tok)
    for i in range(tok):  # node 1 on: its own branch only; node 0's row is seen by itself alone
        c.mask[:, i] = np.uint64(1 << i)
    want, size = c.want()
    rng = np.random.default_rng(5)
    held = np.zeros((c.n_pages, c.page), bool)
    for s in range(c.n):
        for j in range(c.lens[s] + c.n_tok[s]):
            held[R.slot(c.table[s], j, c.page, c.n_pages)] = True
    junk = np.array([np.nan, np.inf, -np.inf, 65504.0], c.k.dtype)
    for x in (c.k, c.v):
        x[0] = np.nan
        x[1][~held] = rng.choice(junk, x[1][~held].shape)
    c.check(c.run(ctx), want, size)
    if tok > 1:
        # a NaN row that only token 0 sees: every other token's result stays the same
        at = R.slot(c.table[0], c.lens[0], c.page, c.n_pages)
        c.k[1][at], c.v[1][at] = np.nan, np.inf
        got = c.run(ctx)
        assert np.isnan(got[0, 0]).all()
        want[0, 0], got[0, 0] = 0, 0
        size[0, 0] = 0
        c.check(got, want, size)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("tok", [1, 9])
def test_attn_infinities_in_sight(ctx, tok, kv):
    """What the formula gives: a score of -inf has no weight, one of +inf or NaN makes the row NaN,
    a value of +-inf the element."""
    c = Case(13, 4, 2, 64, kv, 16, [50, 50, 50, 50], [tok] * 4, tok, rope=False)
    c.q[:] = np.abs(c.q)
    spot = [R.slot(c.table[s], 20, c.page, c.n_pages) for s in range(4)]
    c.k[1][spot[0]] = -np.inf
    c.k[1][spot[1]] = np.inf
    c.v[1][spot[2]][:, 5] = np.inf
    c.v[1][spot[2]][:, 9] = -np.inf
    c.k[1][spot[3]][0, 3] = np.nan
    with np.errstate(all="ignore"):
        want, size = c.want()
    want[1], size[1] = np.nan, np.nan
    want[3][:, :2] = np.nan  # KV head 0's query heads
    c.check(c.run(ctx), want, size)


@pytest.mark.parametrize("tok", [1, 12])
def test_attn_magnitudes(ctx, tok):
    """Keys from 1e-6 to 1e4 of one row next to queries that even them out, values over the whole
    range of fp32: no digits are lost to a shared scale."""
    c = Case(17, 4, 2, 128, "f32", 16, [90, 33], [tok, tok], tok, rope=False)
    scale = (10.0 ** np.linspace(-6, 4, 128)).astype(np.float32)
    c.k *= scale
    c.q /= scale
    c.v *= (10.0 ** np.linspace(-30, 30, 128)).astype(np.float32)
    want, size = c.want()
    got = c.run(ctx)
    live = np.arange(tok)[None] < c.n_tok[:, None]
    # per score: (hd + 6) U sum|q_d k_d| / sqrt(hd), |q_d k_d| at most 6 sigma squares apart
    a, b = got[live], want[live]
    assert np.all(np.abs(a - b) <= 2 * ((134) * U * 40 + 110 * U) * size[live])
    rel = np.abs(a - b) / size[live]
    assert np.sqrt(np.mean(rel ** 2)) <= 2e-6


def test_attn_bad_tables(ctx):
    """Entries that are no page hold no rows; lengths past the table are cut to it."""
    c = Case(19, 4, 2, 64, "f32", 16, [100, 100, 100], [4, 4, 4], 4)
    c.table[0, 2], c.table[1, 3], c.table[1, 0] = -1, c.n_pages, 2 ** 31 - 1
    c.table[2, :] = -7
    want, size = c.want()
    assert not want[2].any()
    c.check(c.run(ctx), want, size)
    c.lens[:] = [2 ** 31 - 1, -5, 100]
    got = c.run(ctx, max_len=2 ** 31 - 1)
    cut = Case(19, 4, 2, 64, "f32", 16, [100, 100, 100], [4, 4, 4], 4)
    cut.table, cut.lens = c.table, np.array([c.ld * 16, 0, 100], np.int32)
    cut.n_pos, cut.cos, cut.sin, cut.pos = c.n_pos, c.cos, c.sin, c.pos
    cut.check(got, *cut.want())


def test_attn_shared_pages(ctx):
    """Sequences whose tables name the same pages, one of them the same page twice."""
    c = Case(23, 8, 2, 128, "f16", 16, [200, 200, 64], [1, 1, 1], 1)
    c.table[1, :10] = c.table[0, :10]
    c.table[2, 1] = c.table[2, 0]
    c.check(c.run(ctx), *c.want())


@pytest.mark.parametrize("tok", [1, 3])
def test_attn_many_sequences(ctx, tok):
    """More sequences than one launch deals out, some of them empty."""
    rng = np.random.default_rng(47)
    n = 700
    lens = np.where(rng.random(n) < 0.2, 0, rng.integers(0, 60, n))
    lens[[0, 255, 256, 511, 699]] = [200, 33, 150, 0, 90]
    n_tok = np.where(rng.random(n) < 0.1, 0, rng.integers(1, tok + 1, n))
    c = Case(48, 4, 2, 64, "f16", 8, lens.tolist(), n_tok.tolist(), tok, mask=None)
    c.check(c.run(ctx), *c.want())


@pytest.mark.parametrize("heads,tok", [(64, 1), (64, 5), (40, 13)])
def test_attn_one_kv_head(ctx, heads, tok):
    """Every query head on one KV head: row tiles of several kinds, partly filled."""
    c = Case(heads, heads, 1, 64, "f32", 1024, [1500, 20], [tok, max(1, tok - 1)], tok)
    c.check(c.run(ctx), *c.want())


def test_attn_same_bits_each_time(ctx):
    c = Case(29, 32, 8, 128, "f32", 16, [2500, 40], [24, 24], 24)
    a = c.run(ctx)
    for _ in range(3):
        assert np.array_equal(a.view(np.uint32), c.run(ctx).view(np.uint32))


def test_attn_offsets_past_32_bits(ctx):
    """Rows behind 2^32 bytes and 2^31 values of a layer."""
    kvh, hd, page = 8, 128, 1024
    n_pages = 2100  # 8.8 GB of K and V each
    row = kvh * hd
    k, v = ctx.alloc(n_pages * page * row * 4), ctx.alloc(n_pages * page * row * 4)
    try:
        c = Case(31, 8, 8, hd, "f32", page, [2000, 30], [1, 3], 3, layers=1, layer=0)
        far = {int(p): n_pages - 1 - i for i, p in enumerate(c.table[c.table >= 0])}
        table = c.table.copy()
        for p, f in far.items():
            table[c.table == p] = f
            for pool, data in ((k, c.k), (v, c.v)):
                ctx.write(pool.at(f * page * row * 4), data[0, p])
        with R.Device(ctx) as d:
            out0 = np.full((c.n * 3, 8 * hd), 777.0, np.float32)
            out = d.up(out0)
            kv = hip.KvPages(k, v, 0, 1, n_pages, page, kvh, hd)
            ctx.attn_paged(out, None, d.up(c.q), kv, 0, d.up(table), c.ld, d.up(c.lens), 2, 3, 2000,
                           8, n_tok=d.up(c.n_tok), mask=d.up(c.mask), pos=d.up(c.pos),
                           cos_t=d.up(c.cos), sin_t=d.up(c.sin), n_pos=c.n_pos)
            c.check(d.get(out, out0).reshape(2, 3, 8, hd), *c.want())
    finally:
        for b in (k, v):
            b.free()
            ctx._bufs.remove(b)


# ---- store ---------------------------------------------------------------------


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("kvh,hd,tok,page,rope,bias", [
    (2, 128, 1, 16, True, True), (8, 64, 5, 8, True, False), (3, 256, 17, 32, False, True),
    (1, 64, 64, 1, True, True), (8, 128, 7, 16, False, False)])
def test_store(ctx, kvh, hd, tok, page, rope, bias, kv):
    rng = np.random.default_rng(tok * hd)
    lens = np.array([0, 3, page * 2 - 1, 50, 9], np.int32)
    n_tok = np.array([tok, max(1, tok // 2), tok, 0, tok], np.int32)
    n, row = len(lens), kvh * hd
    ld = max(-(-(int(x) + tok) // page) for x in lens) + 1
    n_pages = n * ld
    table = R.tables([ld * page] * n, page, ld, n_pages, rng)
    table[4, :] = [-1, n_pages] * (ld // 2) + [-1] * (ld % 2)  # nowhere to go
    kind, dt = R.KV[kv]
    k0 = rng.standard_normal((2, n_pages, page, kvh, hd)).astype(dt)
    v0 = rng.standard_normal(k0.shape).astype(dt)
    xk = rng.standard_normal((n * tok, row + 4)).astype(np.float32)
    xv = rng.standard_normal((n * tok, row + 8)).astype(np.float32)
    bk, bv = (rng.standard_normal(row).astype(np.float32) for _ in range(2))
    cos, sin = hip.rope_table(hd, 1e4, 80)
    pos = rng.integers(0, 80, (n, tok)).astype(np.int32)
    pos[0, 0], pos[1, 0] = -3, 4000  # cut to the table
    with R.Device(ctx) as d:
        k, v = d.up(k0), d.up(v0)
        ctx.kv_store(hip.KvPages(k, v, kind, 2, n_pages, page, kvh, hd), 1, d.up(table), ld,
                     d.up(lens), n, tok, d.up(xk), d.up(xv), k_ld=row + 4, v_ld=row + 8,
                     n_tok=d.up(n_tok), bk=d.up(bk) if bias else None,
                     bv=d.up(bv) if bias else None, pos=d.up(pos) if rope else None,
                     cos_t=d.up(cos), sin_t=d.up(sin), n_pos=80)
        gk, gv = d.get(k, k0), d.get(v, v0)
    wk, wv = k0.astype(np.float64), v0.astype(np.float64)
    size = np.zeros_like(wk)
    c, w = cos.reshape(80, -1), sin.reshape(80, -1)
    for s in range(n):
        for i in range(n_tok[s]):
            at = R.slot(table[s], int(lens[s]) + i, page, n_pages)
            if at is None:
                continue
            a = xk[s * tok + i, :row].astype(np.float64) + (bk if bias else 0)
            size[1][at] = np.abs(a).reshape(kvh, hd)
            if rope:
                half = np.abs(a).reshape(kvh, 2, hd // 2).sum(1)
                size[1][at] = np.concatenate([half, half], -1)
                a = R.turned(a.reshape(kvh, hd), int(np.clip(pos[s, i], 0, 79)), c, w)
            wk[1][at] = a.reshape(kvh, hd)
            wv[1][at] = (xv[s * tok + i, :row].astype(np.float64) +
                         (bv if bias else 0)).reshape(kvh, hd)
    step = U if kv == "f32" else 2.0 ** -11
    assert np.array_equal(gk[0], k0[0]) and np.array_equal(gv[0], v0[0])
    # K: the bias, two products and a sum (4 U of their size), then the page's rounding;
    # fp16 below its normal range: half its smallest step
    assert np.all(np.abs(gk - wk) <= 4 * U * size + step * np.abs(wk) + 2.0 ** -25 * (kv == "f16"))
    assert np.all(np.abs(gv - wv) <= 2 * U * np.abs(wv) + step * np.abs(wv) + U * 4 +
                  2.0 ** -25 * (kv == "f16"))
    still = size[1] == 0
    assert np.array_equal(gk[1][still], k0[1][still])


# ---- fork ----------------------------------------------------------------------


def run_fork(ctx, kind, dt, pool_k, pool_v, table, refs, parent, lens, page, extra, in_place=False):
    layers, n_pages, _, kvh, hd = pool_k.shape
    n, ld = len(parent), table.shape[1]
    with R.Device(ctx) as d:
        k, v, r = d.up(pool_k), d.up(pool_v), d.up(refs)
        t0, i0 = np.full((n, ld), 99, np.int32), np.full(3, 99, np.int32)
        t, i = d.up(t0), d.up(i0)
        r1 = r if in_place else d.up(np.full_like(refs, 99))
        ctx.kv_fork(hip.KvPages(k, v, kind, layers, n_pages, page, kvh, hd), t, r1, i, d.up(table),
                    r, len(table), d.up(np.array(parent, np.int32)),
                    d.up(np.array(lens, np.int32)), n, ld, extra)
        if not in_place:
            assert np.array_equal(d.get(r, refs), refs)
        return d.get(t, t0), d.get(r1, refs), d.get(i, i0), d.get(k, pool_k), d.get(v, pool_v)


def check_fork(got, pool_k, pool_v, table, refs, parent, lens, page, extra):
    t, r, info, k, v = got
    wt, wr, wi, copies = R.fork(table, refs, parent, lens, page, extra, table.shape[1])
    assert np.array_equal(t, wt) and np.array_equal(r, wr) and np.array_equal(info, wi)
    wk, wv = pool_k.copy(), pool_v.copy()
    for a, b, rows in copies:
        wk[:, b, :rows], wv[:, b, :rows] = pool_k[:, a, :rows], pool_v[:, a, :rows]
    assert np.array_equal(k, wk) and np.array_equal(v, wv)
    return copies


@pytest.mark.parametrize("extra", [0, 1, 40])
@pytest.mark.parametrize("page", [1, 4, 16, 64])
@pytest.mark.parametrize("kv", ["f32", "f16"])
def test_fork_random(ctx, kv, page, extra):
    """Rounds of forks after each other, parents at random: dropped, repeated, cut back, out of
    range; other holders of some pages; sometimes too few free pages."""
    kind, dt = R.KV[kv]
    rng = np.random.default_rng(page * 100 + extra)
    for trial in range(6):
        n, n_pages = int(rng.integers(1, 30)), int(rng.integers(60, 400))
        ld = 1 + 200 // page
        k = rng.standard_normal((2, n_pages, page, 1, 64)).astype(dt)
        v = rng.standard_normal(k.shape).astype(dt)
        table = np.full((n, ld), -1, np.int32)
        refs = np.zeros(n_pages, np.int32)
        refs[rng.integers(0, n_pages, 5)] += 1  # held by somebody else
        lens = np.zeros(n, np.int32)
        total = 0
        for step in range(5):
            m = int(rng.integers(1, 30))
            parent = rng.integers(-1, n + 1, m).astype(np.int32)
            ln = np.array([lens[p] if 0 <= p < n else 7 for p in parent], np.int32)
            ln[rng.random(m) < 0.2] //= 2
            ln[rng.random(m) < 0.05] = -1
            got = run_fork(ctx, kind, dt, k, v, table, refs, parent, ln, page, extra,
                           in_place=step % 2 == 1)
            total += len(check_fork(got, k, v, table, refs, parent, ln, page, extra))
            table, refs, _, k, v = got
            n = m
            held = (table >= 0).sum(1) * page  # rows that the pages there are hold
            room = np.maximum(ln, 0) + extra
            lens = np.minimum(np.minimum(room, held), 190).astype(np.int32)
        if extra == 1 and page > 1:  # 40 more rows end on whole pages of 4 most times
            assert total > 0


def test_fork_tables_of_several_hundred(ctx):
    """More sequences and pages than threads walk in one step."""
    rng = np.random.default_rng(1)
    n, page, ld, n_pages = 1500, 4, 12, 20000
    lens = rng.integers(0, 41, n).astype(np.int32)
    table = R.tables(lens, page, ld, n_pages, rng)
    refs = np.zeros(n_pages, np.int32)
    np.add.at(refs, table[table >= 0], 1)
    k = rng.standard_normal((1, n_pages, page, 1, 64)).astype(np.float32)
    parent = np.minimum(rng.integers(0, n, n), rng.integers(0, n, n)).astype(np.int32)
    got = run_fork(ctx, 0, np.float32, k, k, table, refs, parent, lens[parent], page, 3)
    assert len(check_fork(got, k, k, table, refs, parent, lens[parent], page, 3)) > 200


@pytest.mark.parametrize("n_pages", [32768, 32769])
def test_fork_large_pools(ctx, n_pages):
    """Reference counts in LDS and past what LDS holds."""
    rng = np.random.default_rng(n_pages)
    n, page, ld = 40, 2, 500
    lens = rng.integers(0, 900, n).astype(np.int32)
    table = R.tables(lens, page, ld, n_pages, rng)
    refs = np.zeros(n_pages, np.int32)
    np.add.at(refs, table[table >= 0], 1)
    k = rng.standard_normal((1, n_pages, page, 1, 64)).astype(np.float16)
    parent = rng.integers(0, n, 60).astype(np.int32)
    for in_place in (False, True):
        got = run_fork(ctx, 1, np.float16, k, k, table, refs, parent, lens[parent], page, 5, in_place)
        check_fork(got, k, k, table, refs, parent, lens[parent], page, 5)


def test_fork_partial_page_held_in_full_by_a_sibling(ctx):
    """A sequence cut back into a page that its sibling still holds whole gets a copy."""
    k = np.arange(1 * 6 * 16 * 64, dtype=np.float32).reshape(1, 6, 16, 1, 64)
    table = np.array([[4, 2, 1]], np.int32)
    refs = np.array([0, 1, 1, 0, 1, 0], np.int32)
    got = run_fork(ctx, 0, np.float32, k, k, table, refs, [0, 0], [20, 48], 16, 1)
    check_fork(got, k, k, table, refs, [0, 0], [20, 48], 16, 1)
    assert got[0].tolist() == [[4, 0, -1], [4, 2, 1]]


def test_fork_nothing(ctx):
    k = np.ones((1, 3, 2, 1, 64), np.float32)
    refs = np.array([1, 1, 0], np.int32)
    got = run_fork(ctx, 0, np.float32, k, k, np.array([[1, -1]], np.int32), refs, [-1], [0], 2, 1)
    assert got[0].tolist() == [[-1, -1]] and got[1].tolist() == [1, 0, 0]
    assert got[2].tolist() == [0, 0, 2]


# ---- compaction -----------------------------------------------------------------


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("kvh,hd,page,layers", [(2, 64, 4, 3), (8, 128, 16, 2), (1, 256, 1, 1),
                                                (5, 64, 64, 2)])
def test_compact(ctx, kvh, hd, page, layers, kv):
    kind, dt = R.KV[kv]
    rng = np.random.default_rng(hd + page)
    paths = [[], [0], [5], [0, 1, 2, 3], [1, 2, 3], [0, 3, 4, 9, 30, 63], list(range(64)),
             list(range(0, 64, 2)), [3, 3, 4], [4, 2, 9], [2, 70, 71], [-1, 4]]
    n, mp = len(paths), 64
    lens = rng.integers(0, 100, n).astype(np.int32)
    ld = -(-(100 + 64) // page)
    n_pages = n * ld + 1
    table = R.tables([ld * page] * n, page, ld, n_pages, rng)
    table[5, -1] = -1
    path, count = np.full((n, mp), 7, np.int32), np.zeros(n, np.int32)
    for s, p in enumerate(paths):
        path[s, :len(p)], count[s] = p, len(p)
    k0 = rng.standard_normal((layers, n_pages, page, kvh, hd)).astype(dt)
    v0 = rng.standard_normal(k0.shape).astype(dt)
    wk, wv, wl = k0.copy(), v0.copy(), lens.copy()
    for s, p in enumerate(paths):
        last = -1
        for i, b in enumerate(p):
            if b <= last or b >= 64:  # the path ends before it
                break
            last = b
            wl[s] += 1
            src = R.slot(table[s], lens[s] + b, page, n_pages)
            dst = R.slot(table[s], lens[s] + i, page, n_pages)
            if src and dst:
                wk[(slice(None),) + dst] = k0[(slice(None),) + src]
                wv[(slice(None),) + dst] = v0[(slice(None),) + src]
    for in_place in (False, True):
        with R.Device(ctx) as d:
            k, v, ln = d.up(k0), d.up(v0), d.up(lens)
            lo = ln if in_place else d.up(np.zeros_like(lens))
            ctx.kv_compact(hip.KvPages(k, v, kind, layers, n_pages, page, kvh, hd), lo, d.up(table),
                           ld, ln, d.up(path), d.up(count), n, mp)
            assert np.array_equal(d.get(lo, lens), wl)
            assert np.array_equal(d.get(k, k0), wk) and np.array_equal(d.get(v, v0), wv)


# ---- together -------------------------------------------------------------------


def test_draft_verify_compact_decode(ctx):
    """A drafted tree's life: room (fork), store, attention, the accepted way compacted, the rest
    given back, the next token decoded; its attention is that of the contiguous cache
    (axf_hip_attn_decode) over the accepted tokens."""
    rng = np.random.default_rng(41)
    heads, kvh, hd, page, T, held = 8, 2, 128, 16, 13, 75
    row, n_pages, ld = kvh * hd, 12, 8
    parent = R.tree(T, rng)
    mask, depth = hip.tree_masks(parent)
    way = [T - 1]
    while parent[way[0]] >= 0:
        way.insert(0, int(parent[way[0]]))
    total = held + T
    xk, xv = (rng.standard_normal((held + T + 1, row)).astype(np.float32) for _ in range(2))
    cos, sin = hip.rope_table(hd, 1e4, 256)
    with R.Device(ctx) as d:
        pk, pv = (d.up(np.full((1, n_pages, page, kvh, hd), np.nan, np.float32)) for _ in range(2))
        kv = hip.KvPages(pk, pv, 0, 1, n_pages, page, kvh, hd)
        refs, info = d.up(np.zeros(n_pages, np.int32)), d.up(np.zeros(3, np.int32))
        ta, tb = (d.up(np.full((1, ld), -1, np.int32)) for _ in range(2))
        one = d.up(np.zeros(1, np.int32))
        dc, ds = d.up(cos), d.up(sin)

        def fork(src, dst, length, extra):
            ctx.kv_fork(kv, dst, refs, info, src, refs, 1, one, length, 1, ld, extra)

        def store(table, length, k, v, pos, n):
            ctx.kv_store(kv, 0, table, ld, length, 1, n, d.up(k), d.up(v),
                         pos=d.up(np.array(pos, np.int32)), cos_t=dc, sin_t=ds, n_pos=256)

        zero = d.up(np.zeros(1, np.int32))
        fork(ta, tb, zero, held)
        store(tb, zero, xk[:held], xv[:held], range(held), held)
        length = d.up(np.array([held], np.int32))
        fork(tb, ta, length, T)
        store(ta, length, xk[held:total], xv[held:total], depth + held, T)
        q = rng.standard_normal((T, heads * hd)).astype(np.float32)
        out0 = np.zeros((T, heads * hd), np.float32)
        out = d.up(out0)
        ctx.attn_paged(out, None, d.up(q), kv, 0, ta, ld, length, 1, T, held, heads, mask=d.up(mask),
                       pos=d.up((depth + held).astype(np.int32)), cos_t=dc, sin_t=ds, n_pos=256)
        tree_out = d.get(out, out0)
        path = np.zeros((1, T), np.int32)
        path[0, :len(way)] = way
        ctx.kv_compact(kv, length, ta, ld, length, d.up(path), d.up(np.array([len(way)], np.int32)),
                       1, T)
        now = held + len(way)
        assert d.get(length, np.zeros(1, np.int32))[0] == now
        fork(ta, tb, length, 1)
        assert d.get(info, np.zeros(3, np.int32)).tolist() == [0, 0, n_pages - (now // page + 1)]
        store(tb, length, xk[total:], xv[total:], [now], 1)
        q1 = rng.standard_normal((1, heads * hd)).astype(np.float32)
        ctx.attn_paged(out, None, d.up(q1), kv, 0, tb, ld, length, 1, 1, now, heads,
                       pos=d.up(np.array([now], np.int32)), cos_t=dc, sin_t=ds, n_pos=256)
        last = d.get(out, out0)[0]

        # the same over a contiguous cache of the accepted rows
        def contiguous(rows, positions, query, at):
            k = np.stack([R.turned(xk[r].reshape(kvh, hd).astype(np.float64), p, cos.reshape(256, -1),
                                   sin.reshape(256, -1)) for r, p in zip(rows, positions)])
            k = k.astype(np.float32).reshape(len(rows), row)
            turned = R.turned(query.reshape(heads, hd).astype(np.float64), at, cos.reshape(256, -1),
                              sin.reshape(256, -1)).astype(np.float32)
            o0 = np.zeros(heads * hd, np.float32)
            o = d.up(o0)
            ctx.attn_decode(o, None, d.up(turned), d.up(k), d.up(xv[rows]), len(rows), heads, kvh, hd)
            return d.get(o, o0)

        rows = list(range(held)) + [held + w for w in way]
        positions = list(range(held)) + [held + i for i in range(len(way))]
        want = contiguous(rows + [total], positions + [now], q1, now)
        # two fp32 evaluations of one formula, each norm-wise within 2e-6 of it (Case.check),
        # keys turned in fp32 here and in 64 bits there: 4 U of a score's terms
        assert np.linalg.norm(last - want) <= 5e-6 * np.linalg.norm(want)
        for n, w in enumerate(way):
            want = contiguous(rows[:held + n + 1], positions[:held + n + 1], q[w], held + n)
            assert np.linalg.norm(tree_out[w] - want) <= 5e-6 * np.linalg.norm(want)


def test_beam_search(ctx):
    """Whole beam searches of a small random model on the device (store, attention, selection,
    fork), against a 64-bit search that keeps each beam's rows apart."""
    rng = np.random.default_rng(43)
    heads, kvh, hd, V, B, n, steps, page = 4, 2, 64, 211, 3, 2, 12, 4
    row, E = kvh * hd, heads * hd
    wq, wk, wv = (rng.standard_normal((V, x)).astype(np.float32) for x in (E, row, row))
    head = (rng.standard_normal((V, E)) * 0.6).astype(np.float32)
    eos, n_pages, ld = 5, 64, 8
    cos, sin = hip.rope_table(hd, 1e4, 64)
    c2, s2 = cos.reshape(64, -1), sin.reshape(64, -1)
    S = n * B
    with R.Device(ctx) as d:
        pk, pv = (d.up(np.zeros((1, n_pages, page, kvh, hd), np.float32)) for _ in range(2))
        kv = hip.KvPages(pk, pv, 0, 1, n_pages, page, kvh, hd)
        refs, info = d.up(np.zeros(n_pages, np.int32)), d.up(np.zeros(3, np.int32))
        t = [d.up(np.full((S, ld), -1, np.int32)) for _ in range(2)]
        dc, ds = d.up(cos), d.up(sin)
        i0, f0 = np.zeros(S, np.int32), np.zeros(S, np.float32)
        tok_d, par_d, sc_d = d.up(i0), d.up(i0), d.up(f0)
        out0 = np.zeros((S, E), np.float32)
        out = d.up(out0)
        tokens = np.array([[17] * B, [90] * B], np.int32)
        cum = np.full((n, B), -np.inf, np.float32)
        cum[:, 0] = 0
        cum64 = cum.astype(np.float64)
        done = np.zeros((n, B), np.int32)
        parent = np.arange(S, dtype=np.int32)
        seen = [[[] for _ in range(B)] for _ in range(n)]  # the tokens behind each beam
        for step in range(steps):
            length = d.up(np.full(S, step, np.int32))
            ctx.kv_fork(kv, t[1], refs, info, t[0], refs, S, d.up(parent), length, S, ld, 1)
            t.reverse()
            assert d.get(info, np.zeros(3, np.int32))[1] == 0
            flat = tokens.reshape(-1)
            pos = d.up(np.full(S, step, np.int32))
            ctx.kv_store(kv, 0, t[0], ld, length, S, 1, d.up(wk[flat]), d.up(wv[flat]), pos=pos,
                         cos_t=dc, sin_t=ds, n_pos=64)
            ctx.attn_paged(out, None, d.up(wq[flat]), kv, 0, t[0], ld, length, S, 1, step, heads,
                           pos=pos, cos_t=dc, sin_t=ds, n_pos=64)
            logits = d.get(out, out0) @ head.T
            ctx.beam_select(tok_d, par_d, sc_d, d.up(logits.astype(np.float32)), V, d.up(cum), n, B,
                            V, B, done=d.up(done), eos_id=eos)
            got = [d.get(x, y).reshape(n, B) for x, y in ((tok_d, i0), (par_d, i0), (sc_d, f0))]
            # in 64 bits: every beam's own rows
            want64 = np.zeros((n, B, V))
            for s in range(n):
                for b in range(B):
                    way = seen[s][b] + [int(tokens[s, b])]
                    k = np.stack([R.turned(wk[x].reshape(kvh, hd).astype(np.float64), p, c2, s2)
                                  for p, x in enumerate(way)])
                    q = R.turned(wq[way[-1]].reshape(heads, hd).astype(np.float64), step, c2, s2)
                    o = []
                    for h in range(heads):
                        sc = k[:, h // 2] @ q[h] / np.sqrt(hd)
                        w = np.exp(sc - sc.max())
                        o.append(w @ wv[way].reshape(-1, kvh, hd)[:, h // 2].astype(np.float64) / w.sum())
                    want64[s, b] = head.astype(np.float64) @ np.concatenate(o)
            wt, wp, ws = R.select(want64, cum64, done, eos, B)
            assert np.array_equal(got[0], wt) and np.array_equal(got[1], wp), step
            assert np.allclose(got[2], ws, rtol=1e-5, atol=1e-4)
            seen = [[seen[s][p] + [int(tokens[s, p])] for p in wp[s]] for s in range(n)]
            done = np.take_along_axis(done, wp, 1) | (wt == eos)
            tokens, cum, cum64 = wt, got[2], ws
            parent = (wp + np.arange(n)[:, None] * B).reshape(-1).astype(np.int32)
        assert len({tuple(x) for x in seen[0]}) == B
