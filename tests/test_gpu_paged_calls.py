"""Calls for several continuations as the header allows them and other tests do not make: arrays
at 4-byte alignment, two contexts at once, head counts and vocabularies at their limits."""
import numpy as np
import pytest

import paged_ref as R
from llm_core_amd import hip
from test_gpu_paged import U, Case

pytestmark = pytest.mark.gpu


def off(d, a, by=4):
    """The array on the device, `by` bytes behind a 16-byte boundary."""
    raw = np.frombuffer(np.ascontiguousarray(a).tobytes(), np.uint8)
    return d.up(np.concatenate([np.zeros(by, np.uint8), raw])) + by


def put(ctx, d, c, shift):
    """Case.run's call without its wait: (out, what it was)."""
    up = lambda a: off(d, a, shift)  # noqa: E731
    out0 = np.full((c.n * c.max_tok, c.heads * c.hd), 777.0, np.float32)
    out = up(out0)
    kv = hip.KvPages(d.up(c.k), d.up(c.v), c.type, c.layers, c.n_pages, c.page, c.kvh, c.hd)
    args = dict(bq=None if c.bq is None else up(c.bq), n_tok=up(c.n_tok),
                mask=None if c.no_mask else d.up(c.mask), pos=up(c.pos) if c.rope else None,
                cos_t=up(c.cos), sin_t=up(c.sin), n_pos=c.n_pos)
    q, table, lens = up(c.q), up(c.table), up(c.lens)

    def go():
        ctx.attn_paged(out, None, q, kv, c.layer, table, c.ld, lens, c.n, c.max_tok,
                       int(c.lens.max()), c.heads, **args)

    return go, lambda: d.get(out, out0).reshape(c.n, c.max_tok, c.heads, c.hd)


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads,kvh,hd,tok", [(7, 1, 128, 1), (8, 2, 64, 9), (8, 2, 256, 20),
                                              (16, 2, 128, 33)])
def test_attn_words_not_aligned(ctx, heads, kvh, hd, tok, kv):
    c = Case(tok, heads, kvh, hd, kv, 16, [301, 17, 0], [tok, 1, tok], tok, bias=True)
    want = c.want()
    for shift in (4, 8, 12):
        with R.Device(ctx) as d:
            go, get = put(ctx, d, c, shift)
            go()
            c.check(get(), *want)


def test_store_words_not_aligned(ctx):
    rng = np.random.default_rng(3)
    kvh, hd, page, n_pages, tok = 2, 128, 8, 6, 5
    row = kvh * hd
    k0 = np.zeros((1, n_pages, page, kvh, hd), np.float32)
    xk, xv = (rng.standard_normal((tok, row + 1)).astype(np.float32) for _ in range(2))
    bk, bv = (rng.standard_normal(row).astype(np.float32) for _ in range(2))
    table, lens = np.array([[4, 2, 0]], np.int32), np.array([6], np.int32)
    for shift in (4, 8, 12):
        with R.Device(ctx) as d:
            k, v = d.up(k0), d.up(k0)
            ctx.kv_store(hip.KvPages(k, v, 0, 1, n_pages, page, kvh, hd), 0, off(d, table, shift), 3,
                         off(d, lens, shift), 1, tok, off(d, xk, shift), off(d, xv, shift),
                         k_ld=row + 1, v_ld=row + 1, bk=off(d, bk, shift), bv=off(d, bv, shift))
            gk, gv = d.get(k, k0), d.get(v, k0)
        wk, wv = k0.copy(), k0.copy()
        for i in range(tok):
            p, r = R.slot(table[0], 6 + i, page, n_pages)
            wk[0, p, r] = (xk[i, :row] + bk).reshape(kvh, hd)
            wv[0, p, r] = (xv[i, :row] + bv).reshape(kvh, hd)
        assert np.array_equal(gk, wk) and np.array_equal(gv, wv)


def test_two_contexts_at_once(ctx):
    """Calls of two contexts, enqueued by turns and waited for together: each has its own
    workspace, and the same bits as alone."""
    other = hip.Context(0)
    cases = [Case(s, 16, 2, 128, "f32", 16, [1500, 700, 33], [t] * 3, t, rope=False)
             for s, t in ((5, 1), (6, 24))]
    rng = np.random.default_rng(8)
    x = rng.standard_normal((2, 4, 20011)).astype(np.float32)
    cum = -rng.random((2, 4)).astype(np.float32)
    i0, f0 = np.zeros((2, 8), np.int32), np.zeros((2, 8), np.float32)
    try:
        alone = [c.run(ctx) for c in cases]
        with R.Device(ctx) as d, R.Device(other) as e:
            calls = [put(ctx, d, cases[0], 0), put(other, e, cases[1], 0)]
            outs = []
            for cx, dev in ((ctx, d), (other, e)):
                t, p, s = dev.up(i0), dev.up(i0), dev.up(f0)
                outs.append((cx, t, p, s, dev.up(x), dev.up(cum)))
            for _ in range(10):
                for (go, _get), (cx, t, p, s, lx, lc) in zip(calls, outs):
                    go()
                    cx.beam_select(t, p, s, lx, 20011, lc, 2, 4, 20011, 8)
            for (_, get), want in zip(calls, alone):
                assert np.array_equal(get().view(np.uint32), want.view(np.uint32))
            wt, wp, _ = R.select(x, cum, None, -1, 8)
            for (cx, t, p, *_), dev in zip(outs, (d, e)):
                assert np.array_equal(dev.get(t, i0), wt) and np.array_equal(dev.get(p, i0), wp)
    finally:
        other.close()


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("tok", [1, 6, 40])
def test_attn_queries_of_zero(ctx, tok, kv):
    """All scores alike, of either sign of zero: the mean of what a token sees."""
    c = Case(tok, 4, 2, 128, kv, 16, [203, 0, 31], [tok, tok, 1], tok, rope=False)
    c.q[:] = 0.0
    c.q[0, :, ::2] = -0.0
    c.check(c.run(ctx), *c.want())


@pytest.mark.parametrize("heads,kvh,tok", [(1024, 1, 3), (256, 256, 2), (1024, 256, 1)])
def test_attn_most_heads(ctx, heads, kvh, tok):
    c = Case(heads, heads, kvh, 64, "f16", 16, [50, 0], [tok, tok], tok, layers=1, layer=0)
    c.check(c.run(ctx), *c.want())


def test_select_largest_vocabulary(ctx):
    """2^26 logits: equal but for some, the last among them."""
    V = 1 << 26
    x = np.zeros((1, 1, V), np.float32)
    hot = {V - 1: 5.0, 0: 4.0, V // 2 + 1: 4.0, 12345: 3.0, V - 4097: 2.0}
    for t, v in hot.items():
        x[0, 0, t] = v
    lse = np.log((V - len(hot)) + np.exp(np.array(list(hot.values()))).sum())
    i0, f0 = np.zeros((1, 8), np.int32), np.zeros((1, 8), np.float32)
    with R.Device(ctx) as d:
        t, p, s = d.up(i0), d.up(i0), d.up(f0)
        ctx.beam_select(t, p, s, d.up(x), V, d.up(np.zeros((1, 1), np.float32)), 1, 1, V, 8)
        token, score = d.get(t, i0)[0], d.get(s, f0)[0]
    assert token.tolist() == [V - 1, 0, V // 2 + 1, 12345, V - 4097, 1, 2, 3]
    # 2^26 exponentials of at most 3e-15 each off, and the rounding to fp32
    assert np.all(np.abs(score - (x[0, 0, token] - lse)) <= U * 20)


def test_select_infinite_beam(ctx):
    """A score of +inf is a score: all of its beam's tokens come first, by their logits."""
    rng = np.random.default_rng(12)
    x = rng.standard_normal((1, 3, 700)).astype(np.float32)
    cum = np.array([[-1.0, np.inf, -2.0]], np.float32)
    i0, f0 = np.zeros((1, 5), np.int32), np.zeros((1, 5), np.float32)
    with R.Device(ctx) as d:
        t, p, s = d.up(i0), d.up(i0), d.up(f0)
        ctx.beam_select(t, p, s, d.up(x), 700, d.up(cum), 1, 3, 700, 5)
        assert d.get(t, i0)[0].tolist() == np.argsort(-x[0, 1], kind="stable")[:5].tolist()
        assert np.all(d.get(p, i0) == 1) and np.all(d.get(s, f0) == np.inf)


def test_select_scores_past_fp32(ctx):
    """Masks of the type's lowest value, taken twice: the token is there, its score is -inf, and the
    beam is no candidate in the next step."""
    low = np.finfo(np.float32).min
    x = np.full((1, 2, 40), low, np.float32)
    x[0, 0, 7], x[0, 1, 3] = 0.0, 0.0
    cum = np.array([[-1.0, low]], np.float32)
    i0, f0 = np.zeros((1, 2), np.int32), np.zeros((1, 2), np.float32)
    with R.Device(ctx) as d:
        t, p, s = d.up(i0), d.up(i0), d.up(cum)
        lx = d.up(x)
        ctx.beam_select(t, p, s, lx, 40, s, 1, 2, 40, 2)
        assert d.get(t, i0).tolist() == [[7, 0]] and d.get(p, i0).tolist() == [[0, 0]]
        assert d.get(s, f0).tolist() == [[-1.0, low]]
        one = d.up(np.array([[low, -np.inf]], np.float32))
        y = d.up(np.full((1, 2, 40), low, np.float32) + np.eye(2, 40, dtype=np.float32)[None] * -low)
        ctx.beam_select(t, p, s, y, 40, one, 1, 2, 40, 2)
        # beam 0: its unmasked token, then a masked one at twice the lowest value
        assert d.get(t, i0).tolist() == [[0, 1]] and d.get(p, i0).tolist() == [[0, 0]]
        assert d.get(s, f0).tolist() == [[low, -np.inf]]
