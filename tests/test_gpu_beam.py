"""Beam search's selection on the device against a 64-bit restatement (paged_ref)."""
import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


def run(ctx, logits, cum, done, eos, n_out, ld=None, shift=0):
    n, B, V = logits.shape
    ld = ld or V
    x = np.full(n * B * ld + shift, 1e30, np.float32)  # behind the rows: never read as logits
    for r, row in enumerate(logits.reshape(-1, V)):
        x[shift + r * ld:shift + r * ld + V] = row
    i0, f0 = np.full((n, n_out), 99, np.int32), np.zeros((n, n_out), np.float32)
    with R.Device(ctx) as d:
        t, p, s = d.up(i0), d.up(i0), d.up(f0)
        ctx.beam_select(t, p, s, d.up(x) + 4 * shift, ld, d.up(cum), n, B, V, n_out,
                        done=None if done is None else d.up(done), eos_id=eos)
        return d.get(t, i0), d.get(p, i0), d.get(s, f0)


def check(got, logits, cum, done, eos, n_out):
    wt, wp, ws = R.select(logits, cum, done, eos, n_out)
    assert np.array_equal(got[0], wt), (got[0], wt)
    assert np.array_equal(got[1], wp)
    assert np.array_equal(np.isfinite(got[2]), np.isfinite(ws))
    fine = np.isfinite(ws)
    # scores are computed to some 1e-12 and rounded to fp32 once
    assert np.all(np.abs(got[2][fine] - ws[fine]) <= 2.0 ** -24 * np.abs(ws[fine]) + 1e-11)


def logits_of(kind, shape, rng):
    x = (rng.standard_normal(shape) * 3).astype(np.float32)
    if kind == "ascending":
        return np.sort(x, -1)
    if kind == "descending":
        return np.sort(x, -1)[..., ::-1].copy()
    if kind == "blocked":  # the largest with few threads
        x[..., :400] += 30
        return x
    if kind == "strided":
        for e in range(4):
            x[..., e::256] += 40
        return x
    if kind == "equal":
        return np.full(shape, -1.25, np.float32)
    if kind == "few":  # ties, and both zeros
        return rng.choice(np.array([0.0, -0.0, 1.0, 2.0], np.float32), shape)
    if kind == "masked":
        x[rng.random(shape) < 0.9] = -np.inf
        x[rng.random(shape) < 0.02] = np.finfo(np.float32).min
        return x
    return x


KINDS = ["normal", "ascending", "descending", "blocked", "strided", "equal", "few", "masked"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [1, 2, 63, 257, 2048, 2049, 32003])
def test_select(ctx, V, kind):
    rng = np.random.default_rng(V)
    for n, B, n_out in ((1, 1, 1), (1, 4, 8), (3, 5, 10), (2, 16, 16), (1, 3, 64)):
        x = logits_of(kind, (n, B, V), rng)
        cum = (-20 * rng.random((n, B))).astype(np.float32)
        check(run(ctx, x, cum, None, -1, n_out), x, cum, None, -1, n_out)
        done = (rng.random((n, B)) < 0.3).astype(np.int32) * 7
        eos = int(rng.integers(0, V))
        ld = V + int(rng.integers(1, 9))
        got = run(ctx, x, cum, done, eos, n_out, ld=ld, shift=int(rng.integers(0, 4)))
        check(got, x, cum, done, eos, n_out)


@pytest.mark.parametrize("kind", ["normal", "ascending", "equal", "masked"])
@pytest.mark.parametrize("n,B,V,n_out", [(2, 16, 8000, 32), (4, 16, 60000, 32), (3, 20, 4099, 40),
                                         (1, 33, 9001, 33), (2, 64, 2500, 64), (1, 64, 17001, 63)])
def test_select_many_kept(ctx, n, B, V, n_out, kind):
    """n_out no small part of a wave: bounds by 64 lists leave more than can be ranked."""
    rng = np.random.default_rng(n_out + V)
    x = logits_of(kind, (n, B, V), rng)
    for spread in (0.5, 40.0):
        cum = (-spread * rng.random((n, B))).astype(np.float32)
        done = (rng.random((n, B)) < 0.2).astype(np.int32)
        check(run(ctx, x, cum, done, 5, n_out), x, cum, done, 5, n_out)


@pytest.mark.parametrize("n,B,V,n_out", [(2, 8, 151936, 16), (1, 64, 32000, 64), (40, 2, 4099, 4),
                                         (1, 1, 300001, 64)])
def test_select_large(ctx, n, B, V, n_out):
    rng = np.random.default_rng(B)
    x = logits_of("normal", (n, B, V), rng)
    cum = (-5 * rng.random((n, B))).astype(np.float32)
    check(run(ctx, x, cum, None, -1, n_out), x, cum, None, -1, n_out)


def test_first_step(ctx):
    """All beams alike, all but the first unused."""
    rng = np.random.default_rng(2)
    x = np.repeat(rng.standard_normal((2, 1, 1000)).astype(np.float32), 4, 1)
    cum = np.full((2, 4), -np.inf, np.float32)
    cum[:, 0] = 0
    got = run(ctx, x, cum, None, -1, 8)
    assert not got[1].any()
    check(got, x, cum, None, -1, 8)


def test_identical_beams_rank_by_beam(ctx):
    rng = np.random.default_rng(3)
    x = np.repeat(rng.standard_normal((1, 1, 5000)).astype(np.float32), 6, 1)
    cum = np.full((1, 6), -3.5, np.float32)
    got = run(ctx, x, cum, None, -1, 12, ld=5003, shift=1)  # rows of every alignment
    assert got[1].tolist() == [[0, 1, 2, 3, 4, 5] * 2]
    check(got, x, cum, None, -1, 12)


def test_close_scores(ctx):
    """Beams whose continuations differ by less than fp32 could tell."""
    rng = np.random.default_rng(4)
    x = np.repeat(rng.standard_normal((1, 1, 2000)).astype(np.float32), 8, 1)
    order = rng.permutation(8)
    for b in range(8):  # one far-off logit more or less likely: sums apart in the 9th digit
        x[0, b, 7] = np.float32(-12.0 - 0.01 * order[b])
    cum = np.full((1, 8), -1.0, np.float32)
    check(run(ctx, x, cum, None, -1, 24), x, cum, None, -1, 24)


def test_no_distribution(ctx):
    """Rows of -inf, with NaN, with +inf, beams at -inf or NaN: no continuations."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 7, 3000)).astype(np.float32)
    x[0, 0] = -np.inf
    x[0, 1, 2999] = np.nan
    x[0, 2, 17] = np.inf
    x[0, 6] = -np.inf
    x[0, 6, 2500] = np.nan  # in a chunk without a finite logit
    cum = np.zeros((1, 7), np.float32)
    cum[0, 3], cum[0, 5] = -np.inf, np.nan
    got = run(ctx, x, cum, None, -1, 16)
    assert np.all(got[1] == 4)
    x64 = x.copy()
    cum64 = np.where(np.isnan(cum), -np.inf, cum)
    check(got, x64, cum64, None, -1, 16)
    cum[:] = -np.inf
    got = run(ctx, x, cum, np.ones((1, 7), np.int32), 4, 16)
    assert np.all(got[0] == -1) and np.all(got[1] == -1) and np.all(got[2] == -np.inf)


def test_all_done(ctx):
    x = np.zeros((1, 3, 50), np.float32)
    cum = np.array([[-3.0, -1.0, -1.0]], np.float32)
    got = run(ctx, x, cum, np.ones((1, 3), np.int32), 9, 5)
    assert got[0].tolist() == [[9, 9, 9, -1, -1]]
    assert got[1].tolist() == [[1, 2, 0, -1, -1]]
    assert got[2].tolist() == [[-1.0, -1.0, -3.0, -np.inf, -np.inf]]


def test_scores_over_the_beams_own(ctx):
    """score is cum: a search's running scores in one array."""
    rng = np.random.default_rng(7)
    n, B, V = 9, 5, 4099
    x = rng.standard_normal((n, B, V)).astype(np.float32)
    cum = -rng.random((n, B)).astype(np.float32)
    i0 = np.zeros((n, B), np.int32)
    with R.Device(ctx) as d:
        t, p, s = d.up(i0), d.up(i0), d.up(cum)
        ctx.beam_select(t, p, s, d.up(x), V, s, n, B, V, B)
        check((d.get(t, i0), d.get(p, i0), d.get(s, cum)), x, cum, None, -1, B)


def test_many_rows(ctx):
    """More rows than a grid's second dimension holds."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((1100, 60, 40)).astype(np.float32)
    cum = -rng.random((1100, 60)).astype(np.float32)
    check(run(ctx, x, cum, None, -1, 3), x, cum, None, -1, 3)


def test_same_bits_each_time(ctx):
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((4, 8, 32000)) * 2).astype(np.float32)
    cum = -rng.random((4, 8)).astype(np.float32)
    a = run(ctx, x, cum, None, -1, 16)
    for _ in range(3):
        b = run(ctx, x, cum, None, -1, 16)
        assert all(np.array_equal(p.view(np.uint32), q.view(np.uint32)) for p, q in zip(a, b))


def test_closest_scores(ctx):
    """Pairs of beams some 1e-13 apart, by exponentials of unlike arguments: log(1 + e^a) against
    log(1 + e^b + e^c + e^d)."""
    rng = np.random.default_rng(9)
    n = 1024
    e64 = lambda v: np.exp(v.astype(np.float64))  # noqa: E731
    a = -0.01 - 0.7 * rng.random(n).astype(np.float32)
    b = a + np.log(0.2 + 0.6 * rng.random(n)).astype(np.float32)
    c = np.log(e64(a) - e64(b) - 4e-7).astype(np.float32)
    # what is left of e^a: d's fp32 steps, 9.5e-7, are some 4e-13 of the sum
    d = np.log(e64(a) - e64(b) - e64(c)).astype(np.float32)
    x = np.full((n, 2, 4), -np.inf, np.float32)
    x[:, 0, 0], x[:, 0, 1] = 0, a
    x[:, 1] = np.stack([np.zeros(n, np.float32), b, c, d], 1)
    lse = np.log(np.exp(x.astype(np.float64)).sum(-1))
    gap = np.abs(lse[:, 0] - lse[:, 1])
    # exponentials to 3e-15 of their values, sums and logarithms of at most 1.1 to 1e-15 more
    pick = np.flatnonzero((gap > 2e-14) & (gap < 5e-13))
    assert len(pick) > n // 2, len(pick)
    x = np.ascontiguousarray(x[pick])
    cum = np.zeros((len(pick), 2), np.float32)
    got = run(ctx, x, cum, None, -1, 2)
    first = (lse[pick, 1] < lse[pick, 0]).astype(np.int32)
    assert not got[0].any()
    assert np.array_equal(got[1], np.stack([first, 1 - first], 1)), (
        np.count_nonzero(got[1][:, 0] != first), len(pick))
