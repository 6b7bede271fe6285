"""Attention over a cache in pages at the ends of fp32's range, against 64 bits."""
import numpy as np
import pytest

from test_gpu_paged import U, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("std", [1e5, 1e7, 1e9, 1e12, 1e20, 1e30])
@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads,kvh,hd,tok", [(4, 2, 128, 1), (4, 2, 64, 7), (8, 2, 128, 24),
                                              (8, 1, 64, 40), (4, 2, 256, 12)])
def test_large_scores(ctx, heads, kvh, hd, tok, kv, std):
    """Scores of any size: their largest takes all the weight, and its value is the row."""
    c = Case(heads + tok, heads, kvh, hd, kv, 16, [700, 33, 0], [tok, tok, max(1, tok // 2)], tok,
             rope=False, q_std=std)
    want, size = c.want()
    live = np.arange(tok)[None] < c.n_tok[:, None]
    one = np.abs(want) >= size * (1 - 1e-12)  # one key has the weight: sum p |v| = |sum p v|
    # a score's fp32 error, (hd + 6) U of its terms, is far below the gap to the next one
    sure = one.all(-1) & live[..., None]
    assert sure[live].mean() > 0.98
    for max_len in (700, 0):  # split over many workgroups, and over few
        got = c.run(ctx, max_len=max_len).astype(np.float64)
        assert np.all(np.isfinite(got[live]))
        # A weight w of one key that is not 1 but up to 2^0.25: w v from six of nine products of
        # parts cut off after 8 bits each, whose remainders are below 2^-7 and 2^-15 of a value's
        # power of two: the others are below 2 2^-7 2^-15 + 2^-30, 8 U (F16 pages: w in 22 bits, 4
        # U); then roundings of w's sum, its reciprocal, w v and their product: 12 U.  A subnormal
        # fp16 v has the exponent -14 in a product's alignment, whatever its leading zeros: each of
        # its two products with 2^15 w < 2^16 is cut at 2^-24 2^(15 - 14), and both at 2^-22 / 2^15
        low = 2.0 ** -37 if kv == "f16" else 0.0
        assert np.all(np.abs(got - want)[sure] <= 12 * U * size[sure] + low)


@pytest.mark.parametrize("tok", [1, 12, 40])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_small_values(ctx, hd, tok):
    """Values down to the end of fp32's normal range keep their digits."""
    c = Case(61, 4, 2, hd, "f32", 16, [90, 33], [tok, tok], tok, rope=False)
    c.v *= (10.0 ** np.linspace(-36.5, -29, hd)).astype(np.float32)
    want, size = c.want()
    live = np.arange(tok)[None] < c.n_tok[:, None]
    for max_len in (90, 0):
        a, b = c.run(ctx, max_len=max_len)[live], want[live]
        # as Case.check: scores of at most 60 off by (hd + 6) U of their terms; below 2^-126
        # fp32 itself steps by 2^-149, at most once a row summed
        per = 2 * ((hd + 6) * U * 60 + (90 + tok + 16) * U)
        assert np.all(np.abs(a - b) <= per * size[live] + 200 * 2.0 ** -149)
        rel = np.abs(a - b) / size[live]
        assert np.sqrt(np.mean(rel ** 2)) <= 2e-6


@pytest.mark.parametrize("tok", [1, 12, 40])
@pytest.mark.parametrize("low,high", [(-36, -30), (30, 36)])
def test_keys_at_the_ends(ctx, low, high, tok):
    """Keys of 1e-36 or 1e36 next to ordinary ones, under queries that even them out: no
    score loses a term's digits."""
    c = Case(67, 4, 2, 128, "f32", 16, [90, 33], [tok, tok], tok, rope=False)
    scale = np.ones(128, np.float32)
    scale[::2] = (10.0 ** np.linspace(low, high, 64)).astype(np.float32)
    c.k *= scale
    c.q /= scale
    want, size = c.want()
    live = np.arange(tok)[None] < c.n_tok[:, None]
    a, b = c.run(ctx)[live], want[live]
    # per score: (hd + 6) U sum|q_d k_d| / sqrt(hd), |q_d k_d| at most 6 sigma squares apart
    assert np.all(np.abs(a - b) <= 2 * (134 * U * 40 + 150 * U) * size[live])
    rel = np.abs(a - b) / size[live]
    assert np.sqrt(np.mean(rel ** 2)) <= 2e-6
