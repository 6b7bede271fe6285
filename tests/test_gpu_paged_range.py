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


