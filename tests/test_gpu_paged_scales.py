"""Paged attention where pages' scales lie far apart. What a row loses is measured against that row alone: the
sum of p |v| over the keys that it sees, whatever lies in pages that its mask hides and however small its values."""
import math

import pytest
import torch

from paged_fixture import D, Batch, attention64, random_cache
from test_gpu_paged import BF, HF, fused_rows, status_clean  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

FORMS = [1, 4, 60]                          # few rows (G = 2: 2 and 8 rows), many rows


def check_rows(dev, b, cache, q, window=None, sinks=0, scale=None):
    """Within the output's rounding, 11 bits of each weight, and scores in float32 (paged_fixture.tolerance);
    weights below fp16's normal range are off by 2^-25 where the row's largest is 2^7 at least, which is
    2^-32 of the row's largest p 127 s_v for each key; factors through log2 and exp2 of numbers up to 128 are off by
    2^-16. Outputs below float32's normal range may be lost (2^-126, or the type's smallest step)."""
    from uwc_b200 import paged
    sc = 1 / math.sqrt(D) if scale is None else scale
    o, absv, smax = attention64(q, cache, b, sc, window, sinks)
    largest = cache_tops(cache, b, q, sc, window, sinks)
    got = paged.attention(q, cache, *b.device(dev), b.max_new, b.max_len, scale=scale, window=window, sinks=sinks)
    fi = torch.finfo(q.dtype)
    tol = (fi.eps / 2 * o.abs() + (2.0 ** -11 * 1.01 + 2.0 ** -16 + 2.0 ** -16 * smax[..., None]) * absv
           + 2.0 ** -32 * b.max_len * largest[..., None] + max(2.0 ** -126, fi.smallest_normal * fi.eps / 2))
    err = (got.double() - o).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).nan_to_num(math.inf).max()):.3g} tolerances"
    return got


def cache_tops(cache, b, q, scale, window, sinks):
    """Each row's largest p 127 s_v."""
    ones = {**cache, "v": torch.full_like(cache["v"], 127)}
    # p |v| of the value 127 everywhere, summed over the row: no less than its largest
    return attention64(q, ones, b, scale, window, sinks)[1].amax(-1)


def setup(dev, lens, new, ps, Hkv, dtype, seed, amp=1.0):
    b = Batch(lens, new, ps, seed=seed)
    cache = random_cache(b, Hkv, dev, seed, spread=0.0)
    q, _, _ = fused_rows(b.rows, 2 * Hkv, Hkv, dtype, dev, seed, amp)
    return b, cache, q
