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


@pytest.mark.parametrize("new", FORMS)
@pytest.mark.parametrize("small", [0.0, 1e-39, 1e-38, 1e-36, 1e-33, 1e-31, 1e-20])
def test_value_scales_of_almost_nothing(dev, small, new):
    """A head whose values are (almost) nothing, in all pages, in the first ones or in the last ones."""
    for where in (slice(0, None), slice(0, 4), slice(4, None), slice(6, 7)):
        b, cache, q = setup(dev, [140, 137], [new, new], 16, 2, BF, 3)
        for s in range(2):
            pages = b.table[s][:9].tolist()[where]
            cache["sv"][pages, s] = small
        check_rows(dev, b, cache, q)
        check_rows(dev, b, cache, q, window=50, sinks=3)


@pytest.mark.parametrize("small", [1e-4, 1e-6, 1e-9, 1e-12])
def test_rows_do_not_lose_bits_to_pages_that_they_do_not_see(dev, small):
    """A prompt whose first page's values are far smaller than the next ones': its first rows see no others."""
    b, cache, q = setup(dev, [100, 300], [100, 250], 16, 2, BF, 5)
    for s in range(2):
        cache["sv"][b.table[s][0].item()] *= small
        cache["sv"][b.table[s][3].item()] *= small
    check_rows(dev, b, cache, q)
    check_rows(dev, b, cache, q, window=16)


def test_chunks_of_a_prompt_give_its_rows(dev):
    """The first rows alone and as part of the prompt: the same within the rounding of their own values."""
    from uwc_b200 import paged
    b, cache, q = setup(dev, [120], [120], 16, 1, BF, 6)
    cache["sv"][b.table[0][0].item()] *= 1e-9
    all_rows = check_rows(dev, b, cache, q)
    table, start, _ = b.device(dev)
    head = paged.attention(q[:16], cache, table, start, torch.tensor([0, 16], dtype=torch.int32, device=dev), 16, 16)
    o, absv, _ = attention64(q, cache, b, 1 / math.sqrt(D), None, 0)
    off = (head.double() - all_rows[:16].double()).abs()
    assert bool((off <= 2.0 ** -8 * o[:16].abs() + 2.0 ** -9 * absv[:16]).all())


@pytest.mark.parametrize("new", FORMS)
@pytest.mark.parametrize("decades", [6, 12, 20])
def test_unlikely_keys_with_large_values(dev, decades, new):
    """Scores of up to some 60 (in log2) and value scales over many decades: what decides a row's output may be keys
    of next to no probability."""
    for seed in range(4):
        b, cache, q = setup(dev, [333, 90], [new, new], 16, 2, BF, seed, amp=2.0)
        g = torch.Generator(device=dev).manual_seed(seed)
        cache["sv"] = 10.0 ** (decades * (torch.rand(cache["sv"].shape, device=dev, generator=g) - 0.5))
        check_rows(dev, b, cache, q)


@pytest.mark.parametrize("new", FORMS)
@pytest.mark.parametrize("apart", [10, 20, 28, 40])
def test_one_page_of_unlikely_keys_decides(dev, apart, new):
    """Keys of 2^-apart of the others' probability (jittered, no powers of two) whose values are 2^(apart + 5) times
    as large: both kinds reach the output."""
    b, cache, q = setup(dev, [192], [new], 16, 1, BF, 8)
    q.fill_(1.0)
    unit = math.log(2) / 128 * 0.97
    cache["sk"].fill_(1.0)
    cache["k"].zero_()
    page = b.table[0][6].item()                            # 64 keys on from page 2
    cache["k"][page] = -(apart - 2 + torch.arange(16, device=dev, dtype=torch.int8) % 5)[None, :, None]
    cache["sv"].fill_(0.01)
    cache["sv"][page] *= 2.0 ** (apart + 5)
    check_rows(dev, b, cache, q, scale=unit)
