"""The paged operators at the edges of their arguments: integers far outside an int, tensors without a row, batches
without a sequence, queries and keys at the ends of bf16's range, integers of -128 in a caller's pages."""
import math

import numpy as np
import pytest
import torch

from paged_fixture import D, Batch, append_plain, random_cache
from test_gpu_paged import BF, HF, fused_rows, numpy_cache, status_clean, tables  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [-1, -2 ** 31, -2 ** 32, 5 - 2 ** 32, -2 ** 63])
def test_negative_windows_and_sinks_are_refused(dev, value):
    from uwc_b200 import paged
    b = Batch([40], [1], 16)
    cache = random_cache(b, 1, dev)
    q, _, _ = fused_rows(1, 2, 1, BF, dev, 0)
    with pytest.raises(AssertionError):
        paged.attention(q, cache, *b.device(dev), 1, 40, window=value)
    with pytest.raises(AssertionError):
        paged.attention(q, cache, *b.device(dev), 1, 40, window=8, sinks=value)


@pytest.mark.parametrize("value", [2 ** 31, 2 ** 40, 2 ** 63 - 1])
def test_windows_past_every_position_are_none(dev, value):
    from uwc_b200 import paged
    b = Batch([40], [1], 16)
    cache = random_cache(b, 1, dev)
    q, _, _ = fused_rows(1, 2, 1, BF, dev, 0)
    want = paged.attention(q, cache, *b.device(dev), 1, 40)
    assert torch.equal(paged.attention(q, cache, *b.device(dev), 1, 40, window=value), want)
    assert torch.equal(paged.attention(q, cache, *b.device(dev), 1, 40, window=3, sinks=value), want)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_no_rows_and_no_sequences(dev, dtype):
    """Nothing to do is done: tensors of no row, which have no address, and a batch of no sequence."""
    from uwc_b200 import paged
    b = Batch([40, 9], [0, 0], 16)
    cache = random_cache(b, 2, dev)
    before = {n: t.clone() for n, t in cache.items()}
    table, start, cu = b.device(dev)
    _, _, cosd, sind = tables(64, dev)
    q, k, v = fused_rows(0, 4, 2, dtype, dev, 0)
    none = torch.empty(0, b.width, dtype=torch.int32, device=dev), torch.empty(0, dtype=torch.int32, device=dev), cu[:1]
    for t, s, c in ((table, start, cu), none):
        assert paged.append(k, v, cache, t, s, c, 0, cosd, sind) is None
        assert paged.append(k, v, cache, t, s, c, 3, cosd, sind, q=q).shape == (0, 4, D)
        assert paged.attention(q, cache, t, s, c, 0, 40).shape == (0, 4, D)
        x, y = paged.gather(cache, t, s, c, 0, 0, dtype=dtype)
        assert x.shape == y.shape == (0, 2, D) and x.dtype == dtype
    # rows that no sequence covers stay as they are
    q, k, v = fused_rows(3, 4, 2, dtype, dev, 0)
    out = torch.full((3, 4, D), 7.0, dtype=dtype, device=dev)
    paged.attention(q, cache, *none, 1, 40, out=out)
    paged.append(k, v, cache, *none, 1, cosd, sind)
    assert (out == 7.0).all() and all(torch.equal(before[n], cache[n]) for n in cache)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_not_finite_is_refused(dev, scale):
    from uwc_b200 import paged
    for new in (1, 40):
        b = Batch([40], [new], 16)
        q, _, _ = fused_rows(new, 2, 1, BF, dev, 0)
        with pytest.raises(AssertionError):
            paged.attention(q, random_cache(b, 1, dev), *b.device(dev), new, 40, scale=scale)


@pytest.mark.parametrize("e", [100, 116, 125, 127])
def test_queries_up_to_the_largest(dev, e):
    """Single tokens whose largest query value is near 2^e, on keys as much smaller: the scores are ordinary."""
    from test_gpu_paged_scales import check_rows
    b = Batch([300, 17], [1, 1], 64, seed=e)
    cache = random_cache(b, 2, dev, e, spread=0.3)
    q, _, _ = fused_rows(2, 4, 2, BF, dev, e)
    up = math.ldexp(1.0, e - 2)                            # the rows' largest are below 4
    assert float(q.abs().max()) < 4
    cache["sk"] *= 2.0 ** -60
    plain = {**cache, "sk": cache["sk"] * 2.0 ** 60}
    check_rows(dev, b, plain, q)
    check_rows(dev, b, cache, (q.double() * up).to(BF), scale=math.ldexp(1 / math.sqrt(D), 62 - e))


@pytest.mark.parametrize("new", [1, 4, 60])
def test_pages_of_zero_keys_under_large_queries(dev, new):
    """A page whose key scale is 0 (or almost) adds nothing to a score, however large the query."""
    from test_gpu_paged_scales import check_rows
    for small in (0.0, 1e-40, 3e-39):
        b = Batch([200], [new], 16, seed=new)
        cache = random_cache(b, 1, dev, new, spread=0.0)
        q, _, _ = fused_rows(new, 2, 1, BF, dev, new)
        cache["sk"] *= 1e-34
        for at in (1, 5, 9):
            cache["sk"][b.table[0][at].item()] = small
        check_rows(dev, b, cache, (q.double() * 1e34).to(BF))


@pytest.mark.parametrize("new", [1, 20])
def test_held_integers_of_minus_128(dev, new):
    """An old token's integer is rounded in its new scale and not clamped, on either side of the quick quotient."""
    from uwc_b200 import paged
    ps, n = 64, 60
    for s0 in (127.5 / 128, 0.7, 0.9999):                  # -128 s0 / s: a tie, and two that are none
        b = Batch([n], [new], ps)
        cache = paged.new_cache(b.pages, 2, ps, dev)
        for name in ("k", "v"):
            cache[name][:] = (torch.arange(cache[name].numel(), device=dev) % 256 - 128).to(torch.int8).view(cache[name].shape)
        cache["sk"].fill_(s0)
        cache["sv"].fill_(s0)
        x = torch.zeros(new, 2, D, dtype=BF, device=dev)
        x[0, :, 0] = 127.0                                 # the new scale is 1
        cosd, sind = torch.ones(n, D, device=dev), torch.zeros(n, D, device=dev)
        f = x.float().cpu().numpy()
        want = append_plain(f, f, numpy_cache(cache), b, cosd.cpu().numpy(), sind.cpu().numpy())
        paged.append(x, x, cache, *b.device(dev), b.max_new, cosd, sind)
        for name in ("sk", "sv", "k", "v"):
            assert np.array_equal(cache[name].cpu().numpy(), want[name]), (s0, name)
        assert (cache["v"][int(b.table[0, 0]), :, :n - new] == -128).any() == (s0 > 0.99)


@pytest.mark.parametrize("most", [1, 8, 60])
@pytest.mark.parametrize("cu", [(5, -2 ** 31), (1, 2 - 2 ** 31), (2 ** 31 - 1, -2 ** 31), (2 ** 31 - 1, 2 ** 31 - 1 - 60),
                                (-2 ** 31, 2 ** 31 - 1), (-2 ** 31, -2 ** 31)], ids=str)
def test_row_offsets_at_the_ends_of_int(dev, cu, most):
    """Row offsets that are no rows: those of the tensors that they name (rows 0 and on, for a lower end below 0) may
    be written, none else, and the status says so."""
    from uwc_b200 import _lib, paged
    b = Batch([100], [1], 16)
    cache = random_cache(b, 2, dev)
    before = {n: t.clone() for n, t in cache.items()}
    table, _, _ = b.device(dev)
    start = torch.tensor([10], dtype=torch.int32, device=dev)
    c = torch.tensor(cu, dtype=torch.int32, device=dev)
    _, _, cosd, sind = tables(128, dev)
    q, k, v = fused_rows(7, 4, 2, BF, dev, 0)
    out = torch.full((7, 4, D), 7.0, dtype=BF, device=dev)
    named = cu[0] < 0 and cu[1] > 0
    paged.attention(q, cache, table, start, c, most, 100, out=out)
    assert _lib.device_status(clear=True) == _lib.DEV_RANGE
    assert (out[min(most, 7) if named else 0:] == 7.0).all()
    paged.append(k, v, cache, table, start, c, most, cosd, sind, q=q)
    assert _lib.device_status(clear=True) == _lib.DEV_RANGE
    if not named:
        assert all(torch.equal(before[n], cache[n]) for n in cache)
    paged.gather(cache, table, start, c, 7, most)
    assert _lib.device_status(clear=True) == _lib.DEV_RANGE


@pytest.mark.parametrize("max_new", [70, 2 ** 30, 2 ** 31 - 126, 2 ** 31 - 1])
def test_append_with_any_bound_on_new_tokens(dev, max_new):
    """The bound may be as loose as an int is wide (the C entry's; uwc_b200.paged takes it up to 2^30)."""
    from uwc_b200 import _lib, paged
    for ps in (16, 128):
        b = Batch([100, 3], [70, 2], ps)
        cache = random_cache(b, 2, dev)
        want = {n: t.clone() for n, t in cache.items()}
        table, start, cu = b.device(dev)
        _, _, cosd, sind = tables(128, dev)
        q, k, v = (t.contiguous() for t in fused_rows(72, 4, 2, BF, dev, 0))
        rot = paged.append(k, v, want, table, start, cu, 70, cosd, sind, q=q)
        got = torch.empty_like(q)
        a = lambda t: t.data_ptr()
        args = [a(cache["k"]), a(cache["sk"]), a(cache["v"]), a(cache["sv"]), b.pages, ps, 2, a(table), a(start), a(cu), 2,
                b.width, 72, max_new, 0, a(k), 2 * D, D, a(v), 2 * D, D, a(q), 4 * D, D, a(got), 4, a(cosd), a(sind), 128,
                None, None, 1e-6, torch.cuda.current_stream().cuda_stream]
        assert _lib.lib().uwc_paged_append(*args) == _lib.OK
        assert torch.equal(got, rot) and all(torch.equal(cache[n], want[n]) for n in cache)
