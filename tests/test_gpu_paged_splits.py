"""The paged operators where the work is cut: units in dozens of parts, more sequences than a CTA keeps in shared
memory, shares that end inside an item's own cost, and quotients that lie exactly between two integers. The
tolerances are paged_fixture's; append is compared bit for bit."""
import numpy as np
import pytest
import torch

from paged_fixture import D, Batch, append_plain
from test_gpu_paged import BF, HF, check_attention, numpy_cache, status_clean  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,new,H,Hkv", [([20000], [1], 4, 1), ([20000, 7, 9001], [4, 1, 2], 8, 2), ([20000], [70], 1, 1),
                                            ([9000, 130], [300, 130], 4, 2)], ids=lambda v: str(v).replace(" ", ""))
def test_units_in_many_parts(dev, lens, new, H, Hkv):
    b = Batch(lens, new, 64, seed=len(lens))
    check_attention(dev, b, H, Hkv, BF, seed=1)
    check_attention(dev, b, H, Hkv, HF, seed=2, window=5000, sinks=70)


@pytest.mark.parametrize("most", [1, 40])
def test_more_sequences_than_are_kept(dev, most):
    """1100 sequences, some idle, some without a new token, most of them shorter than a tile."""
    r = np.random.default_rng(most)
    new = [int(x) for x in r.integers(0, most + 1, 1100)]
    lens = [None if i % 97 == 5 else n + int(r.integers(0 if n else 1, 60)) for i, n in enumerate(new)]
    lens[1090] = 700 + new[1090]
    check_attention(dev, Batch(lens, new, 16, seed=most), 2, 2 if most == 1 else 1, BF, seed=3)


@pytest.mark.parametrize("new,count", [(33, 40), (1, 200)])
def test_shares_that_end_in_an_items_cost(dev, new, count):
    """Items of one to three tiles, more of them than SMs: the line's cuts fall inside their own cost too."""
    lens = [new + (i * 37) % 300 for i in range(count)]
    check_attention(dev, Batch(lens, [new] * count, 32, seed=new), 16, 4, HF, seed=4)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new", [1, 64])
def test_append_of_ties(dev, dtype, new):
    """Page scales of exactly 2^-3 and values of (i + 1/2) 2^-3 and next to them: rounded to even as divisions are."""
    from uwc_b200 import paged
    ps, Hkv, n = 64, 2, 64
    i = torch.arange(new * Hkv * D, dtype=torch.float32).reshape(new, Hkv, D) * 37 % 254 - 127
    x = ((i + 0.5) * 0.125).to(dtype)
    if dtype == HF:                                        # 11 bits hold the neighbours of a half as well
        step = torch.tensor([0, 1, -1], dtype=torch.int16)[torch.arange(D) % 3]
        x = (x.view(torch.int16) + step).view(dtype)
    x[:, :, 0] = 127 * 0.125                               # the largest: the scale is 2^-3
    b = Batch([n], [new], ps)
    cache = paged.new_cache(b.pages, Hkv, ps, dev)
    cache["sk"].fill_(0.125)
    cache["sv"].fill_(0.125)
    cosd, sind = torch.ones(n, D, device=dev), torch.zeros(n, D, device=dev)   # keys stay as they are
    want = append_plain(x.float().numpy(), x.float().numpy(), numpy_cache(cache), b, cosd.cpu().numpy(), sind.cpu().numpy())
    x = x.to(dev)
    paged.append(x, x, cache, *b.device(dev), b.max_new, cosd, sind)
    for name in ("sk", "sv", "k", "v"):
        assert np.array_equal(cache[name].cpu().numpy(), want[name]), name
    assert float(cache["sv"][int(b.table[0, 0]), 0]) == 0.125
