"""Paged attention whose waits run out, with no fault: the hook makes every second CTA fetch no pages. The call
returns, the status says so, the workspace's counters are zero as after any call, and the next call is right."""
import math
import time

import pytest
import torch

from paged_fixture import Batch, random_cache
from test_gpu_paged import BF, HF, fused_rows

pytestmark = pytest.mark.gpu


@pytest.fixture
def withhold(dev):
    from uwc_b200 import _lib
    L = _lib.lib()
    _lib.device_status(clear=True)

    def hook(on):
        assert L.uwc_test_hook(_lib.HOOK_WITHHOLD, int(on)) == 0
    yield hook
    hook(False)
    assert _lib.device_status(clear=True) == 0


# one long unit in many parts, units of every length, many short items (whole ones among them)
SHAPES = [([20000], [1], 4, 1), ([9000, 20, 3000], [3, 1, 4], 8, 2), ([9000, 130], [300, 130], 4, 2), ([700] * 40, [40] * 40, 8, 2)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,new,H,Hkv", SHAPES, ids=["token", "drafts", "chunks", "prompts"])
def test_counters_are_zero_after_a_timeout(dev, withhold, lens, new, H, Hkv, dtype):
    from uwc_b200 import _lib
    L, b = _lib.lib(), Batch(lens, new, 64, seed=1)
    cache = random_cache(b, Hkv, dev)
    q = fused_rows(b.rows, H, Hkv, dtype, dev, 0)[0].contiguous()
    table, start, cu = b.device(dev)
    n = L.uwc_paged_attention_workspace_bytes(len(lens), b.max_new, b.max_len, H, Hkv, -1, 0)
    ws = torch.zeros(n, dtype=torch.uint8, device=dev)
    p = lambda t: t.data_ptr()

    def call():
        out = torch.empty_like(q)
        rc = L.uwc_paged_attention(p(cache["k"]), p(cache["sk"]), p(cache["v"]), p(cache["sv"]), b.pages, 64, Hkv, p(table), p(start),
                                   p(cu), len(lens), b.width, b.rows, b.max_new, b.max_len, 0 if dtype == BF else 1, p(q),
                                   H * 128, 128, p(out), H, 1 / math.sqrt(128), -1, 0, p(ws), n,
                                   torch.cuda.current_stream().cuda_stream)
        assert rc == _lib.OK
        return out
    want = call()
    assert _lib.device_status(clear=True) == 0 and not ws[:4096].any()
    withhold(True)
    call()
    assert _lib.device_status(clear=True) == _lib.DEV_TIMEOUT
    withhold(False)
    assert not ws[:4096].any()
    assert torch.equal(call(), want) and not ws[:4096].any()


@pytest.mark.parametrize("new", [1, 60])
def test_the_kept_workspace_survives_a_timeout(dev, withhold, new):
    """paged.attention's own workspace, which is kept for the stream."""
    from uwc_b200 import _lib, paged
    b = Batch([15000, 200], [new, new], 64)
    cache = random_cache(b, 2, dev)
    q = fused_rows(b.rows, 8, 2, BF, dev, 0)[0]
    args = (q, cache, *b.device(dev), b.max_new, b.max_len)
    want = paged.attention(*args)
    withhold(True)
    paged.attention(*args)
    assert _lib.device_status(clear=True) == _lib.DEV_TIMEOUT
    withhold(False)
    for _ in range(2):
        assert torch.equal(paged.attention(*args), want)


@pytest.mark.parametrize("new", [1, 60])
def test_a_wait_takes_about_a_second(dev, withhold, new):
    from uwc_b200 import _lib, paged
    b = Batch([3000], [new], 64)
    cache = random_cache(b, 2, dev)
    q = fused_rows(b.rows, 8, 2, BF, dev, 0)[0]
    args = (q, cache, *b.device(dev), b.max_new, b.max_len)
    paged.attention(*args)
    assert _lib.device_status(clear=True) == 0
    withhold(True)
    t = time.perf_counter()
    paged.attention(*args)
    assert _lib.device_status(clear=True) == _lib.DEV_TIMEOUT
    assert 0.02 < time.perf_counter() - t < 8              # one wait, of a second or so, and the way out
