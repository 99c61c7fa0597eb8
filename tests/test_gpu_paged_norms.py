"""paged.append with Qwen3's head norms, bit for bit: the oracle's det_rmsnorm before the rotation, in the few-token
kernel and the page kernel, for every page size, both types, and norms of queries, keys or both."""
import numpy as np
import pytest
import torch

import detq
from paged_fixture import D, Batch, append_plain, random_cache, turn
from test_gpu_paged import BF, HF, fused_rows, numpy_cache, status_clean, tables  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

# new tokens of three sequences and an idle slot: up to 8 run the few-token kernel
NEW = {1: [1, 1, 0, 1], 5: [5, 2, 4, 1], 8: [8, 3, 8, 2], 9: [9, 8, 1, 3], 70: [70, 2, 33, 5]}


@pytest.mark.parametrize("which", ["qk", "q", "k"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("most", NEW)
def test_normed_appends_match_plain_bits(dev, most, ps, dtype, which):
    from uwc_b200 import paged
    new = NEW[most]
    b = Batch([new[0] + 13, new[1], new[2] + 127, None], new, ps, seed=most)
    H, Hkv, eps = 6, 3, 1e-6
    cos, sin, cosd, sind = tables(256, dev)
    q, k, v = fused_rows(b.rows, H, Hkv, dtype, dev, most + ps, amp=3.0)
    k[0, 0] = 0                                            # a head of zeros: eps alone under the root
    g = torch.Generator(device=dev).manual_seed(7)
    qw, kw = (1 + 0.1 * torch.randn(D, device=dev, generator=g) for _ in range(2))
    norm = lambda x, w: detq.det_rmsnorm(x.float().cpu().numpy().reshape(-1, D), w.cpu().numpy(), eps).reshape(x.shape)
    kn = norm(k, kw) if "k" in which else k.float().cpu().numpy()
    qn = norm(q, qw) if "q" in which else q.float().cpu().numpy()
    cache = random_cache(b, Hkv, dev, most)
    want = append_plain(kn, v.float().cpu().numpy(), numpy_cache(cache), b, cos, sin)
    rot = paged.append(k, v, cache, *b.device(dev), b.max_new, cosd, sind, q=q, q_norm=qw if "q" in which else None,
                       k_norm=kw if "k" in which else None, eps=eps)
    for name in ("sk", "sv", "k", "v"):
        assert np.array_equal(cache[name].cpu().numpy(), want[name]), name
    for s, (n, m) in enumerate(zip(b.lens, new)):
        r0 = int(b.cu[s])
        if n is None:
            assert not rot[r0:r0 + m].any()
        elif m:
            p = np.arange(n - m, n)
            w = torch.from_numpy(turn(qn[r0:r0 + m], cos[p][:, None], sin[p][:, None])).to(dtype)
            assert torch.equal(rot[r0:r0 + m].cpu(), w), s
