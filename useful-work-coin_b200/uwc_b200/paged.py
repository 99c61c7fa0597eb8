"""The paged 8-bit KV cache on B200: ragged batches, sliding windows, sinks.

A layer's cache is a dict like detmodel's (k, v, sk, sv), but a pool of pages that sequences take as
they grow: k, v (pages, Hkv, page_size, 128) int8 with one float32 scale for each (page, KV head). The
reference's own cache (runtime/detrt/qwen3.py:216-221) is contiguous, with one start position for the
whole batch; nothing of it changes here.

Every call takes a ragged batch by its device-side description, so a captured CUDA graph serves every
step of a generation: rows cu[s] .. cu[s + 1] - 1 of q, k and v are sequence s's new tokens, at
positions start[s] and on; table[s] lists its pages (position p lies in page table[s, p // page_size];
entries past its last position are never read). start[s] < 0 marks an idle slot. A page id, position or
row out of range is skipped on the device and raises _lib.DEV_RANGE in _lib.device_status().

Row tensors are bf16 or fp16 (n, heads, 128) with contiguous heads' rows; they may be views of a fused
q | k | v row. Inference only: nothing here has a gradient, like every integer path of the package.
"""
from __future__ import annotations

import math

import torch

from ._lib import UWCError

try:
    from . import _paged
except ImportError as e:
    raise UWCError(f"uwc_b200/_paged.so cannot be loaded ({e}): build it with useful-work-coin_b200/build.py") from e

HD = 128
PAGE_SIZES = (16, 32, 64, 128)
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_SCALE = 1.0 / math.sqrt(HD)


def new_cache(pages: int, Hkv: int, page_size: int = 64, device="cuda") -> dict:
    """An empty pool of one layer's pages. Tokens per page: 16, 32, 64 or 128."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt, device=device)
    return dict(k=z(pages, Hkv, page_size, HD), v=z(pages, Hkv, page_size, HD),
                sk=z(pages, Hkv, dt=torch.float32), sv=z(pages, Hkv, dt=torch.float32))


def append(k, v, cache: dict, table, start, cu, max_new: int, cos, sin, q=None, q_norm=None, k_norm=None,
           eps: float = 1e-6):
    """Rotate the new tokens' keys and append them and their values to their pages: k, v (n, Hkv, 128).
    cos / sin: detmodel.rope_table's float32 rows on the device. With q (n, H, 128) the rotated queries
    are returned (contiguous, same type). q_norm / k_norm: float32 weights of a per-head RMSNorm before
    the rotation (Qwen3). max_new: a bound on a sequence's new tokens.

    A page's scale is its largest magnitude / 127: it grows when a new token needs it, and the tokens
    already there, at positions before start[s], are brought to it. Appending a sequence's newest tokens
    again changes nothing. start[s] + new tokens is then the sequence's end: what a page held past it (drafts
    that were rejected, a longer sequence rolled back) is given up and no longer stands for its values, so an
    earlier chunk is not written again under tokens that are to stay."""
    return _paged.append(cache["k"], cache["v"], cache["sk"], cache["sv"], table, start, cu, max_new, k, v, cos, sin, q,
                         q_norm, k_norm, eps)


def gather(cache: dict, table, first, cu, n: int, max_rows: int, dtype=torch.bfloat16):
    """Cached tokens as values: rows cu[s] .. cu[s + 1] - 1 of the two (n, Hkv, 128) tensors returned
    are sequence s's keys and values at positions first[s] and on (at most max_rows of a sequence)."""
    return _paged.gather(cache["k"], cache["v"], cache["sk"], cache["sv"], table, first, cu, n, max_rows, _TYPES[dtype])


def attention(q, cache: dict, table, start, cu, max_new: int, max_len: int, scale: float | None = None,
              window: int | None = None, sinks: int = 0, out=None):
    """Attention of the new tokens' queries q (n, H, 128) over their sequences' pages, which already
    hold their keys and values (append first). The query at position p sees key j when j <= p and,
    with a window, j > p - window or j < sinks. scale: 1 / sqrt(128) by default. max_len: a bound on
    start[s] + new tokens. Returns (n, H, 128) in q's type; rows that see nothing are zero."""
    return _paged.attention(cache["k"], cache["v"], cache["sk"], cache["sv"], table, start, cu, max_new, q, max_len,
                            _SCALE if scale is None else scale, window, sinks, out)
