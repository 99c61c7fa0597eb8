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

from ._lib import check, lib

HD = 128
PAGE_SIZES = (16, 32, 64, 128)
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def new_cache(pages: int, Hkv: int, page_size: int = 64, device="cuda") -> dict:
    """An empty pool of one layer's pages. Tokens per page: 16, 32, 64 or 128."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt, device=device)
    return dict(k=z(pages, Hkv, page_size, HD), v=z(pages, Hkv, page_size, HD),
                sk=z(pages, Hkv, dt=torch.float32), sv=z(pages, Hkv, dt=torch.float32))


def _cache_args(cache: dict, table, start, cu):
    """The cache's and the batch's pointers and sizes, checked."""
    k, v, sk, sv = cache["k"], cache["v"], cache["sk"], cache["sv"]
    pages, Hkv, ps, hd = k.shape
    assert hd == HD and v.shape == k.shape and sk.shape == (pages, Hkv) and sv.shape == (pages, Hkv), (k.shape, sk.shape)
    assert k.dtype == torch.int8 and v.dtype == torch.int8 and sk.dtype == torch.float32 and sv.dtype == torch.float32
    assert k.is_cuda and k.is_contiguous() and v.is_contiguous() and sk.is_contiguous() and sv.is_contiguous()
    assert table.dtype == torch.int32 and start.dtype == torch.int32 and cu.dtype == torch.int32
    seqs, width = table.shape
    assert start.shape == (seqs,) and cu.shape == (seqs + 1,), (table.shape, start.shape, cu.shape)
    assert table.is_contiguous() and start.is_contiguous() and cu.is_contiguous()
    dev = k.device
    for t in (v, sk, sv, table, start, cu):
        assert t.device == dev, "the cache and the batch's description lie on one device"
    return (k.data_ptr(), sk.data_ptr(), v.data_ptr(), sv.data_ptr(), pages, ps, Hkv, table.data_ptr(),
            start.data_ptr(), cu.data_ptr(), seqs, width), dev


def _rows(t: torch.Tensor, n: int, heads: int, dtype, dev):
    """(pointer, token stride, head stride) of a row tensor (n, heads, 128)."""
    assert t.shape == (n, heads, HD) and t.dtype == dtype and t.device == dev, (t.shape, t.dtype, t.device)
    assert t.stride(2) == 1, "a head's 128 values are contiguous"
    return t.data_ptr(), t.stride(0), t.stride(1)


def _current(dev) -> int:
    assert dev.index == torch.cuda.current_device(), "the tensors' device is the current one"
    return torch.cuda.current_stream(dev).cuda_stream


def append(k, v, cache: dict, table, start, cu, max_new: int, cos, sin, q=None, q_norm=None, k_norm=None,
           eps: float = 1e-6):
    """Rotate the new tokens' keys and append them and their values to their pages: k, v (n, Hkv, 128).
    cos / sin: detmodel.rope_table's float32 rows on the device. With q (n, H, 128) the rotated queries
    are returned (contiguous, same type). q_norm / k_norm: float32 weights of a per-head RMSNorm before
    the rotation (Qwen3). max_new: a bound on a sequence's new tokens.

    A page's scale is its largest magnitude / 127: it grows when a new token needs it, and the tokens
    already there are brought to it. Appending the same tokens again changes nothing."""
    args, dev = _cache_args(cache, table, start, cu)
    n, Hkv, dt = k.shape[0], args[6], k.dtype
    assert dt in (torch.bfloat16, torch.float16), dt
    kr, vr = _rows(k, n, Hkv, dt, dev), _rows(v, n, Hkv, dt, dev)
    assert cos.dtype == torch.float32 and sin.dtype == torch.float32 and cos.shape == sin.shape and cos.shape[1] == HD
    assert cos.is_contiguous() and sin.is_contiguous() and cos.device == dev and sin.device == dev
    for w in (q_norm, k_norm):
        assert w is None or (w.shape == (HD,) and w.dtype == torch.float32 and w.is_contiguous() and w.device == dev)
    out, H, qr = None, 0, (None, 0, 0)
    if q is not None:
        H = q.shape[1]
        qr = _rows(q, n, H, dt, dev)
        out = torch.empty((n, H, HD), dtype=dt, device=dev)
    ptr = lambda t: None if t is None else t.data_ptr()
    check(lib().uwc_paged_append(*args, n, max_new, _TYPES[dt], *kr, *vr, *qr, ptr(out), H, cos.data_ptr(),
                                 sin.data_ptr(), cos.shape[0], ptr(q_norm), ptr(k_norm), eps, _current(dev)),
          "paged append")
    return out


def gather(cache: dict, table, first, cu, n: int, max_rows: int, dtype=torch.bfloat16):
    """Cached tokens as values: rows cu[s] .. cu[s + 1] - 1 of the two (n, Hkv, 128) tensors returned
    are sequence s's keys and values at positions first[s] and on (at most max_rows of a sequence)."""
    args, dev = _cache_args(cache, table, first, cu)
    k = torch.empty((n, args[6], HD), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    check(lib().uwc_paged_gather(*args, n, max_rows, _TYPES[dtype], k.data_ptr(), v.data_ptr(), _current(dev)),
          "paged gather")
    return k, v


_WS: dict = {}       # (device, stream) -> workspace, grown on demand
_RETIRED: list = []  # outgrown workspaces: a captured graph may still run on one


def _workspace(dev, stream: int, nbytes: int):
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=dev)     # the graph's own, zeroed by it
    ws = _WS.get((dev.index, stream))
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _RETIRED.append(ws)
            nbytes = max(nbytes, 2 * ws.numel())
        ws = _WS[(dev.index, stream)] = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
    return ws


def attention(q, cache: dict, table, start, cu, max_new: int, max_len: int, scale: float | None = None,
              window: int | None = None, sinks: int = 0, out=None):
    """Attention of the new tokens' queries q (n, H, 128) over their sequences' pages, which already
    hold their keys and values (append first). The query at position p sees key j when j <= p and,
    with a window, j > p - window or j < sinks. scale: 1 / sqrt(128) by default. max_len: a bound on
    start[s] + new tokens. Returns (n, H, 128) in q's type; rows that see nothing are zero."""
    args, dev = _cache_args(cache, table, start, cu)
    n, H, _ = q.shape
    dt = q.dtype
    assert dt in (torch.bfloat16, torch.float16), dt
    assert window is None or window >= 0, window
    assert 0 <= sinks, sinks
    qr = _rows(q, n, H, dt, dev)
    if out is None:
        out = torch.empty((n, H, HD), dtype=dt, device=dev)
    assert out.shape == (n, H, HD) and out.dtype == dt and out.is_contiguous() and out.device == dev
    w = -1 if window is None else min(int(window), 1 << 30)
    sinks = min(int(sinks), 1 << 30)
    stream = _current(dev)
    L = lib()
    nbytes = L.uwc_paged_attention_workspace_bytes(args[10], max_new, max_len, H, args[6], w, sinks)
    ws = _workspace(dev, stream, nbytes) if nbytes else None
    check(L.uwc_paged_attention(*args, n, max_new, max_len, _TYPES[dt], *qr, out.data_ptr(), H,
                                1.0 / math.sqrt(HD) if scale is None else scale, w, sinks,
                                None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), stream),
          "paged attention")
    return out
