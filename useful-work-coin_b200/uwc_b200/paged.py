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
_SCALE = 1.0 / math.sqrt(HD)


def new_cache(pages: int, Hkv: int, page_size: int = 64, device="cuda") -> dict:
    """An empty pool of one layer's pages. Tokens per page: 16, 32, 64 or 128."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: one of {PAGE_SIZES}")
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt, device=device)
    return dict(k=z(pages, Hkv, page_size, HD), v=z(pages, Hkv, page_size, HD),
                sk=z(pages, Hkv, dt=torch.float32), sv=z(pages, Hkv, dt=torch.float32))


_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice
I8, I32, F32, BF16, F16 = torch.int8, torch.int32, torch.float32, torch.bfloat16, torch.float16


def _cache_args(cache: dict, table, start, cu):
    """The cache's and the batch's pointers and sizes, checked, and their device."""
    k, v, sk, sv = cache["k"], cache["v"], cache["sk"], cache["sv"]
    shape = pages, Hkv, ps, hd = k.shape
    scales = (pages, Hkv)
    assert hd == HD and v.shape == shape and sk.shape == scales and sv.shape == scales, (shape, sk.shape, sv.shape)
    assert k.dtype is I8 and v.dtype is I8 and sk.dtype is F32 and sv.dtype is F32
    assert table.dtype is I32 and start.dtype is I32 and cu.dtype is I32
    seqs, width = table.shape
    assert start.shape == (seqs,) and cu.shape == (seqs + 1,), (table.shape, start.shape, cu.shape)
    assert (k.is_contiguous() and v.is_contiguous() and sk.is_contiguous() and sv.is_contiguous()
            and table.is_contiguous() and start.is_contiguous() and cu.is_contiguous())
    dev = k.get_device()
    assert (dev >= 0 and v.get_device() == dev and sk.get_device() == dev and sv.get_device() == dev
            and table.get_device() == dev and start.get_device() == dev and cu.get_device() == dev), \
        "the cache and the batch's description lie on one CUDA device"
    assert dev == _device(), "the tensors' device is the current one"
    return (k.data_ptr(), sk.data_ptr(), v.data_ptr(), sv.data_ptr(), pages, ps, Hkv, table.data_ptr(),
            start.data_ptr(), cu.data_ptr(), seqs, width), dev


def _rows(t: torch.Tensor, n: int, heads: int, dtype, dev: int):
    """(pointer, token stride, head stride) of a row tensor (n, heads, 128)."""
    assert t.shape == (n, heads, HD) and t.dtype is dtype and t.get_device() == dev, (t.shape, t.dtype, t.device)
    tok, head, one = t.stride()
    assert one == 1, "a head's 128 values are contiguous"
    return t.data_ptr(), tok, head


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
    assert dt is BF16 or dt is F16, dt
    kr, vr = _rows(k, n, Hkv, dt, dev), _rows(v, n, Hkv, dt, dev)
    max_pos, hd = cos.shape
    assert hd == HD and sin.shape == cos.shape and cos.dtype is F32 and sin.dtype is F32, (cos.shape, sin.shape)
    assert cos.is_contiguous() and sin.is_contiguous() and cos.get_device() == dev and sin.get_device() == dev
    qn = kn = None
    if q_norm is not None or k_norm is not None:
        for w in (q_norm, k_norm):
            assert w is None or (w.shape == (HD,) and w.dtype is F32 and w.is_contiguous() and w.get_device() == dev)
        qn, kn = (None if w is None else w.data_ptr() for w in (q_norm, k_norm))
    out, po, H, qr = None, None, 0, (None, 0, 0)
    if q is not None:
        H = q.shape[1]
        qr = _rows(q, n, H, dt, dev)
        out = torch.empty((n, H, HD), dtype=dt, device=q.device)
        po = out.data_ptr()
    check(lib().uwc_paged_append(*args, n, max_new, 0 if dt is BF16 else 1, *kr, *vr, *qr, po, H, cos.data_ptr(),
                                 sin.data_ptr(), max_pos, qn, kn, eps, _raw_stream(dev)), "paged append")
    return out


def gather(cache: dict, table, first, cu, n: int, max_rows: int, dtype=torch.bfloat16):
    """Cached tokens as values: rows cu[s] .. cu[s + 1] - 1 of the two (n, Hkv, 128) tensors returned
    are sequence s's keys and values at positions first[s] and on (at most max_rows of a sequence)."""
    args, dev = _cache_args(cache, table, first, cu)
    k = torch.empty((n, args[6], HD), dtype=dtype, device=table.device)
    v = torch.empty_like(k)
    check(lib().uwc_paged_gather(*args, n, max_rows, _TYPES[dtype], k.data_ptr(), v.data_ptr(), _raw_stream(dev)),
          "paged gather")
    return k, v


_WS: dict = {}       # (device, stream) -> its calls' workspace
_COUNTERS = 4096     # bytes at a workspace's start that are zero before a call, and after it


def _workspace(device, dev: int, stream: int, shape):
    """The stream's workspace, as large as any call needs (40 MB), its counters zeroed once: a call leaves
    them so. A captured call gets one of its own size, whose counters the graph zeroes."""
    if not torch.cuda.is_current_stream_capturing():
        ws = _WS.get((dev, stream))
        if ws is not None:
            return ws
        big = 1 << 30
        need = lib().uwc_paged_attention_workspace_bytes
        nbytes = max(need(1, rows, big, 1, 1, -1, 0) for rows in (8, 16, big))
    else:
        nbytes = lib().uwc_paged_attention_workspace_bytes(*shape)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws[:_COUNTERS].zero_()
    if not torch.cuda.is_current_stream_capturing():
        _WS[(dev, stream)] = ws
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
    assert dt is BF16 or dt is F16, dt
    assert window is None or window >= 0, window
    assert sinks >= 0, sinks
    qr = _rows(q, n, H, dt, dev)
    if out is None:
        out = torch.empty((n, H, HD), dtype=dt, device=q.device)
    else:
        assert out.shape == (n, H, HD) and out.dtype is dt and out.is_contiguous() and out.get_device() == dev
    stream = _raw_stream(dev)
    w, sinks = -1 if window is None else min(window, 1 << 30), min(sinks, 1 << 30)
    ws = _workspace(q.device, dev, stream, (args[10], max_new, max_len, H, args[6], w, sinks))
    check(lib().uwc_paged_attention(*args, n, max_new, max_len, 0 if dt is BF16 else 1, *qr, out.data_ptr(), H,
                                    _SCALE if scale is None else scale, w, sinks, ws.data_ptr(), ws.numel(), stream),
          "paged attention")
    return out
