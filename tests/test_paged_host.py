"""The paged cache's refusals, checked without a device: every bad argument is turned away before
anything is launched."""
import ctypes

import pytest


def base_append():
    f = ctypes.c_void_p(0x1000)   # never dereferenced
    return dict(kc=f, sk=f, vc=f, sv=f, pages=4, page_size=64, Hkv=2, table=f, start=f, cu=f, seqs=1, width=4, rows=3,
                max_new=3, dtype=0, k=f, k_tok=256, k_head=128, v=f, v_tok=256, v_head=128, q=f, q_tok=512, q_head=128,
                q_out=f, H=4, cos=f, sin=f, max_pos=64, q_norm=None, k_norm=None, eps=1e-6, stream=None)


def base_attention():
    f = ctypes.c_void_p(0x1000)
    return dict(kc=f, sk=f, vc=f, sv=f, pages=4, page_size=64, Hkv=2, table=f, start=f, cu=f, seqs=1, width=4, rows=3,
                max_new=3, max_len=64, dtype=0, q=f, q_tok=512, q_head=128, out=f, H=4, scale=0.1, window=-1, sinks=0,
                ws=f, ws_bytes=1 << 30, stream=None)


def base_gather():
    f = ctypes.c_void_p(0x1000)
    return dict(kc=f, sk=f, vc=f, sv=f, pages=4, page_size=64, Hkv=2, table=f, first=f, cu=f, seqs=1, width=4, rows=3,
                max_rows=3, dtype=0, k=f, v=f, stream=None)


ODD = ctypes.c_void_p(0x1008)
SHARED = [("kc", None, "ARG"), ("sk", None, "ARG"), ("vc", None, "ARG"), ("sv", None, "ARG"), ("table", None, "ARG"),
          ("cu", None, "ARG"), ("pages", 0, "SHAPE"), ("page_size", 48, "SHAPE"), ("page_size", 256, "SHAPE"),
          ("page_size", 0, "SHAPE"), ("Hkv", 0, "SHAPE"), ("seqs", -1, "SHAPE"), ("seqs", 65536, "SHAPE"),
          ("width", 0, "SHAPE"), ("width", 1 << 26, "SHAPE"), ("rows", -1, "SHAPE"), ("rows", (1 << 30) + 1, "SHAPE"),
          ("kc", ODD, "ALIGN"), ("vc", ODD, "ALIGN"), ("dtype", 7, "ARG"), ("dtype", -1, "ARG")]


@pytest.mark.parametrize("arg,value,code", SHARED + [
    ("start", None, "ARG"), ("k", None, "ARG"), ("v", None, "ARG"), ("cos", None, "ARG"), ("sin", None, "ARG"),
    ("q_out", None, "ARG"), ("dtype", 2, "ARG"), ("max_new", -1, "SHAPE"), ("max_pos", 0, "SHAPE"), ("H", 0, "SHAPE"),
    ("k", ODD, "ALIGN"), ("v", ODD, "ALIGN"), ("q", ODD, "ALIGN"), ("q_out", ODD, "ALIGN"), ("cos", ODD, "ALIGN"),
    ("k_tok", 130, "ALIGN"), ("v_head", 4, "ALIGN"), ("q_tok", -512, "ALIGN")])
def test_append_refuses(arg, value, code):
    from uwc_b200 import _lib
    a = base_append()
    assert arg in a
    a[arg] = value
    assert _lib.lib().uwc_paged_append(*a.values()) == getattr(_lib, f"ERR_{code}")


@pytest.mark.parametrize("arg,value,code", SHARED + [
    ("start", None, "ARG"), ("q", None, "ARG"), ("out", None, "ARG"), ("dtype", 2, "ARG"), ("H", 0, "SHAPE"),
    ("H", 3, "SHAPE"), ("max_len", -1, "SHAPE"), ("sinks", -1, "SHAPE"), ("max_new", -1, "SHAPE"), ("max_new", (1 << 29) + 1, "SHAPE"),
    ("q", ODD, "ALIGN"),
    ("out", ODD, "ALIGN"), ("q_tok", 12, "ALIGN"), ("q_head", 4, "ALIGN")])
def test_attention_refuses(arg, value, code):
    from uwc_b200 import _lib
    a = base_attention()
    assert arg in a
    a[arg] = value
    assert _lib.lib().uwc_paged_attention(*a.values()) == getattr(_lib, f"ERR_{code}")


@pytest.mark.parametrize("arg,value,code", SHARED + [
    ("first", None, "ARG"), ("k", None, "ARG"), ("v", None, "ARG"), ("max_rows", -1, "SHAPE"), ("k", ODD, "ALIGN"),
    ("v", ODD, "ALIGN")])
def test_gather_refuses(arg, value, code):
    from uwc_b200 import _lib
    a = base_gather()
    assert arg in a
    a[arg] = value
    assert _lib.lib().uwc_paged_gather(*a.values()) == getattr(_lib, f"ERR_{code}")


def test_python_refusals():
    """The module's own checks come before the library's: host tensors are not a cache."""
    import torch
    from uwc_b200 import paged
    with pytest.raises(ValueError):
        paged.new_cache(4, 2, 48, "cpu")
    cache = paged.new_cache(4, 2, 64, "cpu")
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        paged.attention(q, cache, z(1, 4), z(1), z(2), 1, 64)
    with pytest.raises(AssertionError):
        paged.gather(cache, z(1, 4), z(1), z(2), 1, 1)
    with pytest.raises(AssertionError):
        paged.append(q[:, :2], q[:, :2], cache, z(1, 4), z(1), z(2), 1, None, None)


@pytest.mark.parametrize("none", [dict(rows=0), dict(seqs=0)], ids=str)
def test_nothing_to_do_needs_no_address(none):
    """Row tensors of no row and descriptions of no sequence have none: the call passes its checks and gets as far as
    the device's."""
    from uwc_b200 import _lib
    names = {"rows": ("k", "v", "q", "q_out", "out"), "seqs": ("table", "start", "first", "cu")}[next(iter(none))]
    for f, base in (("append", base_append), ("attention", base_attention), ("gather", base_gather)):
        a = base()
        a.update(none, **{n: None for n in names if n in a})
        rc = getattr(_lib.lib(), f"uwc_paged_{f}")(*a.values())
        assert rc in (_lib.OK, _lib.ERR_CUDA, _lib.ERR_DEVICE), (f, rc)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_attention_refuses_a_scale_that_is_not_finite(scale):
    from uwc_b200 import _lib
    assert _lib.lib().uwc_paged_attention(*{**base_attention(), "scale": scale}.values()) == _lib.ERR_ARG
