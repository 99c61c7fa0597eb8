"""The paged 8-bit KV cache (uwc_b200.paged) on a B200: append bit for bit against numpy float32 and
within half a step of the 64-bit values, attention against 64 bits over the lengths, page sizes, head
layouts and masks where it can go wrong, ragged and idle sequences, strides, streams, graphs, offsets
past 32 bits, and metadata out of range."""
import math

import numpy as np
import pytest
import torch

from paged_fixture import D, Batch, append_plain, attention64, random_cache, tolerance, turn

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def status_clean(dev):
    from uwc_b200 import _lib
    _lib.device_status(clear=True)
    yield
    assert _lib.device_status(clear=True) == 0, "a paged kernel reported metadata out of range"


def tables(n, dev, theta=1e6):
    from uwc_b200 import detmodel
    cos, sin, _ = detmodel.rope_table(theta, D, n)
    return cos, sin, torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev)


def fused_rows(n, H, Hkv, dtype, dev, seed, amp=1.0):
    """q, k, v as views of one fused row tensor, as a qkv projection leaves them."""
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(n, (H + 2 * Hkv) * D, device=dev, generator=g) * amp).to(dtype)
    cut = lambda a, h: x[:, a * D:(a + h) * D].view(n, h, D)
    return cut(0, H), cut(H, Hkv), cut(H + Hkv, Hkv)


def numpy_cache(c):
    return {k: t.cpu().numpy().copy() for k, t in c.items()}


# ------------------------------------------------------------------ append
APPENDS = [
    # (lens after, new, page size): one token into a started page, at a page's first position, a page exactly
    # filled, from position 0, several pages with a ragged end, idle slots and sequences with no new token
    ([1], [1], 64), ([64], [1], 64), ([65], [1], 64), ([2048], [1], 128), ([37], [37], 16), ([64], [64], 64),
    ([200, 5, 129, 64], [150, 5, 1, 33], 64), ([33, None, 17, 40], [2, 3, 0, 40], 32),
    ([300, 1, 256], [130, 1, 256], 128), ([100, 47, 16, 31], [99, 16, 16, 1], 16),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_matches_plain_bits(dev, case, dtype):
    from uwc_b200 import paged
    lens, new, ps = APPENDS[case]
    H, Hkv = ((16, 8), (3, 1), (28, 4))[case % 3]
    b = Batch(lens, new, ps, seed=case)
    cache = random_cache(b, Hkv, dev, seed=case)
    cos, sin, cosd, sind = tables(max(b.max_len, 1), dev)
    q, k, v = fused_rows(b.rows, H, Hkv, dtype, dev, case)
    want = append_plain(k.float().cpu().numpy(), v.float().cpu().numpy(), numpy_cache(cache), b, cos, sin)
    table, start, cu = b.device(dev)
    rot = paged.append(k, v, cache, table, start, cu, b.max_new, cosd, sind, q=q)
    for name in ("sk", "sv", "k", "v"):
        assert np.array_equal(cache[name].cpu().numpy(), want[name]), name
    qn = q.float().cpu().numpy()
    for s, (n, m) in enumerate(zip(lens, new)):
        r0 = int(b.cu[s])
        if n is None:
            assert not rot[r0:r0 + m].any()
        elif m:
            p = np.arange(n - m, n)
            w = torch.from_numpy(turn(qn[r0:r0 + m], cos[p][:, None], sin[p][:, None])).to(dtype)
            assert torch.equal(rot[r0:r0 + m].cpu(), w), s
    # the same tokens once more: nothing changes
    before = numpy_cache(cache)
    paged.append(k, v, cache, table, start, cu, b.max_new, cosd, sind)
    assert all(np.array_equal(before[n], cache[n].cpu().numpy()) for n in before)


def test_append_values_are_within_half_a_step(dev):
    """Token by token over a page: every stored value stays within the steps that its requantizations
    allow of the value that was appended (half a step of each scale that it went through)."""
    from uwc_b200 import paged
    ps, Hkv, n = 16, 2, 16
    b = Batch([n], [n], ps)
    cos, sin, cosd, sind = tables(n, dev)
    _, k, v = fused_rows(n, 2, Hkv, BF, dev, 5)
    cache = paged.new_cache(b.pages, Hkv, ps, dev)
    table, _, _ = b.device(dev)
    off = np.zeros((n, Hkv, 1))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    page = int(b.table[0, 0])
    prev = np.zeros(Hkv)
    for t in range(n):
        paged.append(k[t:t + 1], v[t:t + 1], cache, table, i32([t]), i32([0, 1]), 1, cosd, sind)
        sv = cache["sv"][page].double().cpu().numpy()
        off[t] += 0.5 * sv[:, None]
        off[:t][:, sv > prev] += 0.5 * sv[sv > prev][None, :, None]
        prev = sv
    got = (cache["v"][page].double() * cache["sv"][page].double()[:, None, None]).transpose(0, 1).cpu().numpy()
    assert (np.abs(got - v.double().cpu().numpy()) <= off * (1 + 2.0 ** -18)).all()
    # in one call: half a step of the page's one scale
    paged.append(k, v, cache, table, i32([0]), i32([0, n]), n, cosd, sind)
    s = cache["sk"][page].double().cpu().numpy()[None, :, None]
    got = (cache["k"][page].double() * cache["sk"][page].double()[:, None, None]).transpose(0, 1).cpu().numpy()
    x = k.double().cpu().numpy()
    want = x * cos[:n, None].astype(np.float64) + np.concatenate([-x[..., 64:], x[..., :64]], -1) * sin[:n, None].astype(np.float64)
    # the rotation's three roundings are 2^-24 of values below 2 * 127 s
    assert (np.abs(got - want) <= s * (0.5 + 3 * 254 * 2.0 ** -24)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_of_zeros_infinities_and_nan(dev, dtype):
    """Neither infinities nor NaN move a page's scale: +-127 and 0; a page of zeros has scale 0."""
    from uwc_b200 import paged
    b = Batch([20, 16, 9], [20, 16, 4], 16)
    cos, sin, cosd, sind = tables(32, dev)
    _, k, v = fused_rows(b.rows, 1, 2, dtype, dev, 3)
    v[3, 0, 5], v[4, 1, 0], v[5, 0, 127], v[38, 1, 1] = math.inf, -math.inf, math.nan, math.nan
    v[20:36] = 0
    k[20:36] = 0
    v[30, 1, 7] = math.inf                          # a page of zeros and one infinity: nothing to scale by
    cache = random_cache(b, 2, dev)
    want = append_plain(k.float().cpu().numpy(), v.float().cpu().numpy(), numpy_cache(cache), b, cos, sin)
    paged.append(k, v, cache, *b.device(dev), b.max_new, cosd, sind)
    for name in ("sk", "sv", "k", "v"):
        assert np.array_equal(cache[name].cpu().numpy(), want[name]), name
    assert torch.isfinite(cache["sv"]).all()


def test_append_norms_are_det_rmsnorm(dev):
    """q_norm / k_norm: the oracle's det_rmsnorm before the rotation, bit for bit."""
    import detq
    from uwc_b200 import paged
    b = Batch([70, 64], [70, 1], 64)
    H, Hkv, eps = 4, 2, 1e-6
    cos, sin, cosd, sind = tables(80, dev)
    q, k, v = fused_rows(b.rows, H, Hkv, BF, dev, 11)
    g = torch.Generator(device=dev).manual_seed(2)
    qw, kw = (1 + 0.1 * torch.randn(D, device=dev, generator=g) for _ in range(2))
    norm = lambda x, w: detq.det_rmsnorm(x.float().cpu().numpy().reshape(-1, D), w.cpu().numpy(), eps).reshape(x.shape)
    cache = random_cache(b, Hkv, dev)
    want = append_plain(norm(k, kw), v.float().cpu().numpy(), numpy_cache(cache), b, cos, sin)
    rot = paged.append(k, v, cache, *b.device(dev), b.max_new, cosd, sind, q=q, q_norm=qw, k_norm=kw, eps=eps)
    for name in ("sk", "sv", "k", "v"):
        assert np.array_equal(cache[name].cpu().numpy(), want[name]), name
    pos = np.concatenate([np.arange(70), [63]])
    w = turn(norm(q, qw), cos[pos][:, None], sin[pos][:, None])
    assert torch.equal(rot.cpu(), torch.from_numpy(w).to(BF))


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("ps", [16, 128])
def test_gather_reads_values(dev, ps, dtype):
    from uwc_b200 import paged
    lens = [150, 1, None, 129, 40]
    b = Batch(lens, [150, 1, 2, 7, 0], ps, extra_rows=3)
    cache = random_cache(b, 3, dev)
    table, first, cu = b.device(dev)
    k, v = paged.gather(cache, table, first, cu, b.rows, b.max_new, dtype=dtype)
    for s, (n, m) in enumerate(zip(lens, b.new)):
        r0 = int(b.cu[s])
        if n is None:
            assert not k[r0:r0 + m].any() and not v[r0:r0 + m].any()
            continue
        for t in range(m):
            p = n - m + t
            page = int(b.table[s, p // ps])
            for got, d, sc in ((k, "k", "sk"), (v, "v", "sv")):
                want = (cache[d][page, :, p % ps].float() * cache[sc][page][:, None]).to(dtype)
                assert torch.equal(got[r0 + t], want)


# ------------------------------------------------------------------ attention
def check_attention(dev, b, H, Hkv, dtype, window=None, sinks=0, scale=None, seed=0, spread=1.0, amp=1.0, **kw):
    from uwc_b200 import paged
    cache = random_cache(b, Hkv, dev, seed, spread)
    q, _, _ = fused_rows(b.rows, H, Hkv, dtype, dev, seed, amp)
    table, start, cu = b.device(dev)
    sc = 1 / math.sqrt(D) if scale is None else scale
    o, absv, smax = attention64(q, cache, b, sc, window, sinks)
    out = torch.full((b.rows, H, D), 7.0, dtype=dtype, device=dev)
    got = paged.attention(q, cache, table, start, cu, kw.get("max_new", b.max_new), kw.get("max_len", b.max_len),
                          scale=scale, window=window, sinks=sinks, out=out)
    assert got is out
    used = int(b.cu[-1])
    assert (out[used:] == 7.0).all(), "rows that no sequence covers were written"
    err = (out[:used].double() - o[:used]).abs()
    tol = tolerance(o, absv, smax, dtype)[:used]
    worst = (err - tol).max() if used else torch.tensor(-1.0)
    assert worst <= 0, f"off by {float((err / tol).max()):.2f} tolerances at {int((err / tol).argmax())}"
    again = paged.attention(q, cache, table, start, cu, b.max_new, b.max_len, scale=scale, window=window, sinks=sinks)
    assert torch.equal(again[:used], out[:used]) or "max_new" in kw or "max_len" in kw
    return out


SINGLE = [[1], [2], [15, 16, 17], [63, 64, 65], [127, 128, 129, 1], [500, 3, 1000, 257, 2047]]


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", SINGLE, ids=lambda v: "-".join(map(str, v)))
def test_single_tokens(dev, lens, ps):
    b = Batch(lens, [1] * len(lens), ps, seed=ps)
    check_attention(dev, b, 16, 8, BF, seed=len(lens))
    check_attention(dev, b, 8, 2, HF, seed=len(lens))


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (2, 1), (6, 2), (7, 1), (32, 4), (9, 1), (16, 1), (24, 1), (64, 2)])
def test_head_layouts(dev, H, Hkv):
    b = Batch([300, 17, 64], [1, 1, 1], 32, seed=H)
    check_attention(dev, b, H, Hkv, BF, seed=H)
    b = Batch([300, 17, 64], [40, 17, 3], 32, seed=H)
    check_attention(dev, b, H, Hkv, HF, seed=H)


MASKS = [(None, 0), (0, 0), (0, 3), (1, 0), (1, 1), (5, 2), (64, 0), (100, 4), (128, 130), (257, 16), (5000, 4)]


@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("ps", [16, 64])
def test_masks_single_tokens(dev, window, sinks, ps):
    lens = [1, 5, 64, 130, 700, 1301]
    check_attention(dev, Batch(lens, [1] * 6, ps), 8, 2, BF, window, sinks)


@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("ps", [16, 128])
def test_masks_many_rows(dev, window, sinks, ps):
    lens, new = [1, 5, 400, 130, 700, 1301], [1, 5, 400, 1, 200, 300]
    check_attention(dev, Batch(lens, new, ps), 4, 2, HF, window, sinks)
    check_attention(dev, Batch(lens, new, ps), 4, 1, BF, window, sinks)


@pytest.mark.parametrize("new", [[2, 1, 2], [3, 3, 1], [4, 4, 4], [8, 1, 5], [16, 2, 16], [33, 1, 32], [65, 64, 63],
                                 [129, 128, 127], [256, 255, 257], [511, 1, 513]], ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("back", [0, 1, 777])
def test_new_token_counts(dev, new, back):
    b = Batch([n + back for n in new], new, 64, seed=back)
    check_attention(dev, b, 8, 4, BF, seed=back)
    check_attention(dev, b, 8, 1, HF, seed=back, window=90, sinks=4)


def test_idle_slots_and_empty_sequences(dev):
    for new in ([1, 1, 0, 1, 1], [70, 20, 0, 1, 33]):
        b = Batch([200, None, 50, 1, 90], new, 16, extra_rows=5)
        out = check_attention(dev, b, 8, 2, BF)
        r0 = int(b.cu[1])
        assert not out[r0:r0 + new[1]].any()


def test_rows_that_see_nothing_are_zero(dev):
    for new in ([1, 1], [50, 30]):
        b = Batch([300, 40], new, 64)
        out = check_attention(dev, b, 4, 2, BF, window=0, sinks=0)
        assert not out[:int(b.cu[-1])].any()


@pytest.mark.parametrize("new", [1, 90])
def test_loose_bounds_and_wide_tables(dev, new):
    """max_new and max_len are bounds, the table may be wider than any sequence."""
    b = Batch([700, 301, 64], [new, min(new, 33), 1], 64, width=40)
    check_attention(dev, b, 8, 2, BF, max_new=300, max_len=2500)


def test_max_len_too_small_is_slow_not_wrong(dev):
    b = Batch([3000, 301], [1, 1], 64)
    check_attention(dev, b, 8, 2, BF, max_len=10)
    b = Batch([3000, 301], [100, 1], 64)
    check_attention(dev, b, 8, 2, BF, max_len=10)


@pytest.mark.parametrize("new", [1, 60])
def test_scales_far_apart(dev, new):
    """Pages whose scales lie orders of magnitude apart, among them the keys that the softmax picks."""
    for seed in range(3):
        check_attention(dev, Batch([800, 333], [new, new], 16, seed=seed), 8, 2, HF, seed=seed, spread=3.0, amp=0.3)


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("amp", [1e-6, 30.0])
def test_flat_and_peaked_scores(dev, amp, new):
    check_attention(dev, Batch([800, 333], [new, new], 64), 8, 2, BF, amp=amp)


def test_negative_and_large_scale_argument(dev):
    for new in (1, 40):
        check_attention(dev, Batch([300, 20], [new, 7], 32), 4, 2, BF, scale=-0.05)
        check_attention(dev, Batch([300, 20], [new, 7], 32), 4, 2, BF, scale=0.0)


@pytest.mark.parametrize("new", [1, 5, 80])
def test_nan_in_a_row_stays_in_it(dev, new):
    from uwc_b200 import paged
    b = Batch([200, 90], [new, min(new, 9)], 64)
    cache = random_cache(b, 2, dev)
    q, _, _ = fused_rows(b.rows, 8, 2, BF, dev, 1)
    table, start, cu = b.device(dev)
    good = paged.attention(q, cache, table, start, cu, b.max_new, b.max_len)
    q[0, 3, 17] = math.nan
    got = paged.attention(q, cache, table, start, cu, b.max_new, b.max_len)
    assert got[0, 3].isnan().all()
    got[0, 3] = good[0, 3]
    assert torch.equal(got, good)


@pytest.mark.parametrize("new", [1, 70])
def test_what_the_mask_hides_is_not_read(dev, new):
    """Values and scales past a sequence's end, in unseen pages and in pages of others may be anything."""
    from uwc_b200 import paged
    lens = [333, 40]
    b = Batch(lens, [new, min(new, 40)], 64, spare=3)
    cache = random_cache(b, 2, dev)
    q, _, _ = fused_rows(b.rows, 4, 2, HF, dev, 1)
    table, start, cu = b.device(dev)
    args = dict(window=100, sinks=2)
    good = paged.attention(q, cache, table, start, cu, b.max_new, b.max_len, **args)
    mine = set(int(x) for x in b.table.ravel() if x >= 0)
    # sequence 0 sees the sinks' page and those from position 333 - new - 99 on
    lo = (333 - new - 99) // 64
    unseen = set(range(b.pages)) - mine | {int(b.table[0, i]) for i in range(1, lo)}
    assert unseen
    for p in unseen:
        cache["sk"][p], cache["sv"][p] = math.nan, math.inf
        cache["k"][p], cache["v"][p] = -128, 127
    last = int(b.table[0, 5])
    cache["k"][last, :, 333 % 64:], cache["v"][last, :, 333 % 64:] = 127, -128
    wide = torch.full((2, 40), 1 << 30, dtype=torch.int32, device=dev)     # entries past the end: never read
    for s, n in enumerate(lens):
        wide[s, :-(-n // 64)] = table[s, :-(-n // 64)]
    got = paged.attention(q, cache, wide, start, cu, b.max_new, b.max_len, **args)
    assert torch.equal(got, good)


def test_offsets_past_32_bits(dev):
    """A pool of over 2^31 bytes: the sequence's pages lie at its end."""
    from uwc_b200 import paged
    pages, Hkv, ps = 17000, 8, 128
    e = lambda *s, dt=torch.int8: torch.empty(*s, dtype=dt, device=dev)
    cache = dict(k=e(pages, Hkv, ps, D), v=e(pages, Hkv, ps, D), sk=e(pages, Hkv, dt=torch.float32),
                 sv=e(pages, Hkv, dt=torch.float32))
    assert cache["k"].numel() > 2 ** 31
    for new in ([1, 1], [300, 40]):
        b = Batch([600, 200], new, ps)
        small = random_cache(b, Hkv, dev)
        at = pages - b.pages
        for n in cache:
            cache[n][at:] = small[n]
        q, k, v = fused_rows(b.rows, 16, Hkv, BF, dev, 2)
        table, start, cu = b.device(dev)
        far = torch.where(table >= 0, table + at, -1).to(torch.int32)
        cos, sin, cosd, sind = tables(600, dev)
        for c, t in ((small, table), (cache, far)):
            paged.append(k, v, c, t, start, cu, b.max_new, cosd, sind)
        assert all(torch.equal(cache[n][at:], small[n]) for n in cache)
        near = paged.attention(q, small, table, start, cu, b.max_new, b.max_len)
        assert torch.equal(paged.attention(q, cache, far, start, cu, b.max_new, b.max_len), near)
        g0, g1 = (paged.gather(c, t, start, cu, b.rows, b.max_new) for c, t in ((small, table), (cache, far)))
        assert torch.equal(g0[0], g1[0]) and torch.equal(g0[1], g1[1])


def test_strided_rows(dev):
    """Token and head strides other than the fused row's: a head-major tensor and every second token."""
    from uwc_b200 import paged
    b = Batch([150, 20], [60, 5], 16)
    cache = random_cache(b, 2, dev)
    table, start, cu = b.device(dev)
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(8, 2 * b.rows, D, device=dev, generator=g).to(HF)
    q = x.transpose(0, 1)[::2]
    assert q.stride() == (2 * D, 2 * b.rows * D, 1)
    dense = q.contiguous()
    a, c = (paged.attention(t, cache, table, start, cu, b.max_new, b.max_len) for t in (q, dense))
    assert torch.equal(a, c)
    _, _, cosd, sind = tables(160, dev)
    one, two = ({n: t.clone() for n, t in cache.items()} for _ in range(2))
    r1 = paged.append(q[:, :2], q[:, 2:4], one, table, start, cu, b.max_new, cosd, sind, q=q)
    r2 = paged.append(dense[:, :2].contiguous(), dense[:, 2:4].contiguous(), two, table, start, cu, b.max_new, cosd, sind, q=dense)
    assert torch.equal(r1, r2) and all(torch.equal(one[n], two[n]) for n in one)


def test_batch_and_splits_do_not_share_state(dev):
    """Calls of different shapes in a row on two streams: each gives what it gives alone."""
    from uwc_b200 import paged
    shapes = [(Batch([5000], [1], 64), 8, 2), (Batch([700] * 9, [1] * 9, 16), 16, 8), (Batch([3000], [80], 64), 8, 2),
              (Batch([1], [1], 128), 4, 4), (Batch([9000, 20], [3, 3], 128), 4, 1)]
    work = []
    for i, (b, H, Hkv) in enumerate(shapes):
        cache, (q, _, _) = random_cache(b, Hkv, dev, i), fused_rows(b.rows, H, Hkv, BF, dev, i)
        work.append((q, cache, *b.device(dev), b.max_new, b.max_len))
    alone = []
    for w in work:
        alone.append(paged.attention(*w))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for r in range(6):
        for i, w in enumerate(work):
            with torch.cuda.stream(streams[(i + r) % 2]):
                got.append((i, paged.attention(*w)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i, o in got)


@pytest.mark.parametrize("H,Hkv", [(8, 2), (32, 1)])
def test_one_graph_serves_every_step(dev, H, Hkv):
    """append + attention captured once over static buffers, replayed with other positions and rows."""
    from uwc_b200 import paged
    S, ps, cap = 3, 16, 256
    table = torch.arange(S * cap // ps, dtype=torch.int32, device=dev).view(S, -1)
    _, _, cosd, sind = tables(cap, dev)
    q, k, v = fused_rows(S, H, Hkv, BF, dev, 0)
    start = torch.zeros(S, dtype=torch.int32, device=dev)
    cu = torch.arange(S + 1, dtype=torch.int32, device=dev)
    caches = [paged.new_cache(S * cap // ps, Hkv, ps, dev) for _ in range(2)]

    def step(c):
        return paged.attention(paged.append(k, v, c, table, start, cu, 1, cosd, sind, q=q), c, table, start, cu, 1, cap)
    step(caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    for t in caches[0].values():
        t.zero_()                                 # the two warm-up steps' tokens
    for t in range(40):
        for x, y in zip((q, k, v), fused_rows(S, H, Hkv, BF, dev, t)):
            x.copy_(y)
        start.copy_(torch.tensor([t, 2 * t, -1 if t % 3 == 0 else t], dtype=torch.int32))
        graph.replay()
        want = step(caches[1])
        assert torch.equal(out, want), t


# ------------------------------------------------------------------ metadata out of range
def test_metadata_out_of_range_is_skipped_and_reported(dev):
    from uwc_b200 import _lib, paged
    b = Batch([100, 80], [1, 60], 16)
    cache = random_cache(b, 2, dev)
    q, k, v = fused_rows(b.rows, 4, 2, BF, dev, 0)
    table, start, cu = b.device(dev)
    _, _, cosd, sind = tables(128, dev)
    reported = lambda: _lib.device_status(clear=True)

    def both(t, s, c, max_new, cos=cosd, sin=sind):
        before = {n: x.clone() for n, x in cache.items()}
        paged.append(k, v, cache, t, s, c, max_new, cos, sin, q=q)
        one = reported()
        same = {n: torch.equal(cache[n], before[n]) for n in cache}
        for n in cache:
            cache[n].copy_(before[n])
        paged.attention(q, cache, t, s, c, max_new, 128)
        return one, reported(), same

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    bad = table.clone()
    bad[0, 6] = b.pages                                     # the new token's page lies outside the pool
    assert both(bad, start, cu, 60)[:2] == (2, 2)
    bad[0, 6] = -1
    assert both(bad, start, cu, 60)[:2] == (2, 2)
    assert both(table, i32([16 * b.width, 20]), cu, 60)[:2] == (2, 2)        # past the table
    assert both(table, i32([2 ** 31 - 1, 20]), cu, 60)[:2] == (2, 2)
    assert both(table, start, i32([0, 1, 100]), 60)[:2] == (2, 2)            # rows past the tensors
    assert both(table, start, i32([-5, 1, 61]), 60)[:2] == (2, 2)
    assert both(table, start, i32([0, -7, 61]), 60)[:2] == (2, 2)
    assert both(table, start, cu, 59)[:2] == (2, 2)                          # more new tokens than max_new
    one, two, same = both(table, start, cu, 60, cosd[:64].contiguous(), sind[:64].contiguous())   # no rotation row
    assert (one, two) == (2, 0)
    one, two, same = both(table, i32([-1, -4]), cu, 60)                      # idle: nothing is touched
    assert (one, two) == (0, 0) and all(same.values())
    first = i32([0, 0])
    paged.gather(cache, bad, first, i32([0, 100, 100]), 100, 100)
    assert reported() == 2
