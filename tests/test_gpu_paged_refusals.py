"""What uwc_b200.paged refuses, on tensors of a device: every check of its torch side, each from a call that is right but
for one argument, and none of them leaves anything written."""
import pytest
import torch

from paged_fixture import D, Batch, random_cache
from test_gpu_paged import BF, HF, fused_rows, status_clean, tables  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def good(dev):
    b = Batch([100, 40], [3, 2], 16)
    table, start, cu = b.device(dev)
    q, k, v = fused_rows(5, 4, 2, BF, dev, 0)
    _, _, cos, sin = tables(128, dev)
    return dict(cache=random_cache(b, 2, dev), table=table, start=start, cu=cu, q=q, k=k, v=v, cos=cos, sin=sin)


def calls(a):
    from uwc_b200 import paged
    c = (a["cache"], a["table"], a["start"], a["cu"])
    return dict(append=lambda **o: paged.append(a["k"], a["v"], *c, a.get("max_new", 3), a["cos"], a["sin"], q=a["q"], **o),
                attention=lambda **o: paged.attention(a["q"], *c, a.get("max_new", 3), a.get("max_len", 100), **o),
                gather=lambda **o: paged.gather(*c, a.get("n", 5), a.get("max_rows", 3), **o))


ALL, ROWS, ATT, APP, GAT = ("append", "attention", "gather"), ("append", "attention"), ("attention",), ("append",), ("gather",)
wide = lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]]   # the same values, not contiguous
CASES = [
    # what is replaced, by what of itself, who refuses it
    ("cache.k", lambda t: t.cpu(), ALL), ("cache.v", lambda t: t.cpu(), ALL), ("cache.sk", lambda t: t.cpu(), ALL),
    ("cache.sv", lambda t: t.cpu(), ALL), ("cache.k", lambda t: None, ALL), ("cache.sv", lambda t: 3, ALL),
    ("cache.k", lambda t: t.view(torch.uint8), ALL), ("cache.v", lambda t: t.short(), ALL), ("cache.sk", lambda t: t.half(), ALL),
    ("cache.sv", lambda t: t.double(), ALL), ("cache.k", lambda t: t[..., :64], ALL), ("cache.k", lambda t: t[0], ALL),
    ("cache.v", lambda t: t[:-1], ALL), ("cache.v", lambda t: t[:, :1], ALL), ("cache.sk", lambda t: t[:-1], ALL),
    ("cache.sv", lambda t: t[:, :1], ALL), ("cache.k", lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), ALL),
    ("cache.v", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), ALL),
    ("cache.sk", lambda t: t.t().contiguous().t(), ALL),
    ("table", lambda t: t.cpu(), ALL), ("start", lambda t: t.cpu(), ALL), ("cu", lambda t: t.cpu(), ALL),
    ("table", lambda t: t.long(), ALL), ("start", lambda t: t.long(), ALL), ("cu", lambda t: t.float(), ALL),
    ("table", lambda t: t[:1], ALL), ("table", lambda t: t[0], ALL), ("start", lambda t: t[:1], ALL), ("cu", lambda t: t[:2], ALL),
    ("cu", lambda t: t[None], ALL), ("table", wide, ALL), ("table", lambda t: t[:, :0], ALL), ("table", lambda t: None, ALL),
    ("start", lambda t: [97, 38], ALL), ("cu", lambda t: (0, 3, 5), ALL),
    ("q", lambda t: t.cpu(), ROWS), ("q", lambda t: t.float(), ROWS), ("q", lambda t: t[0], ROWS), ("q", lambda t: t[..., :64], ROWS),
    ("q", lambda t: t[..., ::2].repeat(1, 1, 2)[..., ::2], ROWS), ("q", lambda t: t.transpose(1, 2), ROWS),
    ("q", lambda t: t[:, :3], ATT), ("q", lambda t: t[:, :0], ATT), ("q", lambda t: t[:4], APP), ("q", lambda t: t.half(), APP),
    ("q", lambda t: torch.zeros(5, 4 * D + 4, dtype=BF, device=t.device)[:, 4:].view(5, 4, D), ROWS),          # 8 bytes off
    ("q", lambda t: torch.zeros(5, 4 * D + 4, dtype=BF, device=t.device)[:, :4 * D].view(5, 4, D), ROWS),      # a stride of 4 past
    ("k", lambda t: t.cpu(), APP), ("k", lambda t: t.double(), APP), ("k", lambda t: t[:, :1], APP), ("v", lambda t: t[:4], APP),
    ("v", lambda t: t.half(), APP), ("v", lambda t: t[..., :64], APP), ("k", lambda t: None, APP), ("v", lambda t: 1.0, APP),
    ("cos", lambda t: t.cpu(), APP), ("cos", lambda t: t.half(), APP), ("sin", lambda t: t[:, :64], APP), ("sin", lambda t: t[:64], APP),
    ("cos", wide, APP), ("sin", lambda t: t[0], APP),
    ("max_new", lambda _: -1, ROWS), ("max_new", lambda _: 2 ** 30 + 1, ROWS), ("max_new", lambda _: 2 ** 40, ROWS),
    ("max_len", lambda _: -1, ATT), ("max_len", lambda _: 2 ** 31, ATT), ("n", lambda _: -1, GAT), ("n", lambda _: 2 ** 32, GAT),
    ("max_rows", lambda _: -3, GAT),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_one_wrong_argument(dev, case):
    what, wrong, who = CASES[case]
    a = good(dev)
    before = {n: t.clone() for n, t in a["cache"].items()}
    group, name = (a["cache"], what[6:]) if what.startswith("cache.") else (a, what)
    right = group.get(name)
    group[name] = wrong(right)
    for f in who:
        with pytest.raises(AssertionError):
            calls(a)[f]()
    group[name] = right
    torch.cuda.synchronize()
    assert all(torch.equal(before[n], a["cache"][n]) for n in before)


def test_the_calls_are_right_otherwise(dev):
    a = good(dev)
    for call in calls(a).values():
        call()


@pytest.mark.parametrize("which", ["q_norm", "k_norm"])
@pytest.mark.parametrize("wrong", [lambda w: w.cpu(), lambda w: w.half(), lambda w: w[:64], lambda w: w[None], lambda w: 1.0,
                                   lambda w: torch.cat([w, w])[::2]], ids=range(6))
def test_norm_weights(dev, which, wrong):
    a = good(dev)
    before = {n: t.clone() for n, t in a["cache"].items()}
    with pytest.raises(AssertionError):
        calls(a)["append"](**{which: wrong(torch.ones(D, device=dev))})
    assert all(torch.equal(before[n], a["cache"][n]) for n in before)


@pytest.mark.parametrize("wrong", [lambda t: t.cpu(), lambda t: t.half(), lambda t: t[:4], lambda t: t[:, :2], lambda t: 0,
                                   lambda t: torch.cat([t, t], 1)[:, :4]], ids=range(6))
def test_outputs(dev, wrong):
    a = good(dev)
    out = torch.full((5, 4, D), 7.0, dtype=BF, device=dev)
    with pytest.raises(AssertionError):
        calls(a)["attention"](out=wrong(out))
    assert (out == 7.0).all()


def test_what_is_no_number(dev):
    a = good(dev)
    for f, bad in (("attention", dict(scale="1")), ("attention", dict(window="8")), ("attention", dict(sinks=None)),
                   ("append", dict(eps="x"))):
        with pytest.raises(TypeError):
            calls(a)[f](**bad)
    with pytest.raises(OverflowError):
        calls(a)["attention"](window=2 ** 70)
    with pytest.raises(KeyError):
        calls(a)["gather"](dtype=torch.int8)
