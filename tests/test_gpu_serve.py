"""PagedBatch (uwc_b200.serve) on a B200: the paged operators as a model calls them. Every attention call that
it makes is checked against 64 bits on its own cache, a decode graph against the same step run call by call, the
hidden rows against the deterministic forward, and the bookkeeping of sequences that come, draft and go."""
import numpy as np
import pytest
import torch

from paged_fixture import Batch, attention64, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(dev):
    pytest.importorskip("transformers")
    import model_fixture as mf
    from uwc_b200.detmodel import DetQwen3
    return DetQwen3(mf.tiny_model(), dev, hadamard_block=mf.HADAMARD_BLOCK, max_pos=512)


@pytest.fixture(autouse=True)
def status_clean(dev):
    from uwc_b200 import _lib
    _lib.device_status(clear=True)
    yield
    assert _lib.device_status(clear=True) == 0, "a paged kernel reported metadata out of range"


@pytest.fixture
def checked(monkeypatch):
    """Checks every paged.attention call against the definition, within paged_fixture's tolerance."""
    from uwc_b200 import paged
    real, calls = paged.attention, []

    def attention(q, cache, table, start, cu, max_new, max_len, scale=None, window=None, sinks=0):
        o = real(q, cache, table, start, cu, max_new, max_len, scale=scale, window=window, sinks=sinks)
        at, end = start.tolist(), cu.tolist()
        new = [b - a for a, b in zip(end, end[1:])]
        b = Batch([None if a < 0 else a + m for a, m in zip(at, new)], new, cache["k"].shape[2])
        b.table, b.cu = table.cpu().numpy(), np.asarray(end, np.int32)
        assert b.max_len <= max_len and b.max_new <= max_new
        w, absv, smax = attention64(q, cache, b, scale, window, sinks)
        assert bool(((o.double() - w).abs() <= tolerance(w, absv, smax, o.dtype)).all())
        calls.append(q.shape[0])
        return o

    monkeypatch.setattr(paged, "attention", attention)
    return calls


def prompts(*lens):
    g = torch.Generator().manual_seed(sum(lens))
    return [torch.randint(0, 1024, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("window,sinks,page_size", [(None, 0, 64), (40, 4, 16)])
def test_calls_hold_and_hiddens_follow_the_deterministic_forward(dev, model, checked, window, sinks, page_size):
    """Four ragged prompts in chunks of 50, then steps. Without a window the last rows' final hidden is compared
    with DetQwen3.forward. The two differ where a row is quantized: 1/64 of the row's largest, which is about 4
    standard deviations, so a step of 1/16 and an error of 1/16 / sqrt(12) = 0.018 of a row's size each time; apart
    by sqrt 2 of it, over the model's 8 quantized products 0.026 * sqrt 8 = 0.073 if the residual stream had
    nothing else. 0.1 is allowed."""
    from uwc_b200 import detgpu
    from uwc_b200.serve import PagedBatch
    ps = prompts(1, 37, 64, 130)
    b = PagedBatch(model, 4, 160, page_size=page_size, window=window, sinks=sinks, graph=False)
    seen = []
    real = b._greedy
    b._greedy = lambda x: (seen.append(detgpu.rmsnorm(x, model.norm, model.eps)), real(x))[1]
    toks = [[t] for t in b.admit(ps, chunk=50).values()]
    for _ in range(3):
        for t, n in zip(toks, b.step().values()):
            t.append(n)
    assert len(checked) == 2 * (3 + 3)                      # layers x (chunks + steps)
    if window is None:
        for s, p in enumerate(ps):
            full = torch.tensor([p + toks[s][:-1]], device=dev)
            want = model.forward(full, model.new_cache(1, full.shape[1]), 0)[0, len(p) - 1:]
            got = torch.stack([h[s] for h in seen])
            assert float((got - want).norm() / want.norm()) < 0.1, s


def test_graph_equals_calls(dev, model):
    """The captured step gives the eager step's tokens and cache, bit for bit, with an idle slot among them and
    pages taken on the way."""
    from uwc_b200.serve import PagedBatch
    out = []
    for graph in (False, True):
        b = PagedBatch(model, 5, 200, page_size=16, graph=graph)
        got = [b.admit(prompts(30, 1, 16, 90))]
        got += [b.step() for _ in range(20)]
        b.release(1)
        got += [b.step() for _ in range(3)]
        assert b.active() == [0, 2, 3] and b.len == [53, -1, 39, 113, -1]
        out.append((got, [b.read(s, layer, dtype=torch.float32) for s in (0, 2, 3) for layer in (0, 1)]))
    assert out[0][0] == out[1][0]
    for x, y in zip(out[0][1], out[1][1]):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_drafts(dev, model, checked):
    """A slot keeps the drafts that the model itself would have said and its correction of the next."""
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 3, 128, page_size=32, graph=False)
    first = b.admit(prompts(20, 31, 50))
    checked.clear()
    no_draft = b.verify({0: []})
    assert len(no_draft[0]) == 1 and b.len == [21, 31, 50]
    wrong = {s: [(t + 1) % 1024] * 4 for s, t in first.items()}
    got = b.verify(wrong)
    for s, n in zip(range(3), (21, 31, 50)):
        k = len(got[s])
        assert got[s][:k - 1] == wrong[s][:k - 1] and (k == 5 or got[s][k - 1] != wrong[s][k - 1])
        assert b.len[s] == n + k
    # drafts that repeat what verify itself answers are confirmed as far as they go
    for _ in range(4):
        before = list(b.len)
        guess = {s: [got[s][-1], 7] for s in (0, 2)}
        said = b.verify(guess)
        for s in (0, 2):
            k = len(said[s])
            assert said[s][:k - 1] == guess[s][:k - 1] and b.len[s] == before[s] + k
        assert b.len[1] == before[1]
        got.update(said)
    assert checked and b.step().keys() == {0, 1, 2}


def test_sequences_come_and_go(dev, model):
    """More prompts than slots and pages; the pool is whole again at the end."""
    from uwc_b200 import _lib
    from uwc_b200.serve import PagedBatch
    ps = prompts(40, 3, 17, 64, 9)
    b = PagedBatch(model, 2, 96, pages=9, page_size=16)
    out = b.generate(ps, 6)
    assert [len(t) for t in out] == [6] * 5 and all(0 <= x < 1024 for t in out for x in t)
    assert sorted(b.pool.free) == list(range(9)) and not b.active()
    assert b.generate([], 6) == [] and b.generate(ps, 0) == [[]] * 5 and b.step() == {} and b.verify({}) == {}
    with pytest.raises(_lib.UWCError):
        b.admit(ps)                                         # three more than slots
    with pytest.raises(ValueError):
        b.admit([[]])
    with pytest.raises(ValueError):
        b.admit([ps[3]], reserve=40)                        # past max_len
    b.admit(prompts(90, 40))
    with pytest.raises(ValueError):
        b.verify({0: [1] * 6})                              # past max_len
    for _ in range(6):
        b.step()
    with pytest.raises(ValueError):
        b.step()                                            # slot 0 holds max_len tokens
    with pytest.raises(_lib.UWCError):
        b.generate(ps, 1)
    with pytest.raises(ValueError):
        b.read(0, 0, 90, 7)
    b.release(0)
    with pytest.raises(ValueError):
        b.release(0)
    with pytest.raises(ValueError):
        b.verify({0: [1]})
    assert list(b.step()) == [1]


def test_pool_runs_out(dev, model):
    from uwc_b200 import _lib
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 2, 96, pages=4, page_size=16)
    b.admit(prompts(32, 32))
    with pytest.raises(_lib.UWCError):
        b.step()                                            # both want a third page
    b.release(1)
    assert list(b.step()) == [0] and b.len == [33, -1]


def test_refusals(dev, model):
    from uwc_b200.serve import PagedBatch
    for slots, max_len, ps in ((0, 10, 64), (1, 0, 64), (1, 513, 64), (1, 64, 48)):
        with pytest.raises(ValueError):
            PagedBatch(model, slots, max_len, page_size=ps)
