"""PagedBatch.generate at its limits: prompts that cannot be served are refused before any is, what exactly fits is
served, and a call that fails leaves the batch as it found it."""
import pytest
import torch

from test_gpu_serve import model, prompts, status_clean  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def whole(b, pages):
    return not b.active() and sorted(b.pool.free) == list(range(pages)) and bool((b._table == -1).all())


def test_a_bad_prompt_is_refused_before_any_is_served(dev, model):
    from uwc_b200 import _lib
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 2, 96, pages=5, page_size=16, graph=False)
    good = prompts(20, 3, 17, 33)
    calls = []
    real = b._rows
    b._rows = lambda *a: (calls.append(1), real(*a))[1]
    for bad, error in (([], ValueError), (prompts(95)[0], ValueError), (prompts(80)[0], _lib.UWCError)):
        with pytest.raises(error):                          # empty; 95 + 4 of 96 tokens; 6 of 5 pages
            b.generate(good + [bad], 5)
        assert not calls and whole(b, 5)
    out = b.generate(good, 5)
    assert [len(t) for t in out] == [5] * 4 and whole(b, 5)
    one = PagedBatch(model, 1, 96, page_size=16, graph=False)
    assert [one.generate([p], 5)[0] for p in good] == out


def test_what_exactly_fits_is_served(dev, model):
    """The last token is answered and not cached: 90 + 7 - 1 of 96 tokens, and a page of 16 for 12 + 5 - 1."""
    from uwc_b200.serve import PagedBatch
    long, short = prompts(90)[0], prompts(12)[0]
    b = PagedBatch(model, 1, 96, pages=6, page_size=16, graph=False)
    out = b.generate([long], 7)[0]
    with pytest.raises(ValueError):
        b.generate([long], 8)
    roomy = PagedBatch(model, 1, 200, page_size=16, graph=False)
    assert len(out) == 7 and out == roomy.generate([long], 7)[0]
    one = PagedBatch(model, 3, 96, pages=1, page_size=16, graph=False)
    assert one.generate([short, short[:3], short], 5) == roomy.generate([short, short[:3], short], 5) and whole(one, 1)
    assert one.generate([prompts(16)[0]], 1) == roomy.generate([prompts(16)[0]], 1)


@pytest.mark.parametrize("at", [0, 1, 2, 3, 5])
def test_a_call_that_fails_leaves_the_batch_as_it_was(dev, model, at):
    """An exception in the at-th pass through the model, of an admission or of a step: no slot and no page is lost."""
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 2, 96, pages=8, page_size=16, graph=False)
    ps = prompts(40, 3, 17, 33)
    want = b.generate(ps, 4)
    real, seen = b._greedy, []

    def failing(x):
        seen.append(1)
        if len(seen) == at + 1:
            raise MemoryError("planted")
        return real(x)
    b._greedy = failing
    with pytest.raises(MemoryError):
        b.generate(ps, 4)
    assert len(seen) == at + 1 and whole(b, 8)
    b._greedy = real
    assert b.generate(ps, 4) == want and whole(b, 8)


def test_an_admission_that_fails_takes_nothing(dev, model):
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 3, 96, pages=8, page_size=16, graph=False)
    ps = prompts(40, 20)
    b.admit(ps[:1])
    free = list(b.pool.free)
    real, b._greedy = b._greedy, None                       # not callable
    with pytest.raises(TypeError):
        b.admit(ps[1:], reserve=3)
    b._greedy = real
    assert b.active() == [0] and sorted(b.pool.free) == sorted(free) and bool((b._table[1:] == -1).all())
    b.admit(ps[1:])
    assert b.active() == [0, 1] and list(b.step()) == [0, 1]


def test_chunks_and_reserves_are_checked(dev, model):
    """A reserve below 0 took fewer pages than the prompt fills."""
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 2, 96, pages=8, page_size=16, graph=False)
    for bad in (dict(chunk=0), dict(chunk=-5), dict(reserve=-1), dict(reserve=-40)):
        with pytest.raises(ValueError):
            b.admit(prompts(40), **bad)
        assert whole(b, 8)


@pytest.mark.parametrize("bad", [-1, 1024, 2 ** 31, -2 ** 40])
def test_tokens_that_the_model_has_not_are_refused(dev, model, bad):
    from uwc_b200.serve import PagedBatch
    b = PagedBatch(model, 2, 96, pages=8, page_size=16, graph=False)
    assert model.embed.shape[0] == 1024
    for call in (lambda: b.admit([[5, bad, 7]]), lambda: b.generate([[5], [bad]], 3)):
        with pytest.raises(ValueError):
            call()
        assert whole(b, 8)
    b.admit([[5, 0, 1023]])
    free = len(b.pool.free)
    with pytest.raises(ValueError):
        b.verify({0: [3, bad]})
    assert b.len[0] == 3 and len(b.pool.free) == free and len(b.verify({0: [0, 1023]})[0]) >= 1


def test_prompts_and_drafts_of_any_sequence_type(dev, model):
    """Lists, tuples, arrays and tensors of token ids."""
    import numpy as np
    from uwc_b200.serve import PagedBatch
    ps = prompts(20, 3)
    b = PagedBatch(model, 2, 96, pages=8, page_size=16, graph=False)
    want = b.generate(ps, 4)
    for make in (tuple, np.array, torch.tensor):
        assert b.generate([make(p) for p in ps], 4) == want
        b.admit([make(p) for p in ps])
        said = b.verify({0: make(want[0][1:3]), 1: make([])})
        assert said[0] == want[0][1:4] and said[1] == want[1][1:2]
        b.release(0)
        b.release(1)
        with pytest.raises(ValueError):
            b.admit([make([7, 1024])])
