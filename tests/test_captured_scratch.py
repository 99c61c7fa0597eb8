"""Scratch that a CUDA graph was captured with: it belongs to the graph, so that calls of more rows between two
replays, which replace the device's buffer by a larger one, leave the graph's alone."""
import pytest
import torch


class Spy:
    """The library, with the scratch pointers of uwc_gemm_epi noted and whether a capture was under way."""

    def __init__(self, real):
        self.real, self.seen = real, []

    def __getattr__(self, name):
        f = getattr(self.real, name)
        if name != "uwc_gemm_epi":
            return f

        def call(*args):
            self.seen.append((args[10], args[11], torch.cuda.is_current_stream_capturing()))
            return f(*args)
        return call


def test_a_capture_gets_scratch_of_its_own(monkeypatch):
    from uwc_b200 import ops

    class Sizes:
        @staticmethod
        def uwc_gemm_workspace_bytes(m, n, flags, out_mode):
            return m
    monkeypatch.setattr(ops, "lib", lambda: Sizes)
    monkeypatch.setattr(ops, "_GEMM_WS", {})
    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    get = lambda m: ops.gemm_workspace("cpu", m, 8, 0, 1)
    assert get(0) is None
    kept = get(1000)
    assert get(400) is kept and ops._GEMM_WS == {"cpu": kept}
    capturing = True
    own = get(500)
    assert own.numel() == 500 and own.data_ptr() != kept.data_ptr() and ops._GEMM_WS == {"cpu": kept}
    big = get(5000)
    assert big.numel() == 5000 and ops._GEMM_WS == {"cpu": kept}


@pytest.mark.gpu
def test_a_batch_of_many_slots_keeps_its_scratch(dev, monkeypatch):
    """100 slots: a step's products of 100 rows split k and need scratch; a prompt of 300 tokens needs more."""
    pytest.importorskip("transformers")
    import model_fixture as mf
    from uwc_b200 import ops
    from uwc_b200.detmodel import DetQwen3
    from uwc_b200.serve import PagedBatch
    model = DetQwen3(mf.tiny_model(), dev, hadamard_block=mf.HADAMARD_BLOCK, max_pos=512)
    spy = Spy(ops.lib())
    monkeypatch.setattr(ops, "lib", lambda: spy)
    b = PagedBatch(model, 100, 400, pages=100, page_size=16)
    captured = [(p, n) for p, n, c in spy.seen if c and p]
    assert captured
    pool = b._graph.pool()
    segments = [(s["address"], s["address"] + s["total_size"], tuple(s["segment_pool_id"]))
                for s in torch.cuda.memory_snapshot()]
    for p, n in captured:
        assert [q for a, e, q in segments if a <= p and p + n <= e] == [tuple(pool)]
    # more rows between the replays: the tokens are those of the same calls without a graph
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (3, 300, 20)]
    eager = PagedBatch(model, 100, 400, pages=100, page_size=16, graph=False)
    for x in (b, eager):
        x.said = [x.admit(prompts[:1]), x.step(), x.admit(prompts[1:]), x.step(), x.step()]
    assert b.said == eager.said


def allocated(p):
    """Whether torch's allocator holds the address for some tensor."""
    for s in torch.cuda.memory_snapshot():
        at = s["address"]
        for x in s["blocks"]:
            if at <= p < at + x["size"]:
                return x["state"] == "active_allocated"
            at += x["size"]
    return False


@pytest.mark.gpu
def test_a_graphed_forward_keeps_its_workspace(dev, monkeypatch):
    """The weights of a device share a workspace; a graph's outlives its replacement by a larger one."""
    from uwc_b200 import ops
    monkeypatch.setattr(ops, "_SHARED_WS", {})
    m, n, k = 256, 512, 2048
    g = torch.Generator(device=dev).manual_seed(3)
    i8 = lambda *s: torch.randint(-64, 65, s, device=dev, generator=g, dtype=torch.int8)
    A = i8(m, k)
    w = ops.MinedWeight(Bt=i8(n, k), b_scale=torch.ones(n, device=dev))
    w.setup_block(bytes(range(32)), [0] * 8)
    gf = ops.GraphedForward(w, m, out_mode=ops.OUT_I32)
    p = w._last_ws[m][0].data_ptr()
    ops.shared_workspace(dev, 2 * w._last_ws[m][0].numel())
    want = w.forward(A, gf.a_scale, out_mode=ops.OUT_I32)        # on the larger one
    assert w._last_ws[m][0].data_ptr() != p and allocated(p)
    gf.A.copy_(A)
    assert torch.equal(gf(), want)
