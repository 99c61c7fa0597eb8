"""MinedWeight.winners and the device status: a timeout invalidates the records and is cleared, what a paged call
reported is neither a reason to refuse them nor cleared for it."""
import pytest
import torch


@pytest.fixture
def status(monkeypatch):
    from uwc_b200 import _lib
    bits = [0]

    def read(clear=True):
        st = bits[0]
        if clear:
            bits[0] = 0
        return st
    monkeypatch.setattr(_lib, "device_status", read)
    return bits


def test_winners_refuses_timeouts_alone(status):
    from uwc_b200 import _lib, ops
    w = ops.MinedWeight(Bt=torch.zeros(8, 64, dtype=torch.int8), b_scale=torch.ones(8))
    rec = w._wins_for(64)
    rec[0], rec[1], rec[2] = 1, 16, 32
    want = [(16, 32, bytes(32))]
    assert w.winners(64) == want
    status[0] = _lib.DEV_RANGE
    assert w.winners(64) == want and status[0] == _lib.DEV_RANGE
    for st in (_lib.DEV_TIMEOUT, _lib.DEV_TIMEOUT | _lib.DEV_RANGE):
        status[0] = st
        with pytest.raises(_lib.UWCError):
            w.winners(64)
        assert status[0] == 0 and w.winners(64) == want
