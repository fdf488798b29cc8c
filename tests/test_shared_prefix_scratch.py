"""Scratch memory of attention over shared prefixes that has to start cleared: who makes it, and when others may rely on it.  On the host, with what a device would do left out."""
import pytest
import torch

from mini_inference_engine_b200.kernels import ops

SIZES = (0, 40, 3, 32, 4, 64, 16, 2048, 128, 500)


class Layout:
    def mie_prefix_layout(self, ref, sms):
        ref._obj.walk, ref._obj.most_slots = 1, 1000
        return 0


class Calls:
    def __init__(self):
        self.capturing, self.synchronised = False, 0

    def synchronize(self):
        self.synchronised += 1


@pytest.fixture()
def calls(monkeypatch):
    c = Calls()
    zeros, empty = torch.zeros, torch.empty
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k))
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: c.capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda where=None: c)
    monkeypatch.setattr(ops, "_shared_libs", lambda: (Layout(), None, None))
    monkeypatch.setattr(ops, "num_sms", lambda where=None: 148)
    monkeypatch.setattr(ops, "PREFIX_ONE_BY_ONE_BYTES", (-1, -1))
    monkeypatch.setattr(ops, "_workspaces", {})
    ops._shared_plan.cache_clear()
    yield c
    ops._shared_plan.cache_clear()


def names():
    return {name for _, name in ops._workspaces}


def test_what_one_stream_cleared_others_may_use(calls):
    ops._shared_plan(*SIZES, 77)
    assert {"prefix_marks", "prefix_marks@77"} <= names() and calls.synchronised == 1
    ops._shared_plan(*SIZES, 0)
    assert calls.synchronised == 1                            # (cleared long ago)
    ops._shared_plan(*SIZES[:1], 4000, *SIZES[2:], 0)         # larger: made anew
    assert calls.synchronised == 2


def test_a_launch_captured_first_leaves_nothing_to_others(calls):
    calls.capturing = True
    with pytest.raises(ops._NoScratch):
        ops._shared_plan(*SIZES, 0)
    own = ops._shared_plan.__wrapped__(*SIZES, -1)[2]
    assert "prefix_marks" not in names() and int(own[-1].abs().max()) == 0 and calls.synchronised == 0
    mine = {t.data_ptr() for t in own}
    calls.capturing = False
    kept = ops._shared_plan(*SIZES, 0)[2]
    assert not mine & {t.data_ptr() for t in kept} and calls.synchronised == 1
    calls.capturing = True                                    # from now on captured launches use what is there
    assert ops._shared_plan(*SIZES, 0)[2] is kept
