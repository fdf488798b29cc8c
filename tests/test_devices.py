"""Tensors of another device than the current one are refused before anything is launched: a kernel that followed their addresses would fault.  Host tensors that say they are on a
device stand for those."""
import pytest
import torch

from mini_inference_engine_b200.kernels import ops


class On(torch.Tensor):
    """A host tensor that claims to be on CUDA device ``where``."""
    where = 0

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return self.where


def on(t, where):
    t = t.as_subclass(On)
    t.where = where
    return t


@pytest.fixture(autouse=True)
def current(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream", lambda: pytest.fail("asked for a stream"))
    for name in ("_shared_libs", "_rules_lib", "_shared_plan"):
        monkeypatch.setattr(ops, name, lambda *a: pytest.fail("went to the kernels"))


SHARED = ("q", "k_cache", "v_cache", "block_tables", "row_q_start", "row_q_len", "row_ctx_len", "group_start", "group_prefix", "out")


@pytest.mark.parametrize("stray", SHARED)
def test_shared_prefixes(stray):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    t = dict(q=torch.zeros(2, 64, dtype=torch.bfloat16), k_cache=torch.zeros(3, 1, 16, 16, dtype=torch.bfloat16), v_cache=torch.zeros(3, 1, 16, 16, dtype=torch.bfloat16),
             block_tables=i(2, 2), row_q_start=i(2), row_q_len=i(2), row_ctx_len=i(2), group_start=i(2), group_prefix=i(1), out=torch.zeros(2, 2, 16, dtype=torch.bfloat16))
    t = {k: on(v, int(k == stray)) for k, v in t.items()}
    with pytest.raises(ops.KernelError, match="current device"):
        ops.shared_prefix_attention(t["q"], 64, *(t[k] for k in SHARED[1:]), 2, 1, 16, 16, 0.25)


@pytest.mark.parametrize("stray", ["logits", "temperature", "request", "position", "out", "logprob"])
def test_log_probabilities(stray):
    t = dict(logits=torch.zeros(2, 9), temperature=torch.zeros(2), request=torch.zeros(2, dtype=torch.int64), position=torch.zeros(2, dtype=torch.int32),
             out=torch.zeros(2, dtype=torch.int32), logprob=torch.zeros(2))
    t = {k: on(v, int(k == stray)) for k, v in t.items()}
    with pytest.raises(ops.KernelError, match="current device"):
        ops.sample(t["logits"], t["temperature"], t["request"], t["position"], 0, t["out"], logprob=t["logprob"])


def test_host_tensors():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError, match="CUDA tensors only"):
        ops.shared_prefix_attention(bf(2, 64), 64, bf(3, 1, 16, 16), bf(3, 1, 16, 16), i(2, 2), i(2), i(2), i(2), i(2), i(1), bf(2, 2, 16), 2, 1, 16, 16, 0.25)
