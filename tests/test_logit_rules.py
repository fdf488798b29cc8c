"""What the rules on logits refuse: checked before anything reaches the device."""
import pytest
import torch

from mini_inference_engine_b200.kernels import ops


def i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def f(*shape):
    return torch.zeros(*shape)


TEXT = dict(history=i(4, 9), slot=i(2), prompt_len=i(2), total_len=i(2))


@pytest.mark.parametrize("given,match", [
    (dict(), "one entry a row"),
    (dict(TEXT, slot=i(3)), "one entry a row"),
    (dict(TEXT, repetition=f(3)), "one entry a row"),
    (dict(TEXT, repetition=f(2).double()), "float32"),
    (dict(TEXT, history=i(4, 9).long()), "int32"),
    (dict(TEXT, history=i(9, 4).t()), "contiguous"),
    (dict(TEXT, history=i(36)), "history"),
    (dict(history=i(4, 9), slot=i(2)), "history"),
    (dict(slot=i(2), presence=f(2)), "penalties need a history"),
    (dict(TEXT, bias_tokens=i(4, 3)), "biases"),
    (dict(TEXT, bias_tokens=i(4, 3), bias_values=f(4, 2)), "biases"),
    (dict(TEXT, bias_tokens=i(5, 3), bias_values=f(5, 3)), "same slots"),
    (dict(TEXT, bias_len=i(2)), "without biases"),
    (dict(TEXT, mask=i(1, 2)), "mask_row"),
    (dict(TEXT, mask=i(2), mask_row=i(2)), "mask"),
    (dict(TEXT, mask=i(1, 2).to("meta"), mask_row=i(2)), "one device"),
    (dict(TEXT), "CUDA tensors only"),
])
def test_rules_that_do_not_fit_are_refused(given, match):
    with pytest.raises(ops.KernelError, match=match):
        ops.LogitRules(**given)


def test_choosing_on_the_host_is_refused():
    args = (f(2, 8), f(2), torch.zeros(2, dtype=torch.int64), i(2), 0, i(2))
    with pytest.raises(ops.KernelError, match="append goes with rules"):
        ops.sample(*args, append=True)
    with pytest.raises(ops.KernelError, match="append goes with rules"):
        ops.sample(*args, logprob=f(2), append=True)
    with pytest.raises(ops.KernelError, match="logprob"):
        ops.sample(*args, logprob=f(1))
    with pytest.raises(ops.KernelError, match="CUDA tensors only"):
        ops.sample(*args, logprob=f(2))
