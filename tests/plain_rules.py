"""Rules on logits in 64 bits, one row and one token at a time where that matters: the oracle of the rules' tests."""
import math

import torch

INF = float("inf")


def ruled(x, text=(), prompt_len=0, repetition=1.0, presence=0.0, frequency=0.0, biases=(), mask=None):
    """The row ``x`` under its rules in float64, and a bound on the error of the same in float32 (a rounding is off by half a step,
    2^-24 of the value: two for a penalty's product and sum, one for each step on the logit itself)."""
    x = x.double().clone()
    V = x.numel()
    size = x.abs()
    steps = torch.zeros_like(x)
    for t in {t for t in text if 0 <= t < V}:
        x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
        size[t] = torch.maximum(size[t], x[t].abs())
        steps[t] += 1
    answer = [t for t in text[prompt_len:] if 0 <= t < V]
    for t in set(answer):
        loss = frequency * answer.count(t) + presence
        x[t] -= loss
        size[t] += abs(frequency) * answer.count(t) + abs(presence)
        steps[t] += 3
    for t, b in biases:
        if 0 <= t < V:
            x[t] += b
            if math.isfinite(b):
                size[t] += abs(b)
            steps[t] += 1
    if mask is not None:
        for i in range(V):
            if not (mask[i // 32] >> (i % 32)) & 1:
                x[i] = -INF
    return x, size * steps * 2.0 ** -24


def logprob_bound(x):
    """A bound on the error of log softmax in float32 over the row ``x``: the exponential is off by 2 + 1.173 |argument| steps of 2^-23 (the
    documented bound of the fast one), once for a term and once for all the times that the maximum moved on; a term passes some hundred sums of half a step
    (a thread's own, the warp's, the block's and the cluster's); and the last logarithm, sum and difference."""
    kept = x[torch.isfinite(x)]
    reach = min(float(kept.max() - kept.min()), 104.0) if kept.numel() else 0.0
    most = float(kept.abs().max()) if kept.numel() else 0.0
    return 2.0 ** -23 * (2 * 1.173 * reach + 2 * 24 + 64 + 4 * (most + 16))
