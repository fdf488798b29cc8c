"""The rules of running requests on the device: every request with rules holds a slot with its text (prompt and answer; the
kernel that chooses a token appends it, so the host need not know it yet) and its biases.  ``step_rules`` draws up the rules of a
step's rows."""
from __future__ import annotations

import numpy as np
import torch

from ..kernels import ops


def mask_words(allowed, vocab: int, banned=()):
    """A grammar's answer as int32 words of one bit an entry (ops.LogitRules), less the ``banned`` entries; None: everything may follow.  Raises
    ValueError for an answer that fits no vocabulary."""
    if allowed is None:
        return None
    words = -(-vocab // 32)
    bits = np.zeros(words * 32, dtype=bool)
    given = np.asarray(allowed if isinstance(allowed, np.ndarray) else list(allowed))
    if given.dtype == bool:
        if given.shape != (vocab,):
            raise ValueError(f"a grammar's truth values are one an entry of the vocabulary ({vocab}), got {given.shape}")
        bits[:vocab] = given
    elif given.size:
        if given.ndim != 1 or not np.issubdtype(given.dtype, np.integer) or given.min() < 0 or given.max() >= vocab:
            raise ValueError(f"a grammar allows token ids in [0, {vocab}), or one truth value an entry")
        bits[given] = True
    bits[list(banned)] = False
    return np.packbits(bits, bitorder="little").view(np.int32)


class RuleBook:
    def __init__(self, device, width: int, vocab: int):
        self.device, self.width, self.vocab = torch.device(device), width, vocab
        self.history = torch.zeros(0, width, dtype=torch.int32, device=self.device)
        self.bias_tokens = torch.zeros(0, 0, dtype=torch.int32, device=self.device)
        self.bias_values = torch.zeros(0, 0, dtype=torch.float32, device=self.device)
        self._free: list = []
        self._held: dict = {}                # request id -> slot

    # ------------------------------------------------------------------ slots
    def _grow(self, slots: int, biases: int) -> None:
        """Room for that many texts and biases a text.  (Tensors of before live on until the launches that read them are done: the allocator's stream order.)"""
        old, n = self.history.shape[0], self.bias_tokens.shape[1]
        if slots > old:
            fresh = torch.zeros(slots, self.width, dtype=torch.int32, device=self.device)
            fresh[:old] = self.history
            self.history = fresh
            self._free += range(old, slots)
        if slots > old or biases > n:
            n2 = max(n, biases)
            for name in ("bias_tokens", "bias_values"):
                was = getattr(self, name)
                fresh = torch.zeros(max(slots, old), n2, dtype=was.dtype, device=self.device)
                fresh[:old, :n] = was
                setattr(self, name, fresh)

    def admit(self, seq) -> int:
        """The request's slot; at its first step, one with its text so far in it."""
        slot = self._held.get(seq.seq_id)
        if slot is not None:
            return slot
        bias = seq.params.logit_bias or {}
        if not self._free or len(bias) > self.bias_tokens.shape[1]:
            self._grow(self.history.shape[0] if self._free else max(16, 2 * self.history.shape[0]), len(bias))
        slot = self._free.pop()
        self._held[seq.seq_id] = slot
        self.history[slot, :seq.prompt_len].copy_(torch.from_numpy(seq.prompt_array))
        if bias:
            self.bias_tokens[slot, :len(bias)].copy_(torch.tensor([int(t) for t in bias], dtype=torch.int32))
            self.bias_values[slot, :len(bias)].copy_(torch.tensor([float(b) for b in bias.values()], dtype=torch.float32))
        return slot

    def release(self, seq) -> None:
        slot = self._held.pop(seq.seq_id, None)
        if slot is not None:
            self._free.append(slot)          # (a step in flight may still append to it: the next text is written behind that step)

    # ------------------------------------------------------------------ a step
    def step_rules(self, seqs) -> ops.LogitRules:
        """The rules of rows that sample for ``seqs``, one row each, in this order; a request's tokens include those that a step in flight
        is still choosing (they are on the device when this step's kernel runs)."""
        k = len(seqs)
        ints = np.zeros((5, k), dtype=np.int32)              # slot, prompt_len, total_len, bias_len, mask_row
        reals = np.zeros((3, k), dtype=np.float32)           # repetition, presence, frequency
        reals[0] = 1.0
        ints[0] = ints[4] = -1
        masks = []
        for i, s in enumerate(seqs):
            p = s.params
            if not s.has_rules:
                continue
            ints[:4, i] = self.admit(s), s.prompt_len, len(s.token_ids), len(p.logit_bias or ())
            reals[:, i] = p.repetition_penalty, p.presence_penalty, p.frequency_penalty
            if s.mask is not None:
                ints[4, i] = len(masks)
                masks.append(s.mask)
        packed = torch.from_numpy(np.concatenate([ints, reals.view(np.int32)])).to(self.device)
        mask = torch.from_numpy(np.stack(masks)).to(self.device) if masks else None
        f = packed.view(torch.float32)
        some = self.history.shape[0] > 0
        biases = some and self.bias_tokens.shape[1] > 0
        return ops.LogitRules(self.history if some else None, packed[0], packed[1], packed[2], repetition=f[5] if some else None,
                              presence=f[6] if some else None, frequency=f[7] if some else None, bias_tokens=self.bias_tokens if biases else None,
                              bias_values=self.bias_values if biases else None, bias_len=packed[3] if biases else None,
                              mask=mask, mask_row=packed[4] if mask is not None else None)
