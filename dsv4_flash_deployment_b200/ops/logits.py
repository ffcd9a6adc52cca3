"""Rules on logits before sampling: penalties for repeated tokens, per-token biases
and grammar masks (``csrc/logits.cu``), and the token history the penalties read.

    z = l / rho if l > 0 else l * rho      tokens of the prompt or the output
    z -= frequency * count + presence      tokens of the output
    z += bias                              -inf bans the token
    z = -inf                               tokens the row's mask does not allow

in fp32, rounded once to the logits' type.  CPU tensors run the torch oracle math;
CUDA tensors always run the extension, on the current stream of their device.
"""

from __future__ import annotations

import torch

from ..ref import numerics as N
from . import _ext
from .gemm import ErrorWord


class TokenHistory:
    """Which tokens each sequence slot has seen: ``seen`` int32 [n_slots, ceil(V / 32)]
    (a bit per token of the prompt or the output) and ``counts`` int32 [n_slots, V]
    (occurrences in the output).  129280 entries take 533 KB a slot."""

    __slots__ = ("seen", "counts")

    def __init__(self, seen: torch.Tensor, counts: torch.Tensor):
        self.seen, self.counts = seen, counts

    @classmethod
    def empty(cls, n_slots: int, vocab: int, device) -> "TokenHistory":
        return cls(torch.zeros(n_slots, (vocab + 31) // 32, dtype=torch.int32, device=device),
                   torch.zeros(n_slots, vocab, dtype=torch.int32, device=device))

    def reset(self, slot: int) -> None:
        if not 0 <= slot < len(self.counts):
            raise IndexError(f"slot {slot} of {len(self.counts)}")
        self.seen[slot].zero_()
        self.counts[slot].zero_()

    def add(self, ids: torch.Tensor, slots: torch.Tensor, generated: torch.Tensor) -> None:
        """Adds tokens ``ids`` [n] of slots ``slots`` [n] (int32): ``generated`` int32 [n]
        > 0 counts the token as output, 0 marks it as the prompt's, < 0 (or a negative
        slot) skips it.  A token or slot outside the tables is left out and reported
        in the device error word."""
        if self.counts.is_cuda:
            _ext.load().history_add(ids, slots, generated, self.seen, self.counts, ErrorWord.get(ids.device))
            return
        n_slots, v = self.counts.shape
        for i, s, g in zip(ids.tolist(), slots.tolist(), generated.tolist()):
            if g < 0 or s < 0:
                continue
            if s >= n_slots or not 0 <= i < v:
                raise RuntimeError(f"token {i} of slot {s}: outside the history")
            bit = 1 << (i & 31)
            self.seen[s, i >> 5] |= bit - (1 << 32) if bit >> 31 else bit
            self.counts[s, i] += int(g > 0)


class RowRules:
    """The rules of a batch's rows, as device tensors.  Each kind is set on its own;
    a kind that is not set does nothing."""

    __slots__ = ("slots", "repetition", "frequency", "presence", "bias_off", "bias_ids", "bias_vals", "mask_rows",
                 "mask")

    def __init__(self):
        self.slots = self.repetition = self.frequency = self.presence = None
        self.bias_off = self.bias_ids = self.bias_vals = None
        self.mask_rows = self.mask = None

    def penalties(self, slots: torch.Tensor, repetition: torch.Tensor, frequency: torch.Tensor,
                  presence: torch.Tensor) -> "RowRules":
        """Row s reads the history of ``slots[s]`` (int32; negative: no penalties for this
        row); ``repetition`` > 0 (1: off), ``frequency``, ``presence`` (0: off), fp32 [S]."""
        self.slots, self.repetition, self.frequency, self.presence = slots, repetition, frequency, presence
        return self

    def biases(self, offsets: torch.Tensor, ids: torch.Tensor, values: torch.Tensor) -> "RowRules":
        """Row s adds ``values[i]`` (fp32, finite or -inf) to token ``ids[i]`` for i in
        ``offsets[s] .. offsets[s + 1]`` (int32 [S + 1]).  The ids of a row ascend (a
        token given twice: its values add up); entries out of order are not found."""
        self.bias_off, self.bias_ids, self.bias_vals = offsets, ids, values
        return self

    def masks(self, rows: torch.Tensor, words: torch.Tensor) -> "RowRules":
        """Row s keeps the tokens whose bit is set in ``words[rows[s]]`` (int32 [S];
        negative: no mask).  Words int32 [n, >= ceil(V / 32)], bit j of word i = token
        32 i + j."""
        self.mask_rows, self.mask = rows, words
        return self


def apply_logits_rules(logits: torch.Tensor, rules: RowRules, history: TokenHistory | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Applies ``rules`` to ``logits`` [S, V] (bf16, fp16 or fp32, contiguous rows, up to
    65535 of them) into ``out`` (None: in place; else it may not overlap the logits) and
    returns it.  ``history`` is needed with penalties.  A slot or mask row outside its
    table leaves the row without that rule and is reported in the device error word."""
    r = rules
    if r.slots is not None and history is None:
        raise ValueError("penalties need a token history")
    if out is None:
        out = logits
    if logits.is_cuda:
        seen, counts = (history.seen, history.counts) if r.slots is not None else (None, None)
        _ext.load().logits_rules(logits, out, r.slots, r.repetition, r.frequency, r.presence, seen, counts, r.bias_off,
                                 r.bias_ids, r.bias_vals, r.mask_rows, r.mask, ErrorWord.get(logits.device))
        return out
    s, v = logits.shape
    kw = {}
    if r.slots is not None:
        if history.counts.shape[1] != v:
            raise RuntimeError(f"history of {history.counts.shape[1]} tokens, logits of {v}")
        if s and int(r.slots.max()) >= history.counts.shape[0]:
            raise RuntimeError("a slot outside the history")
        use = (r.slots >= 0)[:, None]
        at = r.slots.clamp_min(0).long()
        kw = dict(seen=N.unpack_bits(history.seen[at], v) & use, counts=history.counts[at] * use,
                  repetition=r.repetition, frequency=r.frequency, presence=r.presence)
    if r.bias_off is not None:
        rows = torch.repeat_interleave(torch.arange(s), (r.bias_off[1:] - r.bias_off[:-1]).long())
        b = slice(int(r.bias_off[0]), int(r.bias_off[-1]))
        kw["bias"] = torch.zeros(s, v).index_put((rows, r.bias_ids[b].long()), r.bias_vals[b], accumulate=True)
    if r.mask is not None:
        if r.mask.shape[1] < (v + 31) // 32:
            raise RuntimeError(f"mask: int32 words [n, >= {(v + 31) // 32}] expected")
        if s and int(r.mask_rows.max()) >= r.mask.shape[0]:
            raise RuntimeError("a mask row outside the masks")
        allowed = N.unpack_bits(r.mask, v) if len(r.mask) else torch.ones(1, v, dtype=torch.bool)
        kw["allowed"] = allowed[r.mask_rows.clamp_min(0).long()] | (r.mask_rows < 0)[:, None]
    return out.copy_(N.logits_rules(logits, **kw))
