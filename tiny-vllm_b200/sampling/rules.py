"""Rules that stand between a request's logits and its next token, kept on the device slot by slot.

A request that has rules (``SamplingParams.has_rules``: penalties for tokens it has seen, biases, allowed tokens) holds a
slot.  What a step then needs is the slots of its rows: the counts are made in the kernel from the tokens that the slot
keeps, and the sampled tokens join them there, without a word to the host.  The reference has no such rules.
"""

from __future__ import annotations

from typing import Sequence

import torch

from ..ops import kernels
from .params import SamplingParams


class LogitRules:
    """The rules of up to ``slots`` requests over a vocabulary of ``vocab`` tokens; ``room``: the most tokens a request
    has in all (later ones are not remembered).

    Room for biases and masks is made when a request brings some (``biases`` of a slot, and masks with ``masks``, at once).  A step that is
    recorded into a graph keeps the room it had: from then on a request that needs more is refused."""

    def __init__(self, *, vocab: int, slots: int, room: int, device, biases: int = 0, masks: bool = False) -> None:
        if vocab < 1 or slots < 1 or room < 1:
            raise ValueError("rules need a vocabulary, slots and room for tokens")
        self.vocab, self.slots, self.room, self.device = vocab, slots, room, torch.device(device)
        self.penalties = torch.tensor([[1.0, 0.0, 0.0]] * slots, dtype=torch.float32, device=device)
        self.lengths = torch.zeros((slots, 2), dtype=torch.int32, device=device)
        self.history = torch.zeros((slots, room), dtype=torch.int32, device=device)
        if not 0 <= biases <= kernels.LOGIT_RULES_MAX_BIASES:
            raise ValueError(f"a slot holds up to {kernels.LOGIT_RULES_MAX_BIASES} biases")
        self.bias_tokens = self.bias_values = self.masks = self.mask_rows = None
        self._recorded = False
        if biases:
            self._make_biases(biases)
        if masks:
            self._make_masks()

    def _make_biases(self, width: int) -> None:
        """Rows of ``width`` biases, with what is held already; -1: no bias."""
        tokens = torch.full((self.slots, width), -1, dtype=torch.int32, device=self.device)
        values = torch.zeros((self.slots, width), dtype=torch.float32, device=self.device)
        if self.bias_tokens is not None:
            held = self.bias_tokens.shape[1]
            tokens[:, :held], values[:, :held] = self.bias_tokens, self.bias_values
        self.bias_tokens, self.bias_values = tokens, values

    def _make_masks(self) -> None:
        self.masks = torch.zeros((self.slots, -(-self.vocab // 32)), dtype=torch.int32, device=self.device)
        self.mask_rows = torch.full((self.slots,), -1, dtype=torch.int32, device=self.device)

    def check(self, params: SamplingParams) -> None:
        """Refuse rules that name tokens outside the vocabulary."""
        named = [token for token, _ in params.logit_bias] + list(params.allowed_token_ids or ())
        for token in named:
            if token >= self.vocab:
                raise ValueError(f"a rule names token {token}, the vocabulary has {self.vocab}")

    @torch.inference_mode()
    def set(self, slot: int, params: SamplingParams, prompt: Sequence[int], answer: Sequence[int] = ()) -> None:
        """The slot's request from now on: its rules and the tokens it has so far."""
        if type(slot) is not int or not 0 <= slot < self.slots:
            raise ValueError(f"{slot!r} is not one of the {self.slots} slots")
        self.check(params)
        most = len(params.logit_bias)
        held = 0 if self.bias_tokens is None else self.bias_tokens.shape[1]
        if self._recorded and (most > held or params.allowed_token_ids is not None and self.masks is None):
            raise ValueError(f"the rules are part of a recorded step with room for {held} biases a slot and "
                             f"{'no masks' if self.masks is None else 'masks'}; make them with biases= and masks= for more")
        tokens = torch.tensor((*prompt, *answer)[:self.room], dtype=torch.int32)
        self.history[slot, :tokens.shape[0]] = tokens.to(self.device)
        self.lengths[slot] = torch.tensor([tokens.shape[0], min(len(prompt), self.room)], dtype=torch.int32).to(self.device)
        self.penalties[slot] = torch.tensor([params.repetition_penalty, params.presence_penalty, params.frequency_penalty],
                                            dtype=torch.float32).to(self.device)
        if most > held:                                  # wider rows, by doubling
            self._make_biases(min(max(most, 2 * held, 32), kernels.LOGIT_RULES_MAX_BIASES))
        if self.bias_tokens is not None:
            self.bias_tokens[slot] = -1
            if most:
                self.bias_tokens[slot, :most] = torch.tensor([t for t, _ in params.logit_bias], dtype=torch.int32).to(self.device)
                self.bias_values[slot, :most] = torch.tensor([b for _, b in params.logit_bias], dtype=torch.float32).to(self.device)
        if params.allowed_token_ids is not None:
            if self.masks is None:
                self._make_masks()
            self.masks[slot] = pack_mask(params.allowed_token_ids, self.vocab).to(self.device)
        if self.mask_rows is not None:
            self.mask_rows[slot] = slot if params.allowed_token_ids is not None else -1

    def apply(self, logits: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """The rows' logits under the rules of ``slots`` (int32 on the device, a row each; -1: a row without rules)."""
        if logits.dim() != 2 or logits.shape[1] != self.vocab:
            raise ValueError(f"the rules are those of {self.vocab} tokens")
        result = kernels.logit_rules(logits, slots=slots, penalties=self.penalties, lengths=self.lengths, history=self.history,
                                     bias_tokens=self.bias_tokens, bias_values=self.bias_values, masks=self.masks,
                                     mask_rows=self.mask_rows, out=out)
        self._recorded = self._recorded or torch.cuda.is_current_stream_capturing()       # (the graph has these tensors' addresses)
        return result

    def append(self, tokens: torch.Tensor, slots: torch.Tensor) -> None:
        """The rows' next tokens (int32 on the device) join what their slots remember."""
        kernels.append_tokens(tokens, slots=slots, lengths=self.lengths, history=self.history)


def pack_mask(allowed: Sequence[int], vocab: int) -> torch.Tensor:
    """int32 words of a mask over ``vocab`` tokens: bit v % 32 of word v // 32 is token v."""
    bits = torch.zeros(-(-vocab // 32) * 32, dtype=torch.int64)
    bits[torch.tensor(list(allowed), dtype=torch.int64)] = 1
    words = (bits.view(-1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)
