"""Rules on logits before a token is chosen: penalties for repeated tokens, biases, grammar masks.

``process_logits`` writes the processed logits (for a sampler); ``choose_tokens`` reduces them to the
greedy token in the same pass and writes no logits.  Both take everything from the device, so a
captured decode step replays with the histories, masks and penalties of that step.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..ops._ext import require


@dataclass
class TokenHistory:
    """Token ids of every row so far: ``ids`` ``[B, capacity]`` int32, of which the first ``lengths[b]``
    are valid (none where it is negative) and the first ``prompt_lengths[b]`` (``None``: none) are the
    prompt's; the capacity stays under 2^20."""

    ids: torch.Tensor
    lengths: torch.Tensor
    prompt_lengths: torch.Tensor | None = None

    @classmethod
    def start(cls, prompts: torch.Tensor, lengths: torch.Tensor, new_tokens: int,
              prefix: torch.Tensor | None = None) -> "TokenHistory":
        """History of left-aligned ``prompts`` ``[B, T]`` with room for ``new_tokens`` more; ``prefix`` ``[P]``: a
        prompt that every row has in front of its own."""
        P = 0 if prefix is None else prefix.shape[0]
        n = lengths.to(prompts.device, torch.int32).contiguous() + P
        ids = torch.zeros((prompts.shape[0], P + prompts.shape[1] + new_tokens), dtype=torch.int32, device=prompts.device)
        if P:
            ids[:, :P] = prefix.to(prompts.device)
        ids[:, P: P + prompts.shape[1]] = prompts
        return cls(ids, n.clone(), n)

    def append(self, tokens: torch.Tensor) -> None:
        """Add ``tokens`` ``[B]`` (negative: none); a full row keeps what it has.  No host read."""
        if self.ids.shape[1] == 0:
            return
        place = self.lengths.long().clamp(min=0)
        room = (place < self.ids.shape[1]) & (tokens >= 0)
        at = place.clamp(max=self.ids.shape[1] - 1)[:, None]
        kept = torch.where(room[:, None], tokens[:, None].to(torch.int32), self.ids.gather(1, at))
        self.ids.scatter_(1, at, kept)
        self.lengths.copy_(torch.where(room, (place + 1).to(torch.int32), self.lengths))


@dataclass
class LogitsRules:
    """What is done to each row's logits, in this order (each step rounded to fp32):

    * ``repetition`` ``[B]``: a token of the history has its logit divided by it (positive logits) or
      multiplied by it (others);
    * ``frequency`` / ``presence`` ``[B]``: subtracted per occurrence in the output / once if there is one;
    * ``bias_ids`` / ``bias_values`` ``[B, n]``: added to single tokens (a token listed twice gets the
      sum; ids outside the vocabulary, as -1, are skipped; at most 2047 entries);
    * ``mask`` ``[M, >= ceil(V / 32)]`` int32, bit ``t % 32`` of word ``t // 32`` set where token ``t`` is
      allowed, the others become -inf; ``mask_rows`` ``[B]`` int32 names each row's mask (negative: no
      mask; ``M`` or more: nothing is allowed), by default mask ``b`` for row ``b``.

    Penalties are fp32, absent ones are left out.  A history or biases take up to 393,216 columns,
    a call up to 65,535 rows.
    """

    repetition: torch.Tensor | None = None
    presence: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None
    bias_values: torch.Tensor | None = None
    mask: torch.Tensor | None = None
    mask_rows: torch.Tensor | None = None


def process_logits(logits: torch.Tensor, rules: LogitsRules, history: TokenHistory | None = None, *,
                   out: torch.Tensor | None = None, vocab_start: int = 0) -> torch.Tensor:
    """``logits`` ``[B, V]`` (bf16, fp16 or fp32, rows may be strided) after the rules, in a new tensor or
    in ``out`` (which may be ``logits``).  ``vocab_start``: the token id of column 0 when the columns are
    a slice of the vocabulary (a multiple of 8).  No gradients."""
    h = history
    return require().process_logits(logits, out, h.ids if h else None, h.lengths if h else None,
                                    h.prompt_lengths if h else None, rules.repetition, rules.presence, rules.frequency,
                                    rules.bias_ids, rules.bias_values, rules.mask, rules.mask_rows, vocab_start)


def join_choices(values: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    """Tokens ``[B]`` int64 over the whole vocabulary from the choices of its slices (``choose_tokens``): processed
    logits ``values`` and ids ``tokens`` ``[B, slices]``.  As within a slice: NaN is the largest, ties go to the
    lowest id, -1 where no slice has anything."""
    nan = values.isnan()
    score = values.masked_fill(nan.any(1, keepdim=True), float("-inf")).masked_fill(nan, 0.0)
    worse = score < score.amax(1, keepdim=True)
    return tokens.double().masked_fill(worse, float("inf")).amin(1).long()


def choose_tokens(logits: torch.Tensor, rules: LogitsRules, history: TokenHistory | None = None, *,
                  vocab_start: int = 0, append: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Greedy token of each row after the rules: ``(ids [B] int64, their processed logits [B] fp32)``.
    Ties go to the lowest id; a row with nothing above -inf gives id -1 and -inf; NaN counts as the
    largest.  ``append`` adds the chosen tokens to ``history`` in the same launch."""
    h = history
    if append and h is None:
        raise ValueError("append needs a history")
    return require().choose_tokens(logits, h.ids if h else None, h.lengths if h else None,
                                   h.prompt_lengths if h else None, rules.repetition, rules.presence, rules.frequency,
                                   rules.bias_ids, rules.bias_values, rules.mask, rules.mask_rows, vocab_start, append)
