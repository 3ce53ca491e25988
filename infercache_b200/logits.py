"""Logits between the model and the sampler: penalties for repeated tokens,
biases and grammar masks, in one kernel (``ic_process_logits``).

The reference's sampler divides or multiplies the generated tokens' logits by
the repetition penalty in a host loop (two_pass.py:251-279); ``TwoPassEngine``
calls this instead, and a server calls it for its whole batch.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib

Scalar = Union[float, torch.Tensor, None]


def process_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None,
                   token_lens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                   repetition: Scalar = None, presence: Scalar = None, frequency: Scalar = None,
                   bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                   bias_lens: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 logits [S, V] after, in this order,

    * ``repetition`` r: an id among ``tokens[s, :token_lens[s]]`` (prompt and
      answer) has x / r where x > 0 (x * (1 / r) for a number r, as torch
      divides by a number), x * r elsewhere;
    * ``frequency`` f and ``presence`` p: x - (f * n + p) for an id that occurs
      n > 0 times in the answer, ``tokens[s, prompt_lens[s]:token_lens[s]]``;
    * ``bias_ids`` / ``bias_values`` [S, B] (the first ``bias_lens[s]`` of a row):
      x + value; of an id given twice the last value counts;
    * ``mask`` int32 [S, >= ceil(V / 32)]: -inf where bit v % 32 of word
      v // 32 is 0.

    ``logits`` [S, V] is fp32, fp16 or bf16 with contiguous rows; penalties are
    numbers or [S] tensors; missing lengths mean the whole
    row, no prompt.  Ids outside the vocabulary are skipped, so rows may be
    padded with -1.  ``out`` may be ``logits`` itself when it is float32, and does
    not overlap it otherwise.
    """
    return _lib.binding().process_logits(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency,
                                         bias_ids, bias_values, bias_lens, mask, out)
