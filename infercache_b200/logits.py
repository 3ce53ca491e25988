"""Logits between the model and the sampler: penalties for repeated tokens,
biases and grammar masks, in one kernel (``ic_process_logits``).

The reference's sampler divides or multiplies the generated tokens' logits by
the repetition penalty in a host loop (two_pass.py:251-279); ``TwoPassEngine``
calls this instead, and a server calls it for its whole batch.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _lib
from .paged_ops import _device_of, _on

Scalar = Union[float, torch.Tensor, None]


def _per_row(name: str, x: Scalar, default: float, rows: int, dev: torch.device):
    """(tensor or None, number): the kernel takes the number where there is no tensor."""
    if x is None:
        return None, default
    if not isinstance(x, torch.Tensor):
        return None, float(x)
    if x.shape != (rows,) or x.device != dev:
        raise ValueError(f"process_logits: {name} must be a number or a [{rows}] tensor on {dev}")
    return x.to(torch.float32).contiguous(), default


def _ints(name: str, x: Optional[torch.Tensor], shape, dev: torch.device) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if x.dtype not in (torch.int32, torch.int64) or x.dim() != len(shape) or x.device != dev or \
            any(w is not None and n != w for n, w in zip(x.shape, shape)):
        raise ValueError(f"process_logits: {name} must be an int32 or int64 tensor of shape "
                         f"{tuple('any' if w is None else w for w in shape)} on {dev}, got {x.dtype} {tuple(x.shape)}")
    return x.to(torch.int32).contiguous()


def process_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None,
                   token_lens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                   repetition: Scalar = None, presence: Scalar = None, frequency: Scalar = None,
                   bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                   bias_lens: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 logits [S, V] after, in this order,

    * ``repetition`` r: an id among ``tokens[s, :token_lens[s]]`` (prompt and
      answer) has x * (1 / r) where x > 0, x * r elsewhere;
    * ``frequency`` f and ``presence`` p: x - (f * n + p) for an id that occurs
      n > 0 times in the answer, ``tokens[s, prompt_lens[s]:token_lens[s]]``;
    * ``bias_ids`` / ``bias_values`` [S, B] (the first ``bias_lens[s]`` of a row):
      x + value; of an id given twice the last value counts;
    * ``mask`` int32 [S, >= ceil(V / 32)]: -inf where bit v % 32 of word
      v // 32 is 0.

    ``logits`` [S, V] is fp32, fp16 or bf16 with contiguous rows; penalties are
    numbers or [S] tensors; missing lengths mean the whole
    row, no prompt.  Ids outside the vocabulary are skipped, so rows may be
    padded with -1.  ``out`` may be ``logits`` itself when it is float32.
    """
    dev = _device_of("process_logits", logits)
    if logits.dim() != 2:
        raise ValueError(f"process_logits: logits must be [S, V], got {tuple(logits.shape)}")
    S, V = logits.shape
    dt = _lib.dtype_code(logits.dtype)
    if logits.stride(1) != 1 or (S > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    if out is None:
        out = torch.empty((S, V), dtype=torch.float32, device=dev)
    elif out.dtype != torch.float32 or out.shape != (S, V) or out.device != dev or out.stride(1) != 1 or \
            (S > 1 and out.stride(0) < V):
        raise ValueError(f"process_logits: out must be a float32 [{S}, {V}] tensor with contiguous rows on {dev}")
    if tokens is None and (token_lens is not None or prompt_lens is not None):
        raise ValueError("process_logits: token_lens and prompt_lens need tokens")
    if tokens is None and not (repetition is None and presence is None and frequency is None):
        raise ValueError("process_logits: penalties need tokens")
    if (bias_ids is None) != (bias_values is None) or (bias_lens is not None and bias_ids is None):
        raise ValueError("process_logits: bias_ids and bias_values come together")
    tok, tl, pl = _ints("tokens", tokens, (S, None), dev), _ints("token_lens", token_lens, (S,), dev), \
        _ints("prompt_lens", prompt_lens, (S,), dev)
    rep, rep_all = _per_row("repetition", repetition, 1.0, S, dev)
    pres, pres_all = _per_row("presence", presence, 0.0, S, dev)
    freq, freq_all = _per_row("frequency", frequency, 0.0, S, dev)
    ids, bl = _ints("bias_ids", bias_ids, (S, None), dev), _ints("bias_lens", bias_lens, (S,), dev)
    vals = None
    if ids is not None:
        if bias_values.shape != ids.shape or bias_values.device != dev:
            raise ValueError(f"process_logits: bias_values must be {tuple(ids.shape)} on {dev}")
        vals = bias_values.to(torch.float32).contiguous()
    if mask is not None:
        if mask.dtype != torch.int32 or mask.dim() != 2 or mask.shape[0] != S or mask.shape[1] < (V + 31) // 32 or \
                mask.device != dev:
            raise ValueError(f"process_logits: mask must be int32 [{S}, >= {(V + 31) // 32}] on {dev}")
        mask = mask.contiguous()
    if S == 0 or V == 0:
        return out
    p = _lib.ptr
    T, B = tok.shape[1] if tok is not None else 0, ids.shape[1] if ids is not None else 0
    a = _lib.ic_logits_args(logits.data_ptr(), out.data_ptr(), max(logits.stride(0), V), max(out.stride(0), V),
                            p(tok) if T else 0, p(tl), p(pl), p(rep), p(pres), p(freq), p(ids) if B else 0, p(vals), p(bl),
                            p(mask), T, B, mask.shape[1] if mask is not None else 0, S, V, dt, T, B, rep_all,
                            1.0 / rep_all if rep_all else math.inf, pres_all, freq_all, 0)
    _on(dev, "ic_process_logits", a)
    return out
