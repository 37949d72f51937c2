"""Rules on logits before something is drawn from them: penalties for tokens that occurred, a bias, a temperature and a mask,
with their gradient.

``process_logits`` works on token logits ``[..., vocabulary]`` and, with ``dim``, on scores whose vocabulary is another
dimension, such as the model's link scores ``[B, V, V, C]`` with ``dim=2`` (the next node), which the path sampler and the beam
search take.  Formulas and conventions: ``gcn_logits_process`` in ``include/gcn_uelb_hip.h``.
"""
from __future__ import annotations

import math

import torch

from . import lib as L


def pack_mask(mask):
    """A truth value per vocabulary entry ``[..., V]`` as bits ``[..., ceil(V / 32)]`` (int32 words, the lowest bit first):
    1/8 of the memory, and of the reading."""
    if mask.dtype != torch.bool:
        raise TypeError(f"mask holds truth values, got {mask.dtype}")
    rows = torch.nn.functional.pad(mask, (0, -mask.shape[-1] % 32)).unflatten(-1, (-1, 32)).to(torch.int64)
    words = (rows << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def process_logits(logits, *, dim=-1, history=None, history_lens=None, prompt_lens=None, repetition_penalty=1.0, presence_penalty=0.0,
                   frequency_penalty=0.0, bias=None, mask=None, temperature=1.0, masked_value=-math.inf, out=None):
    """The logits after penalties, bias, temperature and mask, of the same shape and type.

    logits: float32, bfloat16 or float16 ``[*lead, V, *inner]`` with the vocabulary at ``dim``.  The other arguments hold rows
    for ``lead``, for its last few dimensions (the same for all others), or one row for all, and apply to all of ``inner``.  The
    outermost dimension of their rows may also be a divisor of the logits' own there: R rows for N = k R rows of logits,
    whose row o uses row o mod R, as link scores [graphs * V, V, C] use a bias [V, V] of the node.
      history ``[*rows, length]``, int32 or int64: entries that occurred; those outside ``[0, V)`` are skipped (padding).
        history_lens, prompt_lens ``[*rows]``: the first history_lens entries count; those before prompt_lens count for the
        repetition penalty only.  The same entry may occur any number of times.
      repetition_penalty, presence_penalty, frequency_penalty, temperature: numbers, or float32 ``[*rows]`` (repetition
        penalties and temperatures must be positive; numbers are checked).
      bias: float32 ``[*rows, V]``.
      mask: what is allowed, as truth values ``[*rows, V]`` or as bits (``pack_mask``); the rest becomes masked_value (rounded
        to the logits' type: -1e9 is -inf in float16).  A row
        whose mask leaves nothing becomes masked_value throughout: with -inf a softmax over it is NaN.
    Differentiable in logits and bias (at x = 0 with the slope below it); penalties and temperatures are constants.
    There is no forward-mode derivative: a tangent on logits, bias or out is refused.  While a stream
    is captured, logits and bias that are leaves of a graph which lives on another stream are refused: its backward pass could
    not be captured.
    out: a tensor for the result, which may be ``logits`` and must not overlap it otherwise, nor any other argument; not with gradients."""
    return L.binding().process_logits(logits, dim, history, history_lens, prompt_lens, repetition_penalty, presence_penalty, frequency_penalty, bias,
                                      mask, temperature, masked_value, out)
