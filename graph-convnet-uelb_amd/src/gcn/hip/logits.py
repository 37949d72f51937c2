"""Rules on logits before something is drawn from them: penalties for tokens that occurred, a bias, a temperature and a mask,
with their gradient.

``process_logits`` works on token logits ``[..., vocabulary]`` and, with ``dim``, on scores whose vocabulary is another
dimension, such as the model's link scores ``[B, V, V, C]`` with ``dim=2`` (the next node), which the path sampler and the beam
search take.  Formulas and conventions: ``gcn_logits_process`` in ``include/gcn_uelb_hip.h``.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import lib as L

_TYPE_ID = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INTS = (torch.int32, torch.int64)


def pack_mask(mask):
    """A truth value per vocabulary entry ``[..., V]`` as bits ``[..., ceil(V / 32)]`` (int32 words, the lowest bit first):
    1/8 of the memory, and of the reading."""
    if mask.dtype != torch.bool:
        raise TypeError(f"mask holds truth values, got {mask.dtype}")
    rows = torch.nn.functional.pad(mask, (0, -mask.shape[-1] % 32)).unflatten(-1, (-1, 32)).to(torch.int64)
    words = (rows << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _rows_of(name, shape, lead):
    """Number of rows of an argument whose leading dimensions are `shape`: all of the logits' leading dimensions, the last few of
    them (the same for all others), or ones."""
    shape = tuple(shape)
    n = math.prod(shape)
    if n == 1:
        return 1
    while shape and shape[0] == 1 and len(shape) > len(lead):
        shape = shape[1:]
    if len(shape) > len(lead) or shape != tuple(lead)[len(lead) - len(shape):]:
        raise ValueError(f"{name}: leading dimensions {shape} do not match the logits' {tuple(lead)} from the last one on")
    return n


def _row_stride(t, dim):
    """The distance between consecutive rows of t[lead..., dim, ...] in elements, None if rows are not dense or not evenly
    spaced."""
    want = 1
    for k in range(t.dim() - 1, dim - 1, -1):
        if t.shape[k] != 1 and t.stride(k) != want:
            return None
        want *= t.shape[k]
    stride, reach = None, None
    for k in range(dim - 1, -1, -1):
        if t.shape[k] == 1:
            continue
        if stride is None:
            stride = t.stride(k)
        elif t.stride(k) != reach:
            return None
        reach = t.stride(k) * t.shape[k]
    return want if stride is None else stride


class _Rules:
    """The checked arguments of a call, and the descriptor that the library takes."""

    def __init__(self, logits, dim, history, history_lens, prompt_lens, penalties, bias, mask, masked_value):
        if not isinstance(logits, torch.Tensor) or logits.dtype not in _TYPE_ID:
            raise TypeError(f"logits are float32, bfloat16 or float16, got {getattr(logits, 'dtype', type(logits))}")
        if logits.dim() == 0 or not -logits.dim() <= dim < logits.dim():
            raise ValueError(f"logits of shape {tuple(logits.shape)} have no dimension {dim}")
        self.dim = dim % logits.dim()
        self.lead, self.vocab = logits.shape[:self.dim], logits.shape[self.dim]
        self.rows, self.inner = math.prod(self.lead), math.prod(logits.shape[self.dim + 1:])
        d = self.desc = L.LogitsDesc(rows=self.rows, vocab=self.vocab, inner=self.inner, type=_TYPE_ID[logits.dtype], masked_value=masked_value,
                                     history_rows=1, bias_rows=1, mask_rows=1, repetition_rows=1, presence_rows=1, frequency_rows=1,
                                     temperature_rows=1)
        self.device = logits.device
        self.kept = []                               # tensors that the descriptor points into
        if history is not None:
            if history.dtype not in _INTS or history.dim() == 0:
                raise TypeError("history holds int32 or int64 entries [..., length]")
            d.history_rows = _rows_of("history", history.shape[:-1], self.lead)
            d.history_len, d.history_wide = history.shape[-1], history.dtype == torch.int64
            d.history = self._place("history", history)
            lens = [t for t in (history_lens, prompt_lens) if t is not None]
            if any(t.dtype not in _INTS for t in lens) or len({t.dtype for t in lens}) > 1:
                raise TypeError("history_lens and prompt_lens are int32 or int64, both alike")
            for name, t in (("history_lens", history_lens), ("prompt_lens", prompt_lens)):
                if t is not None:
                    if t.shape != history.shape[:-1]:
                        raise ValueError(f"{name} has shape {tuple(t.shape)}, the history has rows {tuple(history.shape[:-1])}")
                    d.lens_wide = t.dtype == torch.int64
                    setattr(d, name, self._place(name, t))
        elif history_lens is not None or prompt_lens is not None:
            raise ValueError("history_lens and prompt_lens go with a history")
        for name, value in penalties.items():
            if isinstance(value, torch.Tensor):
                if value.dtype != torch.float32:
                    raise TypeError(f"{name} is a number or float32, got {value.dtype}")
                setattr(d, name + "_rows", _rows_of(name, value.shape, self.lead))
                setattr(d, name + "_t", self._place(name, value.detach()))
            else:
                value = float(value)
                if not math.isfinite(value) or (name in ("repetition", "temperature") and value <= 0):
                    raise ValueError(f"{name} {value}")
                setattr(d, name, value)
        if mask is not None:
            if mask.dtype not in (torch.bool, torch.int32) or mask.dim() == 0:
                raise TypeError("mask holds truth values, or bits in int32 words")
            d.mask_type = 1 if mask.dtype == torch.bool else 2
            if mask.shape[-1] != (self.vocab if d.mask_type == 1 else -(-self.vocab // 32)):
                raise ValueError(f"mask of shape {tuple(mask.shape)} for {self.vocab} entries")
            d.mask_rows = _rows_of("mask", mask.shape[:-1], self.lead)
            d.mask = self._place("mask", mask)
        if bias is not None:
            if bias.dtype != torch.float32 or bias.dim() == 0:
                raise TypeError("bias is float32 [..., vocabulary]")
            if bias.shape[-1] != self.vocab:
                raise ValueError(f"bias of shape {tuple(bias.shape)} for {self.vocab} entries")
            d.bias_rows = _rows_of("bias", bias.shape[:-1], self.lead)
            d.bias = self._place("bias", bias)

    def _place(self, name, t):
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the logits are on {self.device}")
        t = t.contiguous()
        self.kept.append(t)
        return t.data_ptr()

    def dense(self, t):
        """t itself if its rows can be walked, a contiguous copy otherwise; and its row stride."""
        stride = _row_stride(t, self.dim)
        if stride is None or stride < 0:
            t = t.contiguous()
            stride = self.vocab * self.inner
        return t, stride


def _forward(rules, logits, out):
    d = rules.desc
    x, d.in_stride = rules.dense(logits)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    d.out_stride = _row_stride(out, rules.dim)
    with L.device_guard(logits.device):
        L.check(L.load().gcn_logits_process(ctypes.byref(d), x.data_ptr(), out.data_ptr(), L.stream_ptr(logits.device)), "gcn_logits_process")
    return x, out


class ProcessLogitsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, rules):
        x, out = _forward(rules, logits, None)
        # what the gradient reads (not the bias) is saved, for autograd's own check of changes in between
        ctx.save_for_backward(x, *(t for t in rules.kept if t.data_ptr() != rules.desc.bias))
        ctx.rules = rules
        ctx.bias_shape = None if bias is None else bias.shape
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, *_ = ctx.saved_tensors
        rules = ctx.rules
        d = type(rules.desc).from_buffer_copy(rules.desc)
        want_x, want_bias = ctx.needs_input_grad[:2]
        dout = dout.contiguous()
        d.out_stride = rules.vocab * rules.inner
        dx = torch.empty(dout.shape, dtype=x.dtype, device=x.device) if want_x else None
        dbias = torch.zeros(ctx.bias_shape, dtype=torch.float32, device=x.device) if want_bias and rules.rows == 0 else None
        if want_bias and dbias is None:
            dbias = torch.empty(ctx.bias_shape, dtype=torch.float32, device=x.device)
        lib = L.load()
        nbytes = lib.gcn_logits_bwd_ws_bytes(ctypes.byref(d)) if want_bias else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        with L.device_guard(x.device):
            rc = lib.gcn_logits_process_bwd(ctypes.byref(d), x.data_ptr(), dout.data_ptr(), None if dx is None else dx.data_ptr(),
                                            None if dbias is None else dbias.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
                                            L.stream_ptr(x.device))
        L.check(rc, "gcn_logits_process_bwd")
        return dx, dbias, None


def process_logits(logits, *, dim=-1, history=None, history_lens=None, prompt_lens=None, repetition_penalty=1.0, presence_penalty=0.0,
                   frequency_penalty=0.0, bias=None, mask=None, temperature=1.0, masked_value=-math.inf, out=None):
    """The logits after penalties, bias, temperature and mask, of the same shape and type.

    logits: float32, bfloat16 or float16 ``[*lead, V, *inner]`` with the vocabulary at ``dim``.  The other arguments hold rows
    for ``lead``, for its last few dimensions (the same for all others), or one row for all, and apply to all of ``inner``:
      history ``[*rows, length]``, int32 or int64: entries that occurred; those outside ``[0, V)`` are skipped (padding).
        history_lens, prompt_lens ``[*rows]``: the first history_lens entries count; those before prompt_lens count for the
        repetition penalty only.  The same entry may occur any number of times.
      repetition_penalty, presence_penalty, frequency_penalty, temperature: numbers, or float32 ``[*rows]`` (repetition
        penalties and temperatures must be positive; numbers are checked).
      bias: float32 ``[*rows, V]``.
      mask: what is allowed, as truth values ``[*rows, V]`` or as bits (``pack_mask``); the rest becomes masked_value.  A row
        whose mask leaves nothing becomes masked_value throughout: with -inf a softmax over it is NaN.
    Differentiable in logits and bias (at x = 0 with the slope below it); penalties and temperatures are constants.
    out: a tensor for the result, which may be ``logits``; not with gradients."""
    rules = _Rules(logits, dim, history, history_lens, prompt_lens,
                   dict(repetition=repetition_penalty, presence=presence_penalty, frequency=frequency_penalty, temperature=temperature),
                   bias, mask, float(masked_value))
    grad = torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad))
    if out is not None:
        if grad:
            raise ValueError("out does not go with gradients")
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
            raise ValueError("out is a tensor like the logits")
        stride = _row_stride(out, rules.dim)
        if stride is None or (rules.rows > 1 and stride < rules.vocab * rules.inner):
            raise ValueError("out needs dense rows that do not overlap")
    L.require_cuda(logits, "logits")
    if grad:
        return ProcessLogitsFn.apply(logits, bias, rules)
    if logits.numel() == 0:
        return torch.empty_like(logits) if out is None else out
    return _forward(rules, logits.detach(), out)[1]
