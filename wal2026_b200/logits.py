"""Rules on logits: penalties for repeated tokens, biases, grammar masks, temperature (C ABI wrapper).

``logit_rules`` turns the logits of a step's T tokens per sequence into the
probabilities that ``verify_drafts`` takes, or into changed logits.  ``lens``
counts as it does for the paged cache: the tokens a sequence held before the
step, so that row t of sequence b follows ``text[b, : lens[b] + t + 1]``.
``LogitRules`` holds the rules of a decoder's rows (``PagedDecoder.speculate``).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch
from torch import Tensor

from . import _abi
from .kv8 import _call, _cuda, _i32, _is_i32, _on

MAX_VOCAB = 393216
MAX_BIAS = 1024
MAX_TEXT = (1 << 20) - 1


@dataclass
class LogitRules:
    """Rules of the rows of a batch; every tensor may be None, all live on the rows' device.

    repetition, presence, frequency, temperature: fp32 [rows]; bias_ids int32 and
    bias fp32 [rows, n] (-1 for unused places); mask: int32 words of 32 tokens,
    [rows, T, ceil(vocab / 32)] or [rows, 1, ..] for every token of a step.
    """

    repetition: Optional[Tensor] = None
    presence: Optional[Tensor] = None
    frequency: Optional[Tensor] = None
    bias_ids: Optional[Tensor] = None
    bias: Optional[Tensor] = None
    mask: Optional[Tensor] = None
    temperature: Optional[Tensor] = None

    def penalises(self) -> bool:
        return any(t is not None for t in (self.repetition, self.presence, self.frequency))


def pack_mask(allowed: Tensor) -> Tensor:
    """Words of a mask bool [..., V]: int32 [..., ceil(V / 32)], bit v % 32 of word v / 32 set where token v is allowed."""
    V = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _stride(t: Tensor, s: tuple) -> int:
    """Elements between the rows of one sequence (the stride of a single row says nothing)."""
    return s[1] if t.shape[1] > 1 else t.shape[2]


_I32, _F32 = torch.int32, torch.float32


def _is_f32(t: Optional[Tensor], shape: tuple, index: int) -> bool:
    return t is None or (t.dtype is _F32 and t.shape == shape and t.is_contiguous() and t.get_device() == index)


def _maybe_i32(t: Optional[Tensor], shape: tuple, index: int) -> bool:
    return t is None or _is_i32(t, shape, index)


def _why_not(logits, out, text, lens, prompt_lens, new_lens, repetition, presence, frequency, bias_ids, bias, mask,
             temperature) -> None:
    if logits.dim() != 3 or logits.dtype not in _abi.DTYPE_CODE or logits.stride(2) != 1 or logits.numel() == 0:
        raise ValueError("logits must be bf16, fp16 or fp32 [B, T, V] with contiguous rows")
    B, T, V = logits.shape
    if out.dtype != torch.float32 or out.shape != logits.shape or out.stride(2) != 1:
        raise ValueError("out must be fp32 [B, T, V] with contiguous rows")
    if V > MAX_VOCAB:
        raise ValueError(f"logit_rules takes at most {MAX_VOCAB} tokens, got {V}")
    if (repetition is not None or presence is not None or frequency is not None) and (text is None or lens is None):
        raise ValueError("penalties need text and lens")
    if text is not None and (text.dtype != torch.int32 or text.dim() != 2 or text.shape[0] != B
                             or (text.stride(1) != 1 and text.shape[1] > 1)):
        raise ValueError("text must be int32 [B, L] with contiguous rows")
    if text is not None and text.shape[1] > MAX_TEXT:
        raise ValueError(f"logit_rules takes texts of at most {MAX_TEXT} tokens, got {text.shape[1]}")
    for name, t in (("lens", lens), ("prompt_lens", prompt_lens), ("new_lens", new_lens)):
        if t is not None:
            _i32(name, t, B)
    for name, t in (("repetition", repetition), ("presence", presence), ("frequency", frequency), ("temperature", temperature)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (B,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 tensor of shape [{B}]")
    if (bias is None) != (bias_ids is None):
        raise ValueError("bias_ids and bias come together")
    if bias is not None:
        nb = bias_ids.shape[-1] if bias_ids.dim() == 2 else 0
        _i32("bias_ids", bias_ids, B, nb)
        if bias.dtype != torch.float32 or tuple(bias.shape) != (B, nb) or not bias.is_contiguous():
            raise ValueError("bias must be contiguous fp32 like bias_ids")
        if nb > MAX_BIAS:
            raise ValueError(f"logit_rules takes at most {MAX_BIAS} biases a row, got {nb}")
    if mask is not None and (mask.dtype != torch.int32 or tuple(mask.shape) != (B, T, -(-V // 32)) or mask.stride(2) != 1):
        raise ValueError(f"mask must be int32 [B, T, {-(-V // 32)}] with contiguous rows")
    _cuda(logits.device)
    _on(logits.device, out=out, text=text, lens=lens, prompt_lens=prompt_lens, new_lens=new_lens, repetition=repetition,
        presence=presence, frequency=frequency, bias_ids=bias_ids, bias=bias, mask=mask, temperature=temperature)
    raise ValueError("logit_rules: arguments do not fit together")


def logit_rules(logits: Tensor, out: Tensor, *, text: Optional[Tensor] = None, lens: Optional[Tensor] = None,
                prompt_lens: Optional[Tensor] = None, new_lens: Optional[Tensor] = None, repetition: Optional[Tensor] = None,
                presence: Optional[Tensor] = None, frequency: Optional[Tensor] = None, bias_ids: Optional[Tensor] = None,
                bias: Optional[Tensor] = None, mask: Optional[Tensor] = None, temperature: Optional[Tensor] = None,
                softmax: bool = True) -> None:
    """out[b, t] = softmax of the logits of row t of sequence b after the rules (softmax=False: those logits themselves).

    logits: bf16, fp16 or fp32 [B, T, V]; out: fp32 [B, T, V], rows contiguous in
    both.  In this order: a token of ``text[b, : lens[b] + t + 1]`` (int32 [B, L])
    has its logit divided by repetition[b] where positive, multiplied where not;
    frequency[b] times its count and, once, presence[b] come off a token that was
    generated (position prompt_lens[b] or later; None: all); bias[b, i] (fp32 [B,
    n]) is added to token bias_ids[b, i] (int32; equal ones add up); tokens whose
    bit of ``mask`` (int32 words [B, T, ceil(V / 32)], expanded axes allowed) is
    clear, and NaN, are left out; the rest is divided by temperature[b].  out must not
    overlap logits.
    Temperature 0 (or below) gives the first of the largest logits probability 1, and leaves
    logits undivided.  A row with no token left is all zeros (logits: -inf), rows
    t >= new_lens[b] are zeros.  Tokens outside [0, V) count nowhere.
    """
    index, shape, ls, os = logits.get_device(), logits.shape, logits.stride(), out.stride()
    fit = (index >= 0 and len(shape) == 3 and out.shape == shape and ls[2] == 1 and os[2] == 1 and logits.dtype in _abi.DTYPE_CODE
           and out.dtype is _F32 and out.get_device() == index and 0 < shape[2] <= MAX_VOCAB and shape[0] > 0 and shape[1] > 0)
    nb, text_len, ld_text = 0, 0, 0
    if fit:
        B, T, V = shape
        rows = (B,)
        if text is not None:
            ts, t1 = text.shape, text.stride()
            fit = (len(ts) == 2 and ts[0] == B and text.dtype is _I32 and text.get_device() == index and ts[1] <= MAX_TEXT
                   and (t1[1] == 1 or ts[1] <= 1))
            if fit:
                text_len, ld_text = ts[1], t1[0] if B > 1 else ts[1]
        elif repetition is not None or presence is not None or frequency is not None:
            fit = False
        if bias_ids is not None:
            nb = bias_ids.shape[-1] if bias_ids.dim() == 2 else -1
            fit = fit and 0 <= nb <= MAX_BIAS and bias is not None and _is_i32(bias_ids, (B, nb), index) and _is_f32(bias, (B, nb), index)
        if mask is not None:
            ms, m1 = mask.shape, mask.stride()
            fit = fit and ms == (B, T, -(-V // 32)) and m1[2] == 1 and mask.dtype is _I32 and mask.get_device() == index
        fit = (fit and (bias is None) == (bias_ids is None) and _maybe_i32(lens, rows, index) and _maybe_i32(prompt_lens, rows, index)
               and _maybe_i32(new_lens, rows, index) and _is_f32(repetition, rows, index) and _is_f32(presence, rows, index)
               and _is_f32(frequency, rows, index) and _is_f32(temperature, rows, index)
               and (lens is not None or (repetition is None and presence is None and frequency is None)))
    if not fit:
        _why_not(logits, out, text, lens, prompt_lens, new_lens, repetition, presence, frequency, bias_ids, bias, mask, temperature)
    if nb == 0:
        bias_ids = bias = None
    p = _ptr
    rules = _abi.LogitRules(p(text), ld_text, text_len, p(lens), p(prompt_lens), p(new_lens), p(repetition), p(presence), p(frequency),
                            p(bias_ids), p(bias), nb, p(mask), 0 if mask is None else m1[0], 0 if mask is None else m1[1], p(temperature))
    _call(index, "wal_logit_rules_apply", ctypes.byref(rules), logits.data_ptr(), _abi.DTYPE_CODE[logits.dtype], ls[0],
          _stride(logits, ls), B, T, V, out.data_ptr(), os[0], _stride(out, os), 1 if softmax else 0)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()
