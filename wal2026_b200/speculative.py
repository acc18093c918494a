"""Verification of drafted tokens (C ABI wrapper)."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _abi
from .kv8 import _call, _cuda, _i32, _is_i32, _on


def _row_stride(t: Tensor) -> int:
    """Elements between the rows of one sequence (the stride of a single row says nothing)."""
    return t.stride()[1] if t.shape[1] > 1 else t.shape[2]


def _why_not(target, draft, drafts, uniforms, accepted, tokens, draft_lens) -> None:
    dev = target.device
    if target.dtype != torch.float32 or target.dim() != 3 or target.stride(2) != 1 or target.shape[1] < 1:
        raise ValueError("target must be fp32 [B, T + 1, V] with contiguous rows")
    B, T, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    if draft is not None and (draft.dtype != torch.float32 or tuple(draft.shape) != (B, T, V) or draft.stride(2) != 1):
        raise ValueError("draft must be fp32 [B, T, V] with contiguous rows")
    _i32("drafts", drafts, B, T)
    _i32("accepted", accepted, B)
    _i32("tokens", tokens, B, T + 1)
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (B, T + 1) or not uniforms.is_contiguous():
        raise ValueError("uniforms must be fp32 [B, T + 1] contiguous")
    if draft_lens is not None:
        _i32("draft_lens", draft_lens, B)
    _cuda(dev)
    _on(dev, draft=draft, drafts=drafts, uniforms=uniforms, accepted=accepted, tokens=tokens, draft_lens=draft_lens)
    raise ValueError("verify_drafts: arguments do not fit together")


def verify_drafts(target: Tensor, draft: Optional[Tensor], drafts: Tensor, uniforms: Tensor, accepted: Tensor,
                  tokens: Tensor, *, draft_lens: Optional[Tensor] = None) -> None:
    """Keep the drafts that the target's probabilities allow and draw the token after them.

    target: fp32 probabilities [B, T + 1, V]; draft: the drafting model's [B, T,
    V], or None for drafts chosen without probabilities; drafts: int32 [B, T],
    of which draft_lens[b] are real; uniforms: fp32 [B, T + 1] in [0, 1) (draft t
    uses column t, the drawn token column T).  accepted: int32 [B]; tokens: int32
    [B, T + 1] = the kept drafts, the drawn token, then -1.

    Draft t is kept while u_t * q_t(x_t) < p_t(x_t); after a rejection the token
    is drawn from the positive part of p - q, else from p.  Probabilities count
    in whole numbers of 2^-38, so the outcome is the same in any order of
    summation.  A row whose probabilities are all zero gives token -1.
    """
    index, s, s1 = target.get_device(), target.shape, target.stride()
    fit = index >= 0 and len(s) == 3 and s[1] >= 1 and target.dtype is torch.float32 and s1[2] == 1
    if fit:
        B, T, V = s[0], s[1] - 1, s[2]
        fit = ((draft is None or (draft.shape == (B, T, V) and draft.dtype is torch.float32 and draft.stride()[2] == 1
                                  and draft.get_device() == index))
               and _is_i32(drafts, (B, T), index) and _is_i32(accepted, (B,), index) and _is_i32(tokens, (B, T + 1), index)
               and uniforms.shape == (B, T + 1) and uniforms.dtype is torch.float32 and uniforms.is_contiguous()
               and uniforms.get_device() == index and (draft_lens is None or _is_i32(draft_lens, (B,), index)))
    if not fit:
        _why_not(target, draft, drafts, uniforms, accepted, tokens, draft_lens)
    if T == 0:
        draft = None
    d0, d1 = (0, V) if draft is None else (draft.stride()[0], _row_stride(draft))
    _call(index, "wal_verify_drafts", target.data_ptr(), s1[0], _row_stride(target), None if draft is None else draft.data_ptr(),
          d0, d1, drafts.data_ptr() if T else None, T, None if draft_lens is None else draft_lens.data_ptr(),
          uniforms.data_ptr(), T + 1, B, T, V, accepted.data_ptr(), tokens.data_ptr(), T + 1)
