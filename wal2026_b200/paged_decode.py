"""Decoding with the paged 8-bit KV cache: prompts, several sequences of their own lengths, drafts, forks.

``PagedDecoder`` drives a ``LlamaStack`` whose sequences keep their positions in
pages of a ``PagedKV8Cache``.  One call takes T new tokens per sequence (a
prompt, one token, or the last token and its drafts); all of its state (tables,
lengths, the last accepted token) lives on the device, so a step launches
without waiting for the host and can be captured into a CUDA graph:

    dec = PagedDecoder(stack, rows=2, max_len=4096, num_pages=256)
    dec.step(prompt, new_lens)                    # [rows, T] tokens, ragged
    dec.advance(new_lens)                         # keep them
    logits = dec.step(tokens)                     # one more each
    accepted, out = dec.speculate(drafts, uniforms, last=tokens, temperature=0.8)
    dec.fork([0, 0])                              # both rows continue sequence 0

With ``share`` the attention reads what forked rows have in common once for all
of them, which pays for many rows of a long prompt; with ``text`` the decoder keeps the rows' tokens, which the penalties of
``LogitRules`` need (``speculate(..., rules=rules)``, or ``logit_rules`` on the
logits of a step).

``python -m wal2026_b200.paged_decode`` runs a small random stack that way.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor

from .decode_ops import residual_rmsnorm, silu_mul
from .kv8 import (PagedKV8Cache, kv8_append, kv8_attention, kv8_attention_shared, kv8_attention_shared_workspace,
                  kv8_attention_workspace, kv_pages_assign, kv_pages_compact, kv_pages_copy, kv_pages_groups)
from .llama import LlamaStack, _linear_into
from .logits import MAX_TEXT, LogitRules, logit_rules
from .runtime import PREFILL_MIN_TOKENS, PackedGroupedBlockRVQLinear
from .speculative import verify_drafts


class _StepBuffers:
    """Activations of steps of up to ``tokens`` tokens per row, and the attention's workspace."""

    def __init__(self, stack: LlamaStack, rows: int, tokens: int, cache: PagedKV8Cache, shared: bool):
        s, l0, dev, bf = stack.shape, stack.layers[0], stack.embed.device, torch.bfloat16
        M, hd = rows * tokens, s.head_dim
        self.tokens = tokens
        self.h = torch.empty(M, s.hidden, device=dev, dtype=bf)
        self.x = torch.empty(M, s.hidden, device=dev, dtype=bf)
        self.qkv = torch.empty(M, (l0.hq + 2 * l0.hkv) * hd, device=dev, dtype=bf)
        self.q = torch.empty(M, l0.hq * hd, device=dev, dtype=bf)
        self.attn = torch.empty(M, l0.hq * hd, device=dev, dtype=bf)
        self.gu = torch.empty(M, 2 * l0.mlp, device=dev, dtype=bf)
        self.act = torch.empty(M, l0.mlp, device=dev, dtype=bf)
        self.y32 = torch.empty(M, s.hidden, device=dev, dtype=torch.float32)
        self.ws = (kv8_attention_shared_workspace if shared else kv8_attention_workspace)(cache, rows, l0.hq, tokens)

    def first(self, M: int) -> "_StepBuffers":
        """The same buffers for a step of M token rows."""
        view = object.__new__(_StepBuffers)
        view.tokens, view.ws = self.tokens, self.ws
        for name in ("h", "x", "qkv", "q", "attn", "gu", "act", "y32"):
            setattr(view, name, getattr(self, name)[:M])
        return view


def _column(lin, x: Tensor, y: Tensor) -> None:
    """y = x w^T: the GEMV for decode-sized calls, the prefill GEMM for prompts of Block-RVQ linears (4-bit ones have none)."""
    if isinstance(lin, PackedGroupedBlockRVQLinear) and x.shape[0] >= PREFILL_MIN_TOKENS and lin.gemm_into(x, y):
        return
    _linear_into(lin, x, y)


class PagedDecoder:
    """Sequences of a ``LlamaStack`` over one paged 8-bit cache.

    rows: sequences decoded together; max_len: most positions of one sequence,
    rounded up to whole pages;
    num_pages: the pool they share (default: room for every row at max_len).
    ``table`` int32 [rows, max_len / page_size] and ``lens`` int32 [rows] are the
    state; ``info`` after a step holds (pages left free, pages that were wanted
    but not given).

    A step that is not given every page it wants (the pool or a row is full)
    stores nothing and leaves ``table`` and ``lens`` as they were; its logits mean
    nothing, and ``advance`` after it does nothing.  It can be repeated once
    ``fork`` has emptied a row, or with ``new_lens`` 0 for the row that is full.
    ``missing`` int64 [1] sums such pages over all steps, so that a loop which
    never waits for the device can look now and then: 0 means that every step
    was carried out.

    share: rows whose first ``share`` positions (or more) lie in the same pages are
    a group, whose common positions each step reads once (``kv_pages_groups``, and
    ``kv8_attention_shared`` for what that rounds and from where on it pays: a small
    ``share`` makes steps of few rows or short prompts slower); None: every row reads its own.  ``status`` int32 [1] becomes 1, and stays so until
    the caller clears it, where that attention gave up a wait (after 2 s): what the steps
    since its last 0 returned and stored is wrong.  text: keep the rows' tokens in ``text`` int32
    [rows, max_len], by position; ``prompt_lens`` int32 [rows] (0 to begin with, the
    caller's to set) says where what the rows generated starts.
    """

    def __init__(self, stack: LlamaStack, rows: int, max_len: int, *, num_pages: Optional[int] = None,
                 page_size: int = 64, dtype: torch.dtype = torch.int8, share: Optional[int] = None, text: bool = False):
        if rows < 1 or max_len < 1:
            raise ValueError("rows and max_len must be positive")
        if share is not None and share < 1:
            raise ValueError("share must be positive, or None")
        dev, l0 = stack.embed.device, stack.layers[0]
        width = -(-max_len // page_size)
        self.stack, self.rows, self.max_len = stack, rows, width * page_size
        self.cache = PagedKV8Cache.allocate(len(stack.layers), num_pages or rows * width, l0.hkv, stack.shape.head_dim,
                                            page_size=page_size, dtype=dtype, device=dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((rows, width), -1, **i32)
        self.lens = torch.zeros(rows, **i32)
        self.info = torch.zeros(2, **i32)
        self.missing = torch.zeros(1, dtype=torch.int64, device=dev)
        self.status = torch.zeros(1, **i32)
        self._room = torch.ones(1, dtype=torch.bool, device=dev)  # whether the last step got its pages
        self._next = torch.empty_like(self.table)
        self._self = torch.arange(rows, **i32)
        self._zero = torch.zeros(rows, **i32)
        self._ref = torch.empty(self.cache.num_pages, **i32)
        self._src, self._dst = torch.empty(rows, **i32), torch.empty(rows, **i32)
        self.share = share
        self.groups = None if share is None else torch.zeros(4, rows, **i32)
        self.text = self.prompt_lens = None
        if text:
            if self.max_len > MAX_TEXT:
                raise ValueError(f"a decoder keeps texts of at most {MAX_TEXT} tokens, max_len is {self.max_len}")
            self._text = torch.zeros(rows, self.max_len + 1, **i32)  # the last place takes tokens that are not kept
            self.text, self.prompt_lens = self._text[:, :self.max_len], torch.zeros(rows, **i32)
        ang = torch.arange(self.max_len, device=dev, dtype=torch.float32)[:, None] * stack.inv_freq
        self.cos, self.sin = ang.cos().contiguous(), ang.sin().contiguous()
        self._bufs: Optional[_StepBuffers] = None  # of the largest step so far
        self._views: dict[int, _StepBuffers] = {}  # its first rows, by step size
        self._captured: list[_StepBuffers] = []    # sets that a graph uses

    def _buffers(self, T: int) -> _StepBuffers:
        """Buffers of a step of T tokens per row: one set serves all sizes and grows with the largest.

        A set that a graph captured stays when a larger one replaces it, and a
        graph that captures a larger step than any before gets one of its own.
        """
        capturing = torch.cuda.is_current_stream_capturing()
        if self._bufs is None or self._bufs.tokens < T:
            if capturing:
                self._captured.append(_StepBuffers(self.stack, self.rows, T, self.cache, self.share is not None))
                return self._captured[-1]
            if self._bufs is not None:
                for t in vars(self._bufs).values():
                    if isinstance(t, Tensor):
                        t.record_stream(torch.cuda.current_stream(t.device))
            self._bufs, self._views = None, {}
            self._bufs = _StepBuffers(self.stack, self.rows, T, self.cache, self.share is not None)
        if capturing and not any(b is self._bufs for b in self._captured):
            self._captured.append(self._bufs)
        view = self._views.get(T)
        if view is None:
            view = self._views[T] = self._bufs.first(self.rows * T)
        return view

    def _assign(self, parent: Tensor, keep: Tensor, add: Tensor) -> None:
        """The next table, in ``_next``, and the copies it asks for (into pages that no kept token is in)."""
        kv_pages_assign(self.table, parent, keep, add, self.cache.page_size, self._next, self._ref, self._src, self._dst,
                        self.info)
        kv_pages_copy(self.cache, self._src, self._dst)

    def _reserve(self, add: Tensor) -> Tensor:
        """Room for add[row] more tokens each, or for none and everything as it was; the tokens that have room."""
        self._assign(self._self, self.lens, add)
        torch.eq(self.info[1:], 0, out=self._room)
        torch.where(self._room, self._next, self.table, out=self.table)
        self.missing.add_(self.info[1:])
        return add * self._room

    @torch.no_grad()
    def step(self, tokens: Tensor, new_lens: Optional[Tensor] = None) -> Tensor:
        """Logits [rows, T, vocab] (bf16) of T new tokens per row, stored behind the row's present positions.

        tokens: int [rows, T]; new_lens int32 [rows]: how many of them are real
        (logits of the others mean nothing).  Pages are reserved, and shared
        ones copied, as needed; where they run out, nothing is stored (see the
        class).  The rows' lengths stay as they are: ``advance`` keeps the tokens,
        another ``step`` overwrites them.
        """
        B, T = tokens.shape
        if B != self.rows:
            raise ValueError(f"tokens must have {self.rows} rows, got {B}")
        if T == 0:
            raise ValueError("a step takes at least one token per row")
        st, s = self.stack, self.stack.shape
        bufs = self._buffers(T)
        add = self._reserve(torch.full_like(self.lens, T) if new_lens is None else new_lens)
        if self.share is not None:  # the table as it is now serves all layers
            kv_pages_groups(self.table, self.lens, self.cache.page_size, self.groups, least=self.share)
        if self.text is not None:
            t = torch.arange(T, device=self.lens.device)
            at = torch.where(t < add[:, None], self.lens[:, None] + t, self.max_len)
            self._text.scatter_(1, at.long(), tokens.to(torch.int32))
        torch.index_select(st.embed, 0, tokens.reshape(-1), out=bufs.h)
        residual_rmsnorm(bufs.h, st.layers[0].in_norm, s.eps, bufs.x)
        n = len(st.layers)
        for i, layer in enumerate(st.layers):
            _column(layer.qkv, bufs.x, bufs.qkv)
            kv8_append(self.cache, i, bufs.qkv, layer.hq, self.table, self.lens, bufs.q, cos=self.cos, sin=self.sin,
                       new_lens=add)
            if self.share is None:
                kv8_attention(self.cache, i, bufs.q, self.table, self.lens, bufs.attn, bufs.ws, new_lens=add)
            else:
                kv8_attention_shared(self.cache, i, bufs.q, self.table, self.lens, self.groups, bufs.attn, bufs.ws, new_lens=add,
                                     status=self.status)
            self._row_parallel(layer.o, bufs.attn, layer.post_norm, bufs)
            _column(layer.gate_up, bufs.x, bufs.gu)
            silu_mul(bufs.gu, bufs.act)
            self._row_parallel(layer.down, bufs.act, st.layers[i + 1].in_norm if i + 1 < n else st.final_norm, bufs)
        return st.logits(bufs.x).view(B, T, -1)

    def _row_parallel(self, lin, a: Tensor, norm_w: Tensor, bufs: _StepBuffers) -> None:
        if (isinstance(lin, PackedGroupedBlockRVQLinear) and a.shape[0] >= PREFILL_MIN_TOKENS
                and lin.gemm_into(a, bufs.y32)):
            if self.stack.tp.size > 1:
                self.stack.tp.all_reduce_(bufs.y32)
            residual_rmsnorm(bufs.h, norm_w, self.stack.shape.eps, bufs.x, partial=bufs.y32)
        else:
            self.stack._row_parallel_fused(lin, a, 0, norm_w, bufs, "nccl")

    def advance(self, count: Optional[Tensor] = None) -> None:
        """Keep the first count[row] tokens (int32 [rows]; None: one each) of the last step, if it had room for them."""
        self.lens.add_(self._room if count is None else count * self._room)

    @torch.no_grad()
    def speculate(self, drafts: Tensor, uniforms: Tensor, *, last: Tensor, draft_probs: Optional[Tensor] = None,
                  temperature: float = 1.0, draft_lens: Optional[Tensor] = None,
                  rules: Optional[LogitRules] = None) -> tuple[Tensor, Tensor]:
        """One speculative step: run the rows' last tokens and their drafts, keep what the stack's probabilities allow.

        last: int32 [rows], each row's newest token (not stored yet); drafts:
        int32 [rows, T]; uniforms: fp32 [rows, T + 1]; draft_probs: fp32 [rows,
        T, vocab] or None (drafts chosen without probabilities); draft_lens int32
        [rows]: how many drafts of a row are real, -1 for a row that takes no
        part (accepted 0, every token -1, nothing stored).  Temperature 0
        keeps the drafts that are the most likely token.  Returns (accepted
        [rows], tokens [rows, T + 1]: the kept drafts, the drawn token, -1); the
        last token and the kept drafts stay in the cache, and the drawn token is
        the next call's ``last``.  A step that finds no room is one in which no
        row takes part.  rules: penalties, biases, masks and temperatures of the rows
        (``logit_rules``; penalties need a decoder with ``text``); their temperatures
        take the place of ``temperature``.
        """
        B, T = drafts.shape
        if rules is not None and rules.penalises() and self.text is None:
            raise ValueError("penalties need a decoder that keeps its text (text=True)")
        tokens = torch.cat([last.view(B, 1), drafts], dim=1)
        news = torch.full_like(self.lens, T + 1) if draft_lens is None else (draft_lens + 1).to(torch.int32)
        logits = self.step(tokens.clamp(0, self.stack.shape.vocab - 1), news)  # a draft outside is refused below
        if rules is not None:
            heat = rules.temperature
            if heat is None and temperature != 1.0:
                heat = torch.full((B,), float(temperature), device=logits.device)
            mask = rules.mask if rules.mask is None else rules.mask.expand(B, T + 1, -1)
            target = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
            logit_rules(logits, target, text=self.text, lens=self.lens, prompt_lens=self.prompt_lens, new_lens=news,
                        repetition=rules.repetition, presence=rules.presence, frequency=rules.frequency,
                        bias_ids=rules.bias_ids, bias=rules.bias, mask=mask, temperature=heat)
        elif temperature > 0:
            logits = logits.float()
            target = torch.softmax(logits / temperature, dim=-1)
        else:
            logits = logits.float()
            target = torch.zeros_like(logits).scatter_(2, logits.argmax(-1, keepdim=True), 1.0)
        accepted = torch.empty(B, dtype=torch.int32, device=drafts.device)
        out = torch.empty(B, T + 1, dtype=torch.int32, device=drafts.device)
        verify_drafts(target, draft_probs, drafts, uniforms, accepted, out, draft_lens=draft_lens)
        part = self._room if draft_lens is None else self._room & (draft_lens >= 0)
        accepted.mul_(part)
        out.masked_fill_(~part[:, None], -1)
        self.advance(accepted + part)
        return accepted, out

    def fork(self, parent: Sequence[int]) -> None:
        """Row i continues what row parent[i] holds (pages shared until one of them writes); -1 empties the row."""
        p = torch.tensor(list(parent), dtype=torch.int32, device=self.lens.device)
        if p.shape != self.lens.shape:
            raise ValueError(f"fork needs {self.rows} parents")
        if any(not -1 <= int(i) < self.rows for i in parent):
            raise ValueError(f"parents must be rows 0 .. {self.rows - 1}, or -1")
        lens = torch.where(p >= 0, self.lens[p.clamp(min=0).long()], 0)
        self._assign(p, lens, self._zero)  # wants no page
        self.table.copy_(self._next)
        self.lens.copy_(lens)
        if self.text is not None:
            i = p.clamp(min=0).long()
            self._text.copy_(self._text[i])
            self.prompt_lens.copy_(torch.where(p >= 0, self.prompt_lens[i], 0))

    def compact(self) -> None:
        """Move the used pages to the front of the pool (``info``: used pages, moves)."""
        n = self.cache.num_pages
        remap, src, dst = (torch.empty(n, dtype=torch.int32, device=self.lens.device) for _ in range(3))
        kv_pages_compact(self.table, self.lens, self.cache.page_size, self.table, remap, src, dst, self.info)
        kv_pages_copy(self.cache, src, dst)


def main() -> None:
    """Two prompts, a fork, and speculative steps with drafts from the text so far."""
    from .llama import LlamaShape, rvq_llama

    if not torch.cuda.is_available():
        raise SystemExit("paged_decode runs on a CUDA device")
    stack = rvq_llama(LlamaShape(layers=4, hidden=1024, mlp=2048, heads=8, kv_heads=2, vocab=2048), seed=3)
    dec = PagedDecoder(stack, rows=4, max_len=512, num_pages=40, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randint(0, 2048, (4, 37), device="cuda", generator=g)
    lens = torch.tensor([37, 21, 0, 0], dtype=torch.int32, device="cuda")
    logits = dec.step(prompt, lens)
    dec.advance(lens)
    dec.fork([0, 1, 0, 1])  # two samples of each prompt
    last = logits[torch.tensor([0, 1, 0, 1]), torch.tensor([36, 20, 36, 20])].argmax(-1).to(torch.int32)
    text = [[int(t)] for t in last]
    for _ in range(8):
        # a draft is whatever followed the last token before, or the token itself
        drafts = torch.tensor([[row[row.index(row[-1]) + 1 + k] if row.index(row[-1]) + 1 + k < len(row) else row[-1]
                                for k in range(3)] for row in text], dtype=torch.int32, device="cuda")
        accepted, out = dec.speculate(drafts, torch.rand(4, 4, device="cuda", generator=g), last=last, temperature=0.7)
        last = out.gather(1, accepted.view(4, 1).long()).view(4).contiguous()
        for row, toks in zip(text, out.tolist()):
            row += [t for t in toks if t >= 0]
    dec.compact()
    print("lengths", dec.lens.tolist(), "pages used, moved", dec.info.tolist())
    for row in text:
        print(row)


if __name__ == "__main__":
    main()
