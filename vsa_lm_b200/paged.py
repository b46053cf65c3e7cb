"""Paged KV cache of a softmax anchor layer, and its bound by accumulated attention weight.

The reference's anchor cache is one buffer that grows with the text (vsa_lm/decode.py:88-106), the only part of a
hybrid model's decode state that does. Here the rows live in pages that a table names, and with a `budget` each KV head
keeps that many rows: the newest ones and those that got the most attention so far (csrc/paged.cu, csrc/paged_attend.cu,
csrc/paged_prompt.cu). Beams share the pages of their common past.
"""
from __future__ import annotations

import torch

from . import kernels as K


class AnchorKVPaged:
    """Paged bf16 KV cache of one softmax anchor layer: `pages` [2, P, HKV, page, HD] (keys, then values) and an int32
    `table` [B, W] of each sequence's pages, in order; `n` rows are held of every sequence. GPU only. The capacity is
    max_kv_len rounded up to a multiple of 256 tokens and doubles when an append does not fit.

    With a `budget`, `weight` and `order` [B, HKV, W * page] record the softmax weight that each row got so far and its token's
    position. At every `chunk`-th token of the text a head that holds more than `budget` rows drops the others: it keeps its
    `recent` newest rows (half of the budget by default) and those of the largest weight. Between two such tokens the cache
    grows, so up to 2 * chunk rows more are held while steps take at most `chunk` tokens. Rows are then in no order."""

    CHECK_TOKENS = 128

    def __init__(self, B: int, HKV: int, Tmax: int, HD: int, dev, page: int = 64, budget: int | None = None,
                 recent: int | None = None, chunk: int = 128):
        check_budget(page, budget, recent)
        cap = max(256, -(-int(Tmax) // 256) * 256)
        if budget is not None:
            cap = min(cap, budget + 2 * chunk)
        W = -(-cap // page)
        self.B, self.budget, self.chunk = B, budget, chunk
        self.recent = None if budget is None else budget // 2 if recent is None else recent
        self.pages = torch.empty(2, B * W, HKV, page, HD, device=dev, dtype=torch.bfloat16)
        self.table = torch.arange(B * W, device=dev, dtype=torch.int32).view(B, W)
        self.own = self.table             # the page of each place that a sequence writes when it gets there
        self.weight = self.order = None
        if budget is not None:
            self.weight = torch.zeros(B, HKV, W * page, device=dev, dtype=torch.float32)
            self.order = torch.zeros(B, HKV, W * page, device=dev, dtype=torch.int32)
        self.n = self.seen = 0            # rows held, tokens seen
        self.status = K.DeviceStatus(dev) if self.pages.is_cuda else None

    def check_status(self, block: bool = True) -> None:
        """Raise RuntimeError if a kernel of an earlier step reported an error (block=False: only if the copy
        asked for by the last such call has arrived with one)."""
        if self.status is not None:
            if block:
                self.status.settle("paged anchor cache")
            else:
                self.status.check(False)
                self.status.arm("paged anchor cache")

    @property
    def page(self) -> int:
        return self.pages.shape[3]

    @property
    def capacity(self) -> int:
        return self.table.shape[1] * self.page

    @property
    def k(self) -> torch.Tensor:
        return self.read()[0]

    @property
    def v(self) -> torch.Tensor:
        return self.read()[1]

    @property
    def positions(self) -> torch.Tensor:
        """The positions of the held rows, int32 [B, HKV, n] (a cache without a budget holds all: row r is token r)."""
        if self.order is not None:
            return self.order[..., :self.n].clone()
        return torch.arange(self.n, device=self.pages.device, dtype=torch.int32).expand(self.B, self.pages.shape[2], -1)

    def read(self, t0: int = 0, t1: int | None = None) -> torch.Tensor:
        """Rows t0 .. t1 - 1 (all held ones by default) as bf16 [2, B, HKV, t1 - t0, HD]: keys, values."""
        t1 = self.n if t1 is None else t1
        if not 0 <= t0 <= t1 <= self.n:
            raise ValueError(f"rows [{t0}, {t1}) of a cache that holds {self.n}")
        r = torch.arange(t0, t1, device=self.pages.device)
        at = self.table.long()[:, r // self.page]                                   # [B, rows]
        return self.pages[:, at, :, r % self.page].permute(2, 0, 3, 1, 4).contiguous()   # indexed dimensions come first

    def tensors(self) -> list[torch.Tensor]:
        """What holds the tokens."""
        return [self.pages]

    def reserve(self, L: int) -> None:
        """Room for L more tokens: the pages of a sequence double (one copy of the pool) until they fit."""
        if self.n + L <= self.capacity:
            return
        B, W = self.table.shape
        more = W
        while (W + more) * self.page < self.n + L:
            more *= 2
        P = self.pages.shape[1]
        pages = self.pages.new_empty(2, P + B * more, *self.pages.shape[2:])
        pages[:, :P].copy_(self.pages)
        new = torch.arange(P, P + B * more, device=pages.device, dtype=torch.int32).view(B, more)
        shared = self.own is self.table
        self.own = torch.cat((self.own, new), 1)
        self.table = self.own if shared else torch.cat((self.table, new), 1)
        self.pages = pages
        if self.weight is not None:
            self.weight, self.order = (torch.cat((t, t.new_zeros(*t.shape[:2], more * self.page)), 2)
                                       for t in (self.weight, self.order))

    def advance(self, t: int) -> bool:
        """t more tokens are held; past a chunk's end the rows above the budget are dropped (True: rows have moved). At every
        CHECK_TOKENS of them an error of the kernels before the last such point is raised."""
        checks, chunks = self.seen // self.CHECK_TOKENS, self.seen // self.chunk
        self.n += t
        self.seen += t
        if self.status is not None and self.seen // self.CHECK_TOKENS != checks:
            self.status.check(block=True)
            self.status.arm(f"paged anchor cache at {self.seen} tokens")
        if self.budget is None or self.n <= self.budget or self.seen // self.chunk == chunks:
            return False
        self.n = K.paged_evict(pages=self.pages, table=self.table, weight=self.weight, order=self.order, n=self.n,
                               keep=self.budget, recent=self.recent, status=self.status)
        return True

    def repeated(self, times: int) -> "AnchorKVPaged":
        """A cache whose sequences are this cache's, each `times` times in a row (an error that its kernels reported is
        the copy's too). Without a budget full pages are shared, and only the last one is copied for each."""
        new = AnchorKVPaged.__new__(AnchorKVPaged)
        B, W = self.table.shape
        S = B * times
        new.B, new.budget, new.recent, new.chunk, new.n, new.seen = S, self.budget, self.recent, self.chunk, self.n, self.seen
        dev, page = self.pages.device, self.page
        full = 0 if self.budget is not None else self.n // page       # pages that are not written any more
        held = -(-self.n // page)
        new.pages = self.pages.new_empty(2, B * full + S * (W - full), *self.pages.shape[2:])
        old = self.table.long()
        new.pages[:, :B * full] = self.pages[:, old[:, :full].reshape(-1)]
        common = torch.arange(B * full, device=dev, dtype=torch.int32).view(B, full).repeat_interleave(times, 0)
        mine = torch.arange(B * full, B * full + S * (W - full), device=dev, dtype=torch.int32).view(S, W - full)
        if held > full:
            new.pages[:, mine[:, :held - full].reshape(-1).long()] = self.pages[:, old[:, full:held].repeat_interleave(times, 0).reshape(-1)]
        new.own = torch.cat((common, mine), 1)
        new.table = new.own.clone()
        new.weight, new.order = (None if t is None else t.repeat_interleave(times, 0) for t in (self.weight, self.order))
        new.status = None
        if self.status is not None:
            new.status = K.DeviceStatus(dev)
            new.status.word.copy_(self.status.word)
        return new

    def reorder(self, parent: torch.Tensor) -> None:
        """Every beam's rows become those of its parent (int32 [groups, beams], as beam_select gives it: a beam that goes on
        keeps its slot). The table's rows move; of the pages only the one that is not full yet is copied, into the beam's own."""
        if self.budget is not None:
            raise ValueError("a cache with a budget cannot share pages between beams")
        groups, beams = parent.shape
        src = (parent.long() + torch.arange(groups, device=parent.device)[:, None] * beams).view(-1)
        table, at = self.table[src], self.n // self.page
        if self.n % self.page:
            self.pages[:, self.own[:, at].long()] = self.pages[:, table[:, at].long()]
        table[:, at:] = self.own[:, at:]
        self.table.copy_(table)

    def attention(self, ly, h: torch.Tensor, pos_start: int, dev_pos: "K.DevicePosition | None" = None) -> torch.Tensor:
        """An anchor layer's attention for t new tokens h [b, t, D]: q and k normed and rotated, k and v into the pages,
        the causal attention over all held rows; [b, t, H * HD] bf16. With dev_pos (a step captured into a CUDA graph) the
        position comes from the device and the count is left to the caller."""
        from .bolt3 import _fp32_inv_freq, _fp32_weight

        t = h.shape[1]
        if dev_pos is None:
            self.reserve(t)
        q, k, v = ly.q_proj(h), ly.k_proj(h), ly.v_proj(h)
        norm = ly.q_norm is not None
        q = K.paged_append(q=q, k=k, v=v, pages=self.pages, table=self.table, n=self.n, pos0=pos_start,
                           inv_freq=_fp32_inv_freq(ly.rope, h.device),
                           q_norm=_fp32_weight(ly.q_norm, h.device) if norm else None,
                           k_norm=_fp32_weight(ly.k_norm, h.device) if norm else None,
                           eps=ly.q_norm.eps if norm else 0.0, weight=self.weight, order=self.order, status=self.status,
                           dev_pos=dev_pos)
        y = K.paged_attend(q=q, pages=self.pages, table=self.table, n=self.n, sm_scale=ly.HD ** -0.5, weight=self.weight,
                           status=self.status, dev_pos=dev_pos)
        if dev_pos is None:
            self.advance(t)
        return y


def check_budget(page: int, budget: int | None, recent: int | None) -> None:
    if page not in (16, 32, 64, 128):
        raise ValueError(f"pages hold 16, 32, 64 or 128 rows, got {page}")
    if budget is None:
        if recent is not None:
            raise ValueError("a number of recent rows goes with a budget")
    elif budget < 1 or not 0 <= (0 if recent is None else recent) <= budget:
        raise ValueError(f"a budget of {budget} rows with {recent} recent ones: at least 1, and recent within [0, budget]")
