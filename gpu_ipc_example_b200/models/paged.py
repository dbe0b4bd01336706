"""A cache of keys and values in pages, for serving requests of different lengths with `LlamaTP`.

    cache = PagedCache(model, requests=64, max_len=8192, pages=4096)
    batch = cache.extend(new_lens, rows)                 # pages, slots and positions of the step's new tokens
    hidden = model.forward_paged(tokens, batch, cache)   # prompts, chunks of them, single tokens and drafts in one batch
    tokens, accepted = model.verify(last, drafts, draft_probs, cache, accept, sample)
    cache.trim(keep_lens)                                # drafts that were turned down, requests that are done (0)

Lengths, the block table and the list of free pages are on the GPU and no call here reads them back, so steps of one number of rows can be
captured in a CUDA graph; all calls on one cache follow one another, on a stream or by events.  What a call cannot do (no pages left, a
request beyond its row of the table, more tokens than rows) it leaves undone and says so in a word of its own; `check()`, which waits for the GPU, raises it.

The reference has no model code and no cache.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .._ext import load

_REASONS = {1: "pages run out (or do not fit the list they go back to)", 2: "a request is longer than its row of the block table, or shorter than what is to be kept",
            4: "more new tokens than rows", 8: "a negative length"}
_ATTENTION = {1: "a wait inside the attention ran out", 2: "a request had more new tokens than max_new"}


class PagedCacheError(RuntimeError):
    """A step that could not be made, more new tokens than were announced, or a wait inside the attention that ran out."""


@dataclass
class PagedBatch:
    """A step's new tokens, request behind request: request i has the rows cu_new[i] .. cu_new[i + 1] - 1, the rest stands behind them."""
    cu_new: torch.Tensor      # [requests + 1] int32
    slots: torch.Tensor       # [rows] int64: page * page_size + offset; -1 for rows without a token
    positions: torch.Tensor   # [rows] int32
    max_new: int              # no request has more


class PagedCache:
    def __init__(self, model, requests: int, max_len: int, pages: int, page: int = 64):
        """Room for `requests` requests of up to `max_len` tokens (rounded up to whole pages), in `pages` pages of `page` (16, 32, 64 or 128)
        positions that they share: `pages` bounds what all of them hold together."""
        if not model.kernels:
            raise ValueError("a paged cache is for the decode kernels: head_dim 128 and 1, 2, 4 or 8 query heads per KV head")
        if page not in (16, 32, 64, 128):
            raise ValueError(f"pages have 16, 32, 64 or 128 positions, got {page}")
        load()
        cfg, dev = model.cfg, model.dev
        self.page, self.pages, self.requests = page, pages, requests
        shape = (pages, model.hkv, page, cfg.head_dim)
        self.k = [[torch.empty(shape, device=dev, dtype=cfg.dtype) for _ in range(cfg.layers)] for _ in range(model.nlocal)]
        self.v = [[torch.empty(shape, device=dev, dtype=cfg.dtype) for _ in range(cfg.layers)] for _ in range(model.nlocal)]
        self.block_table = torch.full((requests, (max_len + page - 1) // page), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), pages, dtype=torch.int32, device=dev)
        self._said = torch.zeros(1, dtype=torch.int32, device=dev)  # all that extend and trim could not do
        # Scratch of the attention for steps of any size: a captured step goes on using it, so it never makes room for a larger one.
        device = dev.index if dev.index is not None else torch.cuda.current_device()
        self.max_len = self.block_table.shape[1] * page
        need = load().paged_attention_workspace_bytes(model.hq // model.hkv, max(1, min(self.max_len, 1 << 20)), device)
        self.workspace = torch.zeros(need, dtype=torch.uint8, device=dev)
        self.timeout_ms = 2000  # of one wait inside the attention

    def extend(self, new_lens: torch.Tensor, rows: int, max_new: Optional[int] = None) -> PagedBatch:
        """Room for new_lens[i] more tokens of request i ([requests] int32 on the GPU); `rows` is the size of the batch that they are the first
        rows of, `max_new` what no new_lens is above (as many as there are rows, if it is not known: a step of single tokens should say 1, as
        the attention has a faster kernel for requests of up to 16 (new token, query head) pairs a KV head)."""
        cu, slots, positions, status = torch.ops.b200ipc.paged_extend(self.block_table, self.lens, new_lens, self.free_pages, self.n_free, self.page, rows)
        self._said.bitwise_or_(status)
        return PagedBatch(cu, slots, positions, max(1, min(rows if max_new is None else max_new, rows, self.max_len)))

    def trim(self, keep_lens: torch.Tensor) -> None:
        """Request i keeps its first keep_lens[i] tokens; pages that are not needed for them are free again."""
        self._said.bitwise_or_(torch.ops.b200ipc.paged_trim(self.block_table, self.lens, keep_lens, self.free_pages, self.n_free, self.page))

    def check(self) -> None:
        """Raises what extend, trim or the attention found wrong since the last check.  Waits for the GPU."""
        said, attention = int(self._said), int(self.workspace[:4].view(torch.int32))
        if said:
            self._said.zero_()
        if attention:
            self.workspace.zero_()  # counters may have been left half way
        texts = [text for bit, text in _REASONS.items() if said & bit] + [text for bit, text in _ATTENTION.items() if attention & bit]
        if texts:
            raise PagedCacheError("; ".join(texts))
