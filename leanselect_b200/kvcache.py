"""A paged key/value cache in 8 bits for the host model's decode steps.

Pages of 64 tokens hold the keys and values of every KV head as e4m3 codes
with one power-of-two scale per (page, head).  All layers share the block
tables: layer ``i`` keeps its codes in its own arrays under the same page
numbers.  Planning (pages, slots, positions), the cache write and the
attention are :func:`ops.plan_pages`, :func:`ops.append_kv` and
:func:`ops.paged_attn`; this class holds their tensors and what the host knows
of them (every length and the pages taken), so that nothing is read back from
the device and running out of pages is an error on the host.
"""
from __future__ import annotations

from contextlib import contextmanager
from typing import Sequence

import torch

from . import ops
from ._native import LS_MAX_PLAN_BATCH, LS_PAGE_TOKENS


def _pages(n: int) -> int:
    return -(-n // LS_PAGE_TOKENS)


class PagedKVCache:
    """``num_pages`` pages shared by ``batch`` requests of up to ``max_tokens`` tokens each."""

    def __init__(self, num_layers: int, batch: int, max_tokens: int, num_pages: int,
                 num_kv_heads: int, head_dim: int = 128, device: torch.device | str = "cuda"):
        if not 1 <= batch <= LS_MAX_PLAN_BATCH:
            raise ValueError(f"batch must lie in [1, {LS_MAX_PLAN_BATCH}]")
        if num_layers < 1 or max_tokens < 1 or num_pages < 1 or num_kv_heads < 1:
            raise ValueError("layers, tokens, pages and heads must be positive")
        if head_dim != 128:
            raise ValueError("head_dim must be 128")
        self.device = torch.device(device)
        self.batch, self.max_tokens, self.num_pages = batch, max_tokens, num_pages
        shape = (num_pages, num_kv_heads, LS_PAGE_TOKENS, head_dim)

        def codes():
            return torch.empty(shape, dtype=torch.float8_e4m3fn, device=self.device)

        def scales():
            return torch.ones(shape[:2], dtype=torch.float32, device=self.device)

        self._layers = [(codes(), codes(), scales(), scales()) for _ in range(num_layers)]
        self.block_table = torch.full((batch, _pages(max_tokens)), -1, dtype=torch.int32,
                                      device=self.device)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=self.device)
        self.free_head = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.lengths = [0] * batch  # the host's copy of seq_lens
        self.taken = 0              # the host's copy of free_head
        self.rope_len = 0           # length the cached keys' rotary frequencies go by

    def layer(self, i: int):
        """``(k_pages, v_pages, k_scale, v_scale)`` of layer ``i``."""
        return self._layers[i]

    @property
    def max_seqlen(self) -> int:
        return max(self.lengths)

    def plan(self, new_lens: Sequence[int]) -> ops.PagePlan:
        """Make room for ``new_lens[b]`` more tokens of request ``b`` and return the step's plan.

        The cache's lengths include the new tokens from here on; every layer
        then writes them with :func:`ops.append_kv`.
        """
        new = [int(n) for n in new_lens]
        if len(new) != self.batch or min(new) < 0:
            raise ValueError("new_lens must hold one length (>= 0) per request")
        after = [c + n for c, n in zip(self.lengths, new)]
        if max(after) > self.max_tokens:
            raise ValueError(f"a request would exceed the cache's {self.max_tokens} tokens")
        taken = self.taken + sum(_pages(a) - _pages(c) for a, c in zip(after, self.lengths))
        if taken > self.num_pages:
            raise RuntimeError(f"the cache is out of pages: {taken} needed, {self.num_pages} held")
        lens = torch.tensor(new, dtype=torch.int32).to(self.device, non_blocking=True)
        plan = ops.plan_pages(self.seq_lens, lens, self.block_table, self.free_pages,
                              self.free_head, sum(new))
        self.seq_lens, self.free_head = plan.seq_lens, plan.free_head
        self.lengths, self.taken = after, taken
        return plan

    @contextmanager
    def step(self, new_lens: Sequence[int]):
        """:meth:`plan` for a step that may fail on its way through the layers.

        When the block raises, the cache holds the tokens it held before: lengths,
        pages and free list are taken back, rows already written lie behind the
        lengths, and the next plan takes the same pages.  What is not taken back:
        where a layer had written into a half-filled page before the step failed,
        that page's scale may have grown for the new rows, as it would have in a
        step that succeeds.  It stays, and older values below 2^-6 of it have been
        rounded again, by at most 2^-10 of the scale.  (Rows with infinities raise
        it to 2^48 and leave nothing of them: a caller that checks for those does
        so before the write.)
        """
        before = self.seq_lens, self.free_head, self.lengths, self.taken, self.rope_len
        try:
            yield self.plan(new_lens)
        except BaseException:
            self.seq_lens, self.free_head, self.lengths, self.taken, self.rope_len = before
            raise

    def release(self, request: int) -> None:
        """Forget a request: its pages go back to the free list."""
        pages = _pages(self.lengths[request])
        if pages:
            self.taken -= pages
            self.free_pages[self.taken:self.taken + pages] = self.block_table[request, :pages]
            self.free_head = self.free_head - pages
            self.block_table[request, :pages] = -1
        seq = self.seq_lens.clone()
        seq[request] = 0
        self.seq_lens = seq
        self.lengths[request] = 0
