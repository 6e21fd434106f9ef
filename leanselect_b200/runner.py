"""Public prefill entry point: host token ids in, last-token logits out.

``PrefillRunner`` owns a :class:`~leanselect_b200.model.PrefillModel` (or its
sequence-parallel form) and exposes the call a user makes:
``logits = runner(token_ids_on_host, lengths)`` copies the ids to the GPU,
runs the packed prefill and copies the logits back;
``runner.generate(token_ids_on_host, lengths, steps)`` continues the prompts.
"""
from __future__ import annotations

from typing import Sequence

import torch

from .kvcache import PagedKVCache
from .model import MiniCPMShape, PrefillModel


class PrefillRunner:
    def __init__(self, shape: MiniCPMShape, device: torch.device | str = "cuda", seed: int = 0,
                 model: PrefillModel | None = None):
        self.device = torch.device(device)
        self.model = model if model is not None else PrefillModel(shape, self.device, seed=seed)

    def prefill_device(self, ids: torch.Tensor, lengths: Sequence[int], timers=None,
                       key_counts=None, capture=None):
        """Prefill with ids already on the device; returns device logits ``[B, vocab]``."""
        lengths = [int(n) for n in lengths]
        cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(lengths).cumsum(0)
        cu = cu.to(self.device, non_blocking=True)
        return self.model.prefill(ids, cu, lengths, timers=timers, key_counts=key_counts,
                                  capture=capture)

    def __call__(self, ids_host: torch.Tensor, lengths: Sequence[int]) -> torch.Tensor:
        """Host ids (ideally pinned) -> host logits ``[B, vocab]`` fp32."""
        ids = ids_host.to(self.device, non_blocking=True)
        logits = self.prefill_device(ids, lengths)
        out = torch.empty(logits.shape, dtype=logits.dtype, pin_memory=True)
        out.copy_(logits, non_blocking=True)
        torch.cuda.current_stream(self.device).synchronize()
        return out

    def generate(self, ids_host: torch.Tensor, lengths: Sequence[int], steps: int) -> torch.Tensor:
        """Greedy continuation of packed prompts: host token ids ``[B, steps]``.

        The prompts are prefilled with LeanSelect into an 8-bit paged cache
        sized for them; each following token is a decode step over that cache.
        """
        lengths, steps = [int(n) for n in lengths], int(steps)
        if not lengths or min(lengths) < 1 or steps < 1:
            raise ValueError("generate needs non-empty prompts and at least one step")
        s = self.model.shape
        # The last token is returned, not fed back: steps - 1 tokens are cached.
        cache = PagedKVCache(s.num_layers, len(lengths), max(lengths) + steps - 1,
                             sum(-(-(n + steps - 1) // 64) for n in lengths), s.num_kv_heads,
                             s.head_dim, self.device)
        cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(lengths).cumsum(0)
        ids = ids_host.to(self.device, non_blocking=True)
        logits = self.model.prefill(ids, cu.to(self.device, non_blocking=True), lengths,
                                    cache=cache)
        out = [logits.argmax(-1)]
        for _ in range(steps - 1):
            out.append(self.model.decode(out[-1], cache).argmax(-1))
        return torch.stack(out, dim=1).cpu()
