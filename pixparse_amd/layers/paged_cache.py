"""The key-value cache of a decoder in pages of a pool, for batches whose sequences have lengths of their own (next to the contiguous cache of
BartEngine.decode_begin, which the reference's past_key_values corresponds to: models/text_decoder_hf.py:47-78).

One page table and one vector of lengths serve all layers; every layer has a pool of its own, a page of which holds the rows of one head next to
each other (the layout that the attention kernel reads fastest).  A sequence takes as many pages as the positions it may reach.  With
``weights`` every position gathers the attention weight it is given, and ``evict`` cuts each sequence down to the heaviest."""
from typing import List, Optional, Sequence

import torch

from .. import ops
from ..ops import BF16, F32, HEAD_DIM


class PagedCache:
    def __init__(self, layers: int, positions: Sequence[int], kv_heads: int, device, page_size: int = 64, weights: bool = False):
        """positions: the most positions that each sequence will hold"""
        if page_size < 1 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f'page_size {page_size}: a power of two up to 4096')
        if not positions or min(positions) < 1:
            raise ValueError('positions: one or more for every sequence')
        self.page_size, self.kv_heads, self.positions = int(page_size), int(kv_heads), [int(p) for p in positions]
        need = [-(-p // page_size) for p in self.positions]
        host = torch.full((len(need), max(need)), -1, dtype=torch.int32)        # -1: no page; never followed, lengths stay below
        used = 0
        for b, n in enumerate(need):
            host[b, :n] = torch.arange(used, used + n, dtype=torch.int32)
            used += n
        self.table = host.to(device)
        self.lengths = torch.zeros(len(need), dtype=torch.int32, device=device)
        self._cut = torch.zeros_like(self.lengths)
        pool = lambda: torch.empty(used, kv_heads, page_size, HEAD_DIM, dtype=BF16, device=device).permute(0, 2, 1, 3)
        self.k: List[torch.Tensor] = [pool() for _ in range(layers)]
        self.v: List[torch.Tensor] = [pool() for _ in range(layers)]
        self.weights: List[Optional[torch.Tensor]] = [
            torch.zeros(len(need), kv_heads, max(need) * page_size, dtype=F32, device=device) if weights else None for _ in range(layers)]

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor) -> None:
        """rows k / v [B, T, kv_heads*64] to positions starts[b] + t, t < counts[b]; the caller sets `lengths`"""
        ops.paged_append(k, v, self.k[layer], self.v[layer], self.table, starts, counts, weights=self.weights[layer])

    def attend(self, layer: int, q, o, heads: int, scale: float, k_new=None, v_new=None) -> None:
        """one token of every sequence over its first `lengths` positions; k_new / v_new: the rows of the last of them"""
        ops.paged_attn_decode(q, self.k[layer], self.v[layer], self.table, self.lengths, o, heads, scale, k_new=k_new, v_new=v_new,
                              weights=self.weights[layer])

    def evict(self, budget: int, recent: int) -> None:
        """in every layer, per head: the `recent` last positions and the heaviest of the others stay, `budget` in all"""
        for k, v, w in zip(self.k, self.v, self.weights):
            if w is None:
                raise ValueError('this cache gathers no attention weights to evict by')
            ops.cache_evict(k, v, self.table, self.lengths, w, budget, recent, self._cut)
        self.lengths.copy_(self._cut)

    def freeze(self, positions: int) -> None:
        """from now on no sequence holds more than `positions`: the table ends there, and no more weights are gathered (the pools keep their size)"""
        self.table = self.table[:, :-(-positions // self.page_size)].contiguous()
        self.weights = [None] * len(self.weights)
