"""Prompts and decode steps of the MHA and GQA modules over a ``PagedKVCache`` (no counterpart
in the reference, whose modules take contiguous caches only)."""

from __future__ import annotations

from typing import Sequence

import torch

from ..ops.attention_forward import fastest_flash_attn_forward
from ..ops.kv_cache import PagedKVCache


class PagedSteps:
    """For modules with ``_project(x) -> q, k, v``, ``rotary``, ``scale``, ``softcap``,
    ``sliding_window``, ``sink_tokens``, ``head_dim``, ``k_proj`` and ``o_proj``."""

    def _kv_heads(self) -> int:
        return self.k_proj.out_features // self.head_dim

    def _window(self) -> dict:
        """The window's arguments of the attention entry points."""
        sinks = {"sink_tokens": self.sink_tokens} if self.sink_tokens else {}
        return dict(sliding_window=self.sliding_window, **sinks)

    def new_paged_cache(self, max_pages: int, page_size: int = 64) -> PagedKVCache:
        w = self.k_proj.weight
        return PagedKVCache(max_pages=max_pages, page_size=page_size, num_heads=self._kv_heads(),
                            head_dim=self.head_dim, dtype=w.dtype, device=w.device)

    def prefill_with_cache(self, x: torch.Tensor, cache: PagedKVCache,
                           seq_ids: Sequence[int]) -> torch.Tensor:
        """``forward(x, causal=True)`` of the prompts of new sequences ``seq_ids`` (positions
        0 .. S - 1) that also stores their keys and values in ``cache``."""
        if any(cache.sequences.get(s, {"len": 0})["len"] for s in seq_ids):
            raise ValueError("prefill_with_cache starts new sequences (positions 0..S-1)")
        B, S, _ = x.shape
        q, k, v = self._project(x)
        if self.rotary is not None:
            q, k = self.rotary(q, k)
        cache.append_batch(seq_ids, k, v)
        attn, _ = fastest_flash_attn_forward(
            q, k, v, scale=self.scale, causal=True, softcap=self.softcap,
            num_kv_heads=self._kv_heads(), **self._window())
        return self.o_proj(attn.transpose(1, 2).contiguous().view(B, S, -1))

    def decode_step(self, x: torch.Tensor, cache: PagedKVCache, seq_ids: Sequence[int],
                    evict: bool = False) -> torch.Tensor:
        """One new token per sequence: x ``[B, 1, hidden]`` -> ``[B, 1, hidden]``, the causal
        forward of each whole sequence at its last position. The token's key (rotated) and
        value enter the cache in one launch, then all sequences decode in place. With ``evict``
        pages that the sliding window has left behind (and that hold no sink) are released."""
        B = x.size(0)
        if x.dim() != 3 or x.size(1) != 1 or len(seq_ids) != B:
            raise ValueError("decode_step takes x [B, 1, hidden] and one seq id per row")
        q, k, v = self._project(x)
        if self.rotary is None:
            cache.append_batch(seq_ids, k, v)
        else:
            q = cache.append_batch(seq_ids, k, v, q=q, rotary=self.rotary)
        attn, _ = cache.decode(q[:, :, 0], seq_ids, scale=self.scale, softcap=self.softcap,
                               **self._window())
        if evict and self.sliding_window is not None:
            for s in seq_ids:
                cache.evict(s, self.sliding_window, self.sink_tokens)
        return self.o_proj(attn.reshape(B, 1, -1))
