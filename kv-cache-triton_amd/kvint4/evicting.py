"""Caches that evict: of each KV head only the rows that drew most attention stay.

A layer's cache keeps, next to its rows, the softmax weights that every query
so far gave each row, summed over the KV head's query heads
(``ops.attention_with_key_weights``). When it holds more than ``budget +
slack`` rows, each KV head keeps ``budget`` of them: the first ``sink``, the
last ``recent``, and of the rest those of the greatest weight
(``ops.select_keys``, ``ops.move_rows``). Keys keep the positions they were
rotated to, so the tokens after an eviction continue the true count
(``get_seq_length`` reports the tokens seen, not the rows stored).

The reference's cache drops nothing (models/llama3/kv_cache.py:76-105). Family
classes: ``kvint4.llama3.kv_cache.EvictingQuantizedKVCache`` and the GPT-2 one.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .cache_base import _ROUND, _LayerQuantizedKV, _round_up


class EvictingKVCache:
    """Mixin before a QuantizedKVCache class.

    budget  rows per KV head that an eviction keeps
    recent  of them, the last ones, always kept (default: half the budget)
    sink    of them, the first ones, always kept (default: 4, or what is left)
    slack   rows over the budget that a layer may hold before it evicts
            (default: a quarter of the budget, at least 64)

    Every sequence of the batch has one length; forward passes take no
    attention mask (no padding), and the attention modules must be swapped.
    """

    def __init__(self, group_size: int = 32, reserve_tokens: int = 0, *, budget: int, recent: Optional[int] = None,
                 sink: Optional[int] = None, slack: Optional[int] = None):
        super().__init__(group_size, reserve_tokens)
        self.budget = int(budget)
        if self.budget < 1:
            raise ValueError("budget must be >= 1")
        self.recent = self.budget // 2 if recent is None else int(recent)
        self.sink = min(4, self.budget - self.recent) if sink is None else int(sink)
        self.slack = max(64, self.budget // 4) if slack is None else int(slack)
        if min(self.recent, self.sink, self.slack) < 0 or self.recent + self.sink > self.budget:
            raise ValueError(f"the budget ({self.budget}) must hold sink ({self.sink}) and recent ({self.recent}), "
                             f"and slack ({self.slack}) be >= 0")
        self._weights: dict[int, torch.Tensor] = {}  # fp32 [B, H_kv, capacity] of each layer
        self._seen: dict[int, int] = {}              # tokens seen by each layer
        self._fresh: dict[int, int] = {}             # of its last rows, how many are its last tokens
        self.evictions = 0

    # -- lengths ---------------------------------------------------------------
    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Tokens seen (the next token's position), not rows stored."""
        return self._seen.get(layer_idx, 0)

    def stored_rows(self, layer_idx: int = 0) -> int:
        layer = self._layers.get(layer_idx)
        return 0 if layer is None else layer.seq_len

    def get_mask_sizes(self, cache_position, layer_idx: int = 0) -> tuple[int, int]:
        """(rows a mask would cover, the position of the first): the stored
        rows count as the last positions before the new tokens."""
        q = cache_position
        if isinstance(q, torch.Tensor):
            q = int(q.item()) if q.dim() == 0 else int(q.shape[0])
        stored = self.stored_rows(layer_idx)
        return stored + int(q), self.get_seq_length(layer_idx) - stored

    def key_weights(self, layer_idx: int) -> torch.Tensor:
        """[B, H_kv, stored rows] view of a layer's summed weights."""
        return self._weights[layer_idx][:, :, :self.stored_rows(layer_idx)]

    def reset(self) -> None:
        super().reset()
        self._weights.clear()
        self._seen.clear()
        self._fresh.clear()

    # -- appends and attention ---------------------------------------------------
    def _append_quantized(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int) -> None:
        start = self.stored_rows(layer_idx)
        super()._append_quantized(key_states, value_states, layer_idx)
        layer = self._layers[layer_idx]
        B, H = layer.k_packed.shape[:2]
        w = self._weights.get(layer_idx)
        if w is None or w.shape[2] < layer.capacity:
            new = torch.zeros((B, H, layer.capacity), dtype=torch.float32, device=layer.k_packed.device)
            if w is not None:
                new[:, :, :start] = w[:, :, :start]
            self._weights[layer_idx] = new
        else:
            w[:, :, start:layer.seq_len] = 0  # (rows used before an eviction or a crop)
        S = int(key_states.shape[2])
        self._seen[layer_idx] = self._seen.get(layer_idx, 0) + S
        self._fresh[layer_idx] = self._fresh.get(layer_idx, 0) + S

    def attend(self, query_states: torch.Tensor, layer_idx: int, *, n_kv_heads: int, scale: float,
               is_causal: bool) -> torch.Tensor:
        """Attention of query_states [B, H_q, S_q, d] over the layer's rows, with
        their weights added to the sums; evicts where the layer is over."""
        kp, ks, vp, vs = self.get_quantized(layer_idx)
        out = ops.attention_with_key_weights(
            query_states, kp, ks, vp, vs, self.key_weights(layer_idx), n_kv_heads=n_kv_heads,
            group_size=self.group_size, is_causal=is_causal, sm_scale=scale)
        if self.stored_rows(layer_idx) > self.budget + self.slack:
            self.evict(layer_idx)
        return out

    def append_and_attend(self, query_states: torch.Tensor, key_states: torch.Tensor, value_states: torch.Tensor,
                          layer_idx: int, *, n_kv_heads: int, scale: float) -> Optional[torch.Tensor]:
        """One decode token: append, attend, and count its weights."""
        if query_states.shape[2] != 1 or key_states.shape[2] != 1 or not query_states.is_cuda:
            return None
        self.append(key_states, value_states, layer_idx)
        return self.attend(query_states, layer_idx, n_kv_heads=n_kv_heads, scale=scale, is_causal=False)

    def evict(self, layer_idx: int) -> None:
        """Cut a layer to `budget` rows per KV head now (nothing if it holds no
        more). The kept rows go to new buffers, so that a long prompt's memory
        is given back."""
        layer = self._layers[layer_idx]
        n = layer.seq_len
        if n <= self.budget:
            return
        w = self._weights[layer_idx]
        index = ops.select_keys(w, self.budget, recent=self.recent, sink=self.sink, seq_len=n)
        cap = _round_up(max(self.budget + self.slack + 1, self.reserve_tokens), _ROUND)
        src = (layer.k_packed, layer.k_scales, layer.v_packed, layer.v_scales, w)
        dst = [torch.empty((*t.shape[:2], cap, *t.shape[3:]), dtype=t.dtype, device=t.device) for t in src]
        ops.move_rows([t[:, :, :n] for t in src], index, out=dst)
        self._layers[layer_idx] = _LayerQuantizedKV(*dst[:4], self.budget)
        self._weights[layer_idx] = dst[4]
        self._fresh[layer_idx] = min(self._fresh[layer_idx], self.recent)
        self.evictions += 1

    # -- batch and length edits ---------------------------------------------------
    def _gather_batch(self, index: torch.Tensor) -> None:
        super()._gather_batch(index)
        for i, w in self._weights.items():
            self._weights[i] = w[index.to(w.device)].contiguous()

    def crop(self, max_length: int) -> None:
        """Drop the last tokens (HF ``Cache.crop``, counted in tokens seen).
        Only tokens that no eviction has reached can be dropped."""
        max_length = int(max_length)
        drops = {}
        for i, seen in self._seen.items():
            keep = max(seen + max_length, 0) if max_length < 0 else min(max_length, seen) if max_length else seen
            drops[i] = seen - keep
            if drops[i] > self._fresh[i]:
                raise ValueError(f"crop to {keep} tokens reaches behind layer {i}'s last eviction: of its last "
                                 f"{drops[i]} tokens only {self._fresh[i]} are all stored")
        for i, d in drops.items():
            self._layers[i].seq_len -= d
            self._seen[i] -= d
            self._fresh[i] -= d

    def tree(self, mask):
        raise ValueError("a cache that evicts does not take trees of drafts (their weights would count rejected tokens)")

    def attend_tree(self, *args, **kwargs):
        raise ValueError("a cache that evicts does not take trees of drafts")

    def accept(self, *args, **kwargs):
        raise ValueError("a cache that evicts does not take trees of drafts")

    def load_ragged(self, *args, **kwargs) -> None:
        raise ValueError("a cache that evicts holds sequences of one length (load_ragged)")

    def make_static(self, extra_tokens: int) -> None:
        raise ValueError("a cache that evicts cannot be captured: a replay would not evict")

    def update(self, *args, **kwargs):
        raise ValueError("a cache that evicts needs swapped attention modules (it counts the weights they compute)")

    def capacity_nbytes(self) -> int:
        return super().capacity_nbytes() + sum(w.element_size() * w.numel() for w in self._weights.values())
