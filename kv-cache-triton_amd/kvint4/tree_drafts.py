"""Trees of drafted tokens over a cache: what the contiguous and the paged cache share.

A tree's T tokens are appended like any block, attended with a mask that lets
each see the cached tokens, its ancestors and itself (``attend_tree``), and
then cut down to the path that verification accepted (``accept``). The
reference decodes one token at a time (models/llama3/llama3_quant.py:62-88).
"""

from __future__ import annotations

import contextlib
from typing import Optional, Sequence

import torch


def check_parents(parents: Sequence[int]) -> list[int]:
    """Parents of a tree's tokens as ints: each an earlier token's place, or -1
    (the token follows the cached ones)."""
    out = [int(p) for p in parents]
    for t, p in enumerate(out):
        if not -1 <= p < t:
            raise ValueError(f"parents[{t}] = {p}: a token's parent is an earlier token of the tree, or -1")
    return out


def tree_mask(parents: Sequence[int]) -> tuple[torch.Tensor, list[int]]:
    """(bool [T, T] mask of ancestors and selves, depth of each token) of a tree
    given by each token's parent, on the host."""
    parents = check_parents(parents)
    mask = torch.eye(len(parents), dtype=torch.bool)
    depth = [0] * len(parents)
    for t, p in enumerate(parents):
        if p >= 0:
            mask[t] |= mask[p]
            depth[t] = depth[p] + 1
    return mask, depth


def check_paths(paths: Sequence[Sequence[int]], B: int, block: int) -> list[list[int]]:
    """Accepted paths, one per sequence: ascending places in a block of `block` tokens."""
    if len(paths) != B:
        raise ValueError(f"accept needs a path for each of the {B} sequences (got {len(paths)})")
    out = [[int(i) for i in p] for p in paths]
    for p in out:
        if any(not 0 <= i < block for i in p) or any(a >= b for a, b in zip(p, p[1:])):
            raise ValueError(f"a path is ascending places in the block of {block} tokens (got {p})")
    return out


def path_index(paths: list[list[int]]) -> Optional[torch.Tensor]:
    """int32 [B, 1, n] places (-1 past a path's end, on the host), or None where no row has to move."""
    if all(p == list(range(len(p))) for p in paths):
        return None
    n = max(len(p) for p in paths)
    return torch.tensor([p + [-1] * (n - len(p)) for p in paths], dtype=torch.int32)[:, None]


class TreeDrafts:
    """Mixin: the mask that the swapped attention modules attend a tree with."""

    _tree_mask: Optional[torch.Tensor] = None

    @property
    def active_tree(self) -> Optional[torch.Tensor]:
        """The mask of the tree that forward passes run over now, or None."""
        return self._tree_mask

    @contextlib.contextmanager
    def tree(self, mask: torch.Tensor):
        """Inside it, a forward pass of T = mask.shape[-1] tokens through the
        swapped modules appends them and attends them as a tree (bool [T, T] or
        [B, T, T] on the cache's device)."""
        if mask.dtype != torch.bool or mask.dim() not in (2, 3) or mask.shape[-1] != mask.shape[-2]:
            raise ValueError("a tree's mask is bool [T, T] or [B, T, T]")
        if self._tree_mask is not None:
            raise RuntimeError("a tree is already active on this cache")
        self._tree_mask = mask
        try:
            yield self
        finally:
            self._tree_mask = None
