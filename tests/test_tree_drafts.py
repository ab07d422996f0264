"""Host logic of draft trees and of the evicting cache's settings, on the CPU."""

from __future__ import annotations

import pytest
import torch

from kvint4.gpt2.kv_cache import EvictingQuantizedKVCache as GPT2Evicting
from kvint4.llama3.kv_cache import EvictingQuantizedKVCache, QuantizedKVCache
from kvint4.llama3.tree_decode import decode_with_drafts, greedy_paths
from kvint4.paged_cache import PagedQuantizedKVCache
from kvint4.tree_drafts import check_paths, path_index, tree_mask


def test_mask_and_depth_of_a_tree():
    mask, depth = tree_mask([-1, 0, 0, 1, 1, -1, 4])
    want = {0: [0], 1: [0, 1], 2: [0, 2], 3: [0, 1, 3], 4: [0, 1, 4], 5: [5], 6: [0, 1, 4, 6]}
    assert depth == [0, 1, 1, 2, 2, 0, 3]
    for t, seen in want.items():
        assert mask[t].nonzero().flatten().tolist() == seen
    assert tree_mask([])[0].shape == (0, 0)


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 0, 5], [-2]])
def test_parents_must_come_first(parents):
    with pytest.raises(ValueError):
        tree_mask(parents)


def test_paths():
    assert check_paths([[0, 2], []], 2, 3) == [[0, 2], []]
    for bad in ([[0, 2]], [[0, 0], []], [[2, 1], []], [[0, 3], []], [[-1], []]):
        with pytest.raises(ValueError):
            check_paths(bad, 2, 3)
    assert path_index([[0, 1], [0], []]) is None
    assert path_index([[0, 2, 5], [1]]).tolist() == [[[0, 2, 5]], [[1, -1, -1]]]


def test_greedy_paths_follow_the_models_choice():
    #        0
    #      1   2
    #     3 4   5
    parents, tokens = [-1, 0, 0, 1, 1, 2], [[10, 11, 12, 13, 14, 15]]
    assert greedy_paths([[11, 14, 0, 0, 99, 0]], tokens, parents) == ([[0, 1, 4]], [99])
    assert greedy_paths([[12, 0, 77, 0, 0, 0]], tokens, parents) == ([[0, 2]], [77])
    assert greedy_paths([[50, 0, 0, 0, 0, 0]], tokens, parents) == ([[0]], [50])
    # equal siblings: the first; a batch: each its own path
    assert greedy_paths([[7, 1, 2], [8, 1, 2]], [[5, 7, 7], [5, 7, 8]], [-1, 0, 0]) == ([[0, 1], [0, 2]], [1, 2])
    with pytest.raises(ValueError):
        greedy_paths([[0, 0]], [[1, 2]], [-1, -1])


@pytest.mark.parametrize("cache", [QuantizedKVCache(), PagedQuantizedKVCache()], ids=["contiguous", "paged"])
def test_a_tree_is_active_once(cache):
    mask = tree_mask([-1, 0])[0]
    assert cache.active_tree is None
    with cache.tree(mask):
        assert cache.active_tree is mask
        with pytest.raises(RuntimeError):
            with cache.tree(mask):
                pass
    assert cache.active_tree is None
    for bad in (mask.float(), mask[0], torch.ones(2, 3, dtype=torch.bool)):
        with pytest.raises(ValueError):
            with cache.tree(bad):
                pass
    with pytest.raises(ValueError):
        cache.accept(1, [[0]])


@pytest.mark.parametrize("cls", [EvictingQuantizedKVCache, GPT2Evicting])
def test_evicting_settings(cls):
    c = cls(budget=100)
    assert (c.recent, c.sink, c.slack) == (50, 4, 64)
    c = cls(budget=1000, recent=998)
    assert (c.sink, c.slack) == (2, 250)
    for kw in (dict(budget=0), dict(budget=10, recent=11), dict(budget=10, recent=6, sink=5), dict(budget=10, slack=-1),
               dict(budget=10, sink=-1)):
        with pytest.raises(ValueError):
            cls(**kw)
    assert c.get_seq_length() == 0 and c.stored_rows() == 0 and c.get_mask_sizes(5, 0) == (5, 0)


def test_what_an_evicting_cache_refuses():
    c, z = EvictingQuantizedKVCache(budget=8), torch.zeros(1, 1, 1, 32)
    for call in (lambda: c.load_ragged(z, z, 0, torch.ones(1)), lambda: c.make_static(4), lambda: c.update(z, z, 0),
                 lambda: c.tree(torch.ones(1, 1, dtype=torch.bool)), lambda: c.accept(1, [[0]]),
                 lambda: c.attend_tree(z, 0, None)):
        with pytest.raises(ValueError):
            call()


def test_decode_with_drafts_arguments():
    with pytest.raises(ValueError):
        decode_with_drafts(None, None, torch.zeros(2, 1, dtype=torch.int64), None, 4)
    with pytest.raises(ValueError):
        decode_with_drafts(None, None, torch.zeros(1, 1, dtype=torch.int64), None, 0)
    assert decode_with_drafts(None, None, torch.tensor([[3]]), None, 1) == [3]
