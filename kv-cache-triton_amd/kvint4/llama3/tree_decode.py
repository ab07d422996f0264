"""Greedy decoding of a Llama model that verifies a tree of drafted tokens per forward pass.

A draft tree starts at the last token that was decided (its root, whose K/V the
cache does not hold yet) and branches into guesses of what follows. One forward
pass runs all of them over the cache (``verify_tree``): each token attends the
cached ones, its ancestors and itself, at the position its depth gives it. The
greedy continuation is then followed through the tree (``greedy_paths``): from
the root, the child that holds the token the model would emit, as long as there
is one. The cache keeps that path's rows (``cache.accept``), and the tokens are
those of decoding one by one, up to the rounding of the attention kernels.

The reference decodes one token at a time (benchmarks/llama3/
run_llama3_benchmark.py); Hugging Face's assisted decoding verifies a chain.
"""

from __future__ import annotations

from typing import Callable, Sequence

import torch

from ..tree_drafts import check_parents, tree_mask
from .graph_decode import _no_mask_creation
from .llama3_quant import LlamaAttentionQuantized


def verify_tree(model, cache, tokens: torch.Tensor, parents: Sequence[int]) -> torch.Tensor:
    """Logits [B, T, vocab] of a tree of T tokens over the cache, which holds
    their rows afterwards (as its last T).

    model    a Llama causal LM with swapped attention modules
    cache    a QuantizedKVCache or PagedQuantizedKVCache with the prompt in it
    tokens   [B, T] int64 on the model's device: sequence b's tokens, one tree
             for the batch
    parents  T ints: the place of each token's parent in the tree, before its
             own, or -1 (it follows the cached tokens directly)
    """
    if not any(isinstance(m, LlamaAttentionQuantized) for m in model.modules()):
        raise ValueError("the model's attention modules are not LlamaAttentionQuantized "
                         "(call replace_llama_attention_with_quantized first)")
    if tokens.dim() != 2 or tokens.shape[1] != len(parents) or not len(parents):
        raise ValueError(f"tokens must be [B, T] for the tree's T = {len(parents)} tokens (got {tuple(tokens.shape)})")
    mask, depth = tree_mask(parents)
    dev = tokens.device
    start = cache.get_seq_lens(0)
    if start is None:
        start = torch.full((tokens.shape[0],), cache.get_seq_length(), dtype=torch.int64, device=dev)
    pos = start.to(torch.int64)[:, None] + torch.tensor(depth, dtype=torch.int64, device=dev)
    with torch.no_grad(), _no_mask_creation(model), cache.tree(mask.to(dev)):
        out = model(input_ids=tokens, position_ids=pos, past_key_values=cache, use_cache=True)
    return out.logits


def greedy_paths(choice: Sequence[Sequence[int]], tokens: Sequence[Sequence[int]],
                 parents: Sequence[int]) -> tuple[list[list[int]], list[int]]:
    """(accepted places of each sequence, the token that follows each) of a tree
    whose first token is its root. choice[b][t]: the model's token after tree
    token t (the argmax of its logits). Of two children with the same token
    the first is followed."""
    parents = check_parents(parents)
    if not parents or any(p < 0 for p in parents[1:]):
        raise ValueError("a draft tree has one root, its first token")
    children: dict[int, list[int]] = {}
    for t, p in enumerate(parents[1:], 1):
        children.setdefault(p, []).append(t)
    paths, after = [], []
    for pick, toks in zip(choice, tokens):
        at, path = 0, [0]
        while True:
            nxt = next((t for t in children.get(at, ()) if int(toks[t]) == int(pick[at])), None)
            if nxt is None:
                break
            path.append(nxt)
            at = nxt
        paths.append(path)
        after.append(int(pick[at]))
    return paths, after


def decode_with_drafts(model, cache, next_token: torch.Tensor,
                       propose: Callable[[list[int]], tuple[Sequence[int], Sequence[int]]],
                       max_new_tokens: int) -> list[int]:
    """Greedy tokens of one sequence, `max_new_tokens` of them.

    next_token  [1, 1]: the token after the prompt that the cache holds
    propose     called with the tokens decided so far (next_token first);
                returns (draft tokens, parents): the tree under the last of
                them, parents as places among the drafts, -1 for its children
    """
    if next_token.shape != (1, 1):
        raise ValueError("decode_with_drafts decodes one sequence (next_token [1, 1])")
    if int(max_new_tokens) < 1:
        raise ValueError("need max_new_tokens >= 1")
    decided = [int(next_token.item())]
    while len(decided) < max_new_tokens:
        drafts, up = propose(list(decided))
        up = check_parents(up)
        if len(drafts) != len(up):
            raise ValueError("propose must return a parent for every draft")
        toks = [decided[-1], *(int(t) for t in drafts)]
        parents = [-1, *(p + 1 for p in up)]
        logits = verify_tree(model, cache, torch.tensor([toks], dtype=torch.int64, device=next_token.device), parents)
        paths, after = greedy_paths(logits.argmax(-1).tolist(), [toks], parents)
        cache.accept(len(toks), paths)
        decided += [toks[t] for t in paths[0][1:]] + after
    return decided[:max_new_tokens]
