"""GPU: trees of drafts through the caches and the swapped models, as they are used: append, attend, accept, go on.

The rows that stay after ``accept`` are bit for bit those of a cache that only ever saw the accepted tokens; logits of a
tree's tokens are those of decoding each path on its own, within the attention's bound; and greedy decoding with drafts
gives the tokens of plain greedy decoding (fp32 models, whose rounding does not decide between two tokens)."""

from __future__ import annotations

import pytest
import torch
from transformers import GPT2Config, GPT2LMHeadModel, LlamaConfig, LlamaForCausalLM

from kvint4.gpt2.gpt2_quant import replace_gpt2_attention_with_quantized
from kvint4.gpt2.kv_cache import QuantizedKVCache as GPT2Cache
from kvint4.llama3.graph_decode import _no_mask_creation
from kvint4.llama3.kv_cache import QuantizedKVCache
from kvint4.llama3.llama3_quant import replace_llama_attention_with_quantized
from kvint4.llama3.tree_decode import decode_with_drafts, verify_tree
from kvint4.paged_cache import PagedQuantizedKVCache
from kvint4.tree_drafts import tree_mask

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
H, D, LAYERS = 2, 64, 2


def _cache(kind):
    return QuantizedKVCache() if kind == "contiguous" else PagedQuantizedKVCache(page_size=int(kind.split("-")[1]))


def _rows(cache, layer, lens):
    parts = cache.get_quantized(layer)
    return [[p[b, :, :n].clone() for p in parts] for b, n in enumerate(lens)]


@pytest.mark.parametrize("kind", ["contiguous", "paged-16", "paged-64"])
@pytest.mark.parametrize("paths", [[[0, 2, 5], [0, 2, 5]], [[0, 1, 4, 6], [3]], [[0, 1], [0, 1]], [[], [6]],
                                   [[0, 1, 2, 3, 4, 5, 6]] * 2], ids=str)
def test_accept_keeps_the_accepted_rows(kind, paths):
    g = torch.Generator().manual_seed(1)
    B, S, T = 2, 61, 7
    kv = lambda n: torch.randn(B, H, n, D, generator=g).bfloat16().to(DEV)  # noqa: E731
    cache, plain = _cache(kind), [_cache(kind) for _ in range(B)]
    for layer in range(LAYERS):
        k, v, tk, tv, nk, nv = kv(S), kv(S), kv(T), kv(T), kv(2), kv(2)
        cache.append(k, v, layer)
        cache.append(tk, tv, layer)
        for b in range(B):
            at = torch.tensor(paths[b], dtype=torch.int64, device=DEV)
            plain[b].append(torch.cat([k[b:b + 1], tk[b:b + 1, :, at], nk[b:b + 1]], 2),
                            torch.cat([v[b:b + 1], tv[b:b + 1, :, at], nv[b:b + 1]], 2), layer)
        if layer == 0:
            later = {}
        later[layer] = (nk, nv)
    cache.accept(T, paths)
    for layer in range(LAYERS):
        cache.append(*later[layer], layer)
    lens = [S + len(p) + 2 for p in paths]
    for layer in range(LAYERS):
        sl = cache.get_seq_lens(layer)
        assert (sl.tolist() if sl is not None else [cache.get_seq_length(layer)] * B) == lens
        for b, parts in enumerate(_rows(cache, layer, lens)):
            for got, want in zip(parts, plain[b].get_quantized(layer)):
                assert torch.equal(got, want[0, :, :lens[b]])


def test_accept_copies_shared_pages():
    """Two beams share their parent's pages; one's accepted rows do not reach the other."""
    g = torch.Generator().manual_seed(2)
    cache = PagedQuantizedKVCache(page_size=64)
    kv = lambda: torch.randn(1, H, 70, D, generator=g).bfloat16().to(DEV)  # noqa: E731
    cache.append(kv(), kv(), 0)
    cache.batch_repeat_interleave(2)
    before = _rows(cache, 0, [70, 70])
    cache.accept(8, [[0, 5, 7], [0, 1, 2, 3, 4, 5, 6, 7]])
    a, b = _rows(cache, 0, [65, 70])
    at = torch.tensor([*range(63), 67, 69], device=DEV)
    for got, old in zip(a, before[0]):
        assert torch.equal(got, old[:, at])
    for got, old in zip(b, before[1]):
        assert torch.equal(got, old)


def test_ragged_sequences_accept_their_own():
    g = torch.Generator().manual_seed(3)
    kv = lambda n: torch.randn(3, H, n, D, generator=g).bfloat16().to(DEV)  # noqa: E731
    cache = QuantizedKVCache()
    k, v, tk, tv = kv(50), kv(50), kv(5), kv(5)
    lens = [50, 13, 31]
    cache.load_ragged(k, v, 0, torch.tensor(lens))
    cache.append(tk, tv, 0)
    paths = [[1, 3], [0, 2, 4], []]
    cache.accept(5, paths)
    want = [n + len(p) for n, p in zip(lens, paths)]
    assert cache.get_seq_lens(0).tolist() == want and cache.get_seq_length(0) >= max(want)
    for b, parts in enumerate(_rows(cache, 0, want)):
        one = QuantizedKVCache()
        at = torch.tensor(paths[b], dtype=torch.int64, device=DEV)
        one.append(torch.cat([k[b:b + 1, :, :lens[b]], tk[b:b + 1, :, at]], 2),
                   torch.cat([v[b:b + 1, :, :lens[b]], tv[b:b + 1, :, at]], 2), 0)
        for got, ref in zip(parts, one.get_quantized(0)):
            assert torch.equal(got, ref[0])


def _llama(dtype, head_dim=64):
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=256, hidden_size=4 * head_dim, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512)
    model = LlamaForCausalLM(cfg).to(DEV, dtype).eval()
    replace_llama_attention_with_quantized(model)
    return model


@pytest.mark.parametrize("kind", ["contiguous", "paged-64"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_a_tree_are_those_of_its_paths(kind, dtype):
    """fp32: within fp32's rounding of the layers; bf16: within a few bf16 steps of the logits' size (two layers, each
    rounding activations a dozen times at 2^-8)."""
    model = _llama(dtype)
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, 256, (2, 37), generator=g).to(DEV)
    tokens = torch.randint(0, 256, (2, 6), generator=g).to(DEV)
    parents = [-1, 0, 0, 1, 1, 2]
    cache = _cache(kind)
    with torch.no_grad():
        model(input_ids=prompt, past_key_values=cache, use_cache=True)
        got = verify_tree(model, cache, tokens, parents)
        for leaf, path in ((3, [0, 1, 3]), (4, [0, 1, 4]), (5, [0, 2, 5])):
            one = _cache(kind)
            model(input_ids=prompt, past_key_values=one, use_cache=True)
            for t in path:
                want = model(input_ids=tokens[:, t:t + 1], past_key_values=one, use_cache=True).logits[:, -1]
                size = float(want.float().abs().max())
                tol = size * (2.0 ** -12 if dtype == torch.float32 else 24 * 2.0 ** -8)
                assert float((want.float() - got[:, t].float()).abs().max()) <= tol, (leaf, t)


@pytest.mark.parametrize("kind", ["contiguous", "paged-64"])
def test_decoding_with_drafts_gives_the_greedy_tokens(kind):
    model = _llama(torch.float32)
    prompt = torch.randint(0, 256, (1, 20), generator=torch.Generator().manual_seed(5)).to(DEV)
    want, cache = [], _cache(kind)
    with torch.no_grad():
        tok = model(input_ids=prompt, past_key_values=cache, use_cache=True).logits[:, -1].argmax(-1, keepdim=True)
        for _ in range(24):
            want.append(int(tok))
            tok = model(input_ids=tok, past_key_values=cache, use_cache=True).logits[:, -1].argmax(-1, keepdim=True)
    sizes = []

    def propose(decided):
        """Right drafts on one branch and wrong ones beside it, sometimes none right, sometimes no drafts at all."""
        n = len(decided)
        true = want[n:n + 3]
        if n % 5 == 4:
            return [], []
        wrong = [(t + 1) % 256 for t in (true or [0])]
        if n % 4 == 3:
            return wrong, [-1] * len(wrong)
        drafts, up = [wrong[0]], [-1]
        for i, t in enumerate(true):
            drafts += [t, (t + 7) % 256]
            up += [-1 if i == 0 else len(drafts) - 4] * 2
        sizes.append(len(drafts))
        return drafts, up

    cache = _cache(kind)
    with torch.no_grad():
        tok = model(input_ids=prompt, past_key_values=cache, use_cache=True).logits[:, -1].argmax(-1, keepdim=True)
    assert decode_with_drafts(model, cache, tok, propose, 24) == want
    assert sizes


def test_gpt2_attends_trees():
    torch.manual_seed(0)
    cfg = GPT2Config(vocab_size=256, n_positions=128, n_embd=128, n_layer=2, n_head=2)
    model = GPT2LMHeadModel(cfg).to(DEV).eval()
    replace_gpt2_attention_with_quantized(model)
    g = torch.Generator().manual_seed(6)
    prompt, tokens = torch.randint(0, 256, (1, 30), generator=g).to(DEV), torch.randint(0, 256, (1, 4), generator=g).to(DEV)
    mask, depth = tree_mask([-1, 0, 0, 2])
    pos = 30 + torch.tensor([depth], device=DEV)
    cache = GPT2Cache()
    with torch.no_grad():
        model(input_ids=prompt, past_key_values=cache, use_cache=True)
        with _no_mask_creation(model), cache.tree(mask.to(DEV)):
            got = model(input_ids=tokens, position_ids=pos, past_key_values=cache, use_cache=True).logits
        one = GPT2Cache()
        model(input_ids=prompt, past_key_values=one, use_cache=True)
        for t in (0, 2, 3):
            want = model(input_ids=tokens[:, t:t + 1], past_key_values=one, use_cache=True).logits[:, -1]
            assert float((want - got[:, t]).abs().max()) <= float(want.abs().max()) * 2.0 ** -12
