"""GPU: caches that evict, through the swapped models: nothing changes until the budget is passed; then each KV head keeps
the sinks, the recent rows and the heaviest others, bit for bit, and tokens go on at their true positions."""

from __future__ import annotations

import pytest
import torch
from transformers import GPT2Config, GPT2LMHeadModel, LlamaConfig, LlamaForCausalLM

from kvint4.gpt2.gpt2_quant import replace_gpt2_attention_with_quantized
from kvint4.gpt2.kv_cache import EvictingQuantizedKVCache as GPT2Evicting, QuantizedKVCache as GPT2Cache
from kvint4.llama3.graph_decode import GraphedGreedyDecoder
from kvint4.llama3.kv_cache import EvictingQuantizedKVCache, QuantizedKVCache
from kvint4.llama3.llama3_quant import replace_llama_attention_with_quantized
from kvint4.storage import load_cache, save_cache

from _block_ref import Reference, allowed, values

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _llama(dtype=torch.bfloat16):
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=256, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=2048)
    model = LlamaForCausalLM(cfg).to(DEV, dtype).eval()
    replace_llama_attention_with_quantized(model)
    return model


def _gpt2():
    torch.manual_seed(0)
    model = GPT2LMHeadModel(GPT2Config(vocab_size=256, n_positions=1024, n_embd=128, n_layer=2, n_head=2)).to(DEV).eval()
    replace_gpt2_attention_with_quantized(model)
    return model


@pytest.mark.parametrize("family", ["llama-bf16", "llama-f32", "gpt2-f32"])
def test_below_the_budget_nothing_changes(family):
    model = _gpt2() if family == "gpt2-f32" else _llama(torch.float32 if family == "llama-f32" else torch.bfloat16)
    plain = GPT2Cache() if family == "gpt2-f32" else QuantizedKVCache()
    cache = (GPT2Evicting if family == "gpt2-f32" else EvictingQuantizedKVCache)(budget=100, slack=28)
    ids = torch.randint(0, 256, (2, 100), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        a = model(input_ids=ids, past_key_values=plain, use_cache=True).logits[:, -1:]
        b = model(input_ids=ids, past_key_values=cache, use_cache=True).logits[:, -1:]
        for _ in range(10):
            size = float(a.float().abs().max())
            # two layers' activations rounded a dozen times each; fp32: the two kernels' sums
            tol = size * (24 * 2.0 ** -8 if family == "llama-bf16" else 2.0 ** -12)
            assert float((a.float() - b.float()).abs().max()) <= tol
            tok = a[:, -1].argmax(-1, keepdim=True)
            a = model(input_ids=tok, past_key_values=plain, use_cache=True).logits
            b = model(input_ids=tok, past_key_values=cache, use_cache=True).logits
    assert cache.evictions == 0 and cache.get_seq_length() == 110 == cache.stored_rows()
    # every row of every query head spread a weight of 1
    per = model.config.num_attention_heads // cache.key_weights(0).shape[1]
    total = cache.key_weights(0).double().sum(-1)
    assert float((total - 110 * per).abs().max()) <= 110 * per * 2.0 ** -14


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_an_eviction_keeps_the_heaviest_rows(dtype):
    """Attention over the evicted cache is attention over the rows that the weights name, computed apart."""
    g = torch.Generator().manual_seed(2)
    B, Hq, Hkv, D, S = 2, 8, 2, 64, 700
    rnd = lambda h, n: torch.randn(B, h, n, D, generator=g).to(dtype).to(DEV)  # noqa: E731
    k, v, q = rnd(Hkv, S), rnd(Hkv, S), rnd(Hq, S)
    cache = EvictingQuantizedKVCache(budget=200, recent=64, sink=4, slack=32)
    cache.append(k, v, 0)
    before = [t.clone() for t in cache.get_quantized(0)]
    cache.attend(q, 0, n_kv_heads=Hkv, scale=0.3, is_causal=True)
    assert cache.evictions == 1 and cache.stored_rows() == 200 and cache.get_seq_length() == S
    kf, vf = values(before[0], before[1], 32, D), values(before[2], before[3], 32, D)
    ref = Reference(q, kf, vf, allowed("causal", [S] * B, S, S, None, DEV), 0.3)
    # the kept rows: found from the stored bytes; weights equal the reference's within their bound
    kept = cache.get_quantized(0)
    w = cache.key_weights(0)
    for b in range(B):
        for h in range(Hkv):
            same = (kept[0][b, h, :, None] == before[0][b, h, None]).all(-1) & (kept[3][b, h, :, None] == before[3][b, h, None]).all(-1)
            assert bool((same.sum(-1) == 1).all())
            rows = same.int().argmax(-1)
            assert bool((rows[1:] > rows[:-1]).all())
            assert rows[:4].tolist() == [0, 1, 2, 3] and rows[-64:].tolist() == list(range(S - 64, S))
            tol = ref.weight_tolerance(Hq // Hkv * S, torch.zeros_like(ref.weights))[b, h]
            assert bool(((w[b, h].double() - ref.weights[b, h, rows]).abs() <= tol[rows]).all())
            out = torch.ones(S, dtype=torch.bool, device=DEV)
            out[rows] = False
            # no dropped row is heavier than a kept one that was free to go, beyond the bound
            free = rows[4:-64]
            assert float(ref.weights[b, h][out].max()) <= float((ref.weights[b, h, free] + 2 * tol[free]).min())
    # decoding goes on over the kept rows and the new ones
    nk, nv, nq = rnd(Hkv, 1), rnd(Hkv, 1), rnd(Hq, 1)
    got = cache.append_and_attend(nq, nk, nv, 0, n_kv_heads=Hkv, scale=0.3)
    assert cache.stored_rows() == 201 and cache.get_seq_length() == S + 1
    parts = cache.get_quantized(0)
    ref = Reference(nq, values(parts[0], parts[1], 32, D), values(parts[2], parts[3], 32, D),
                    torch.ones(B, 1, 201, dtype=torch.bool, device=DEV), 0.3)
    assert bool(((got.double() - ref.out).abs() <= ref.tolerance(dtype, 0.0 if dtype == torch.float32 else 2.0 ** -11)).all())


def test_a_model_decodes_past_its_budget():
    """generate() with a small budget: tokens come out, positions go on, rows stay within budget and slack."""
    model = _llama()
    ids = torch.randint(0, 256, (2, 300), generator=torch.Generator().manual_seed(3)).to(DEV)
    cache = EvictingQuantizedKVCache(budget=64, slack=16)
    # (no padding among them, also where a token is the pad token's: generate() would make a mask of those)
    kw = dict(input_ids=ids, attention_mask=torch.ones_like(ids), do_sample=False, pad_token_id=0)
    out = model.generate(past_key_values=cache, max_new_tokens=60, **kw)
    assert out.shape == (2, 360)
    assert cache.get_seq_length() == 359 and cache.evictions >= 2 * 4
    assert all(64 <= cache.stored_rows(i) <= 80 for i in range(2))
    full = QuantizedKVCache()
    model.generate(past_key_values=full, max_new_tokens=2, **kw)
    assert cache.capacity_nbytes() < full.capacity_nbytes()


def test_edits_of_the_batch_and_the_length():
    g = torch.Generator().manual_seed(4)
    B, H, D = 3, 2, 64
    rnd = lambda n, h=H: torch.randn(B, h, n, D, generator=g).bfloat16().to(DEV)  # noqa: E731
    cache = EvictingQuantizedKVCache(budget=50, recent=20, sink=2, slack=10)
    cache.append(rnd(90), rnd(90), 0)
    cache.attend(rnd(90, 4), 0, n_kv_heads=H, scale=0.1, is_causal=True)
    assert cache.stored_rows() == 50
    w, rows = cache.key_weights(0).clone(), [t.clone() for t in cache.get_quantized(0)]
    cache.reorder_cache(torch.tensor([2, 0, 0], device=DEV))
    for got, old in zip((cache.key_weights(0), *cache.get_quantized(0)), (w, *rows)):
        assert torch.equal(got, old[[2, 0, 0]])
    with pytest.raises(ValueError, match="eviction"):
        cache.crop(-21)
    cache.crop(-20)
    assert cache.get_seq_length() == 70 and cache.stored_rows() == 30
    assert torch.equal(cache.key_weights(0), w[[2, 0, 0]][:, :, :30])
    cache.append(rnd(3), rnd(3), 0)
    assert bool((cache.key_weights(0)[:, :, 30:] == 0).all()) and cache.get_mask_sizes(2, 0) == (35, 40)
    cache.crop(72)
    assert cache.get_seq_length() == 72 and cache.stored_rows() == 32
    cache.batch_select_indices(torch.tensor([1], device=DEV))
    assert cache.key_weights(0).shape == (1, H, 32)
    cache.reset()
    assert cache.get_seq_length() == 0 and len(cache) == 0


def test_what_it_refuses(tmp_path):
    model = _llama()
    ids = torch.randint(0, 256, (2, 40), generator=torch.Generator().manual_seed(5)).to(DEV)
    cache = EvictingQuantizedKVCache(budget=32)
    mask = torch.ones(2, 40, dtype=torch.int64, device=DEV)
    mask[0, :7] = 0
    with torch.no_grad(), pytest.raises(ValueError, match="mask"):
        model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True)
    cache = EvictingQuantizedKVCache(budget=32)
    with torch.no_grad():
        tok = model(input_ids=ids, past_key_values=cache, use_cache=True).logits[:, -1].argmax(-1, keepdim=True)
    with pytest.raises(ValueError, match="captured"):
        GraphedGreedyDecoder(model, cache, tok, 4)
    with pytest.raises(ValueError, match="saved"):
        save_cache(cache, str(tmp_path / "x"))
    plain = QuantizedKVCache()
    with torch.no_grad():
        model(input_ids=ids, past_key_values=plain, use_cache=True)
    save_cache(plain, str(tmp_path / "y"))
    with pytest.raises(ValueError, match="loaded"):
        load_cache(str(tmp_path / "y"), EvictingQuantizedKVCache(budget=32))
