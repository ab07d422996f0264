"""GPU: softmax weights summed per cached key, alone and beside the attention, against a 64-bit restatement: one token,
chunks and whole prompts, every dtype and head layout, lengths of zero and one, strided sums, repeated calls, graphs."""

from __future__ import annotations

import math

import pytest
import torch

from _block_ref import Reference, allowed, random_cache, values
from kvint4 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

SHAPES = [
    # q, scales, B, Hq, Hkv, D, G, lens, Sq, causal
    ("bf16", "bf16", 1, 32, 8, 128, 32, [517], 1, False),
    ("bf16", "bf16", 3, 64, 8, 128, 32, [1, 64, 300], 1, False),
    ("f16", "f16", 4, 25, 25, 64, 32, [33, 0, 500, 128], 1, False),
    ("bf16", "bf16", 1, 8, 2, 128, 128, [4097], 1, False),
    ("bf16", "f16", 1, 4, 2, 128, 64, [222], 1, False),
    ("f16", "bf16", 1, 4, 2, 64, 64, [222], 1, False),
    ("f16", "f16", 1, 32, 1, 128, 32, [700], 1, False),
    ("bf16", "bf16", 2, 12, 4, 128, 32, [100, 41], 1, False),
    ("f32", "f16", 1, 12, 12, 64, 32, [300], 1, False),
    ("bf16", "bf16", 1, 8, 2, 128, 32, [300], 300, True),
    ("bf16", "bf16", 1, 8, 2, 64, 32, [257], 257, True),
    ("f16", "f16", 1, 8, 8, 128, 64, [1000], 130, True),
    ("bf16", "bf16", 2, 8, 4, 128, 32, [600, 600], 37, True),
    ("bf16", "bf16", 2, 8, 4, 128, 32, [600, 90], 37, True),
    ("bf16", "bf16", 1, 20, 4, 128, 32, [513], 513, True),
    ("bf16", "bf16", 1, 8, 2, 128, 32, [200], 64, False),
    ("f32", "f32", 1, 4, 2, 64, 32, [150], 40, True),
    ("bf16", "bf16", 1, 4, 2, 96, 32, [150], 40, True),
    ("f16", "f16", 1, 2, 2, 37, 5, [90], 20, True),
    ("bf16", "bf16", 2, 8, 2, 128, 32, [20, 3], 33, True),
]


def _case(shape, seed=None):
    q_dt, s_dt, B, Hq, Hkv, D, G, lens, Sq, causal = shape
    g = torch.Generator().manual_seed(sum(map(ord, str(shape))) if seed is None else seed)
    S = max(lens) + (2 if len(set(lens)) > 1 else 0)
    kp, ks = random_cache(B, Hkv, S, D, G, DT[s_dt], g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, DT[s_dt], g, DEV)
    q = torch.randn(B, Hq, Sq, D, generator=g).to(DT[q_dt]).to(DEV)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV) if len(set(lens)) > 1 else None
    before = torch.rand(B, Hkv, S + 5, generator=g).to(DEV) / max(S, 1)
    sm = D ** -0.5
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D),
                    allowed("causal" if causal else "none", lens, Sq, S, None, DEV), sm)
    kw = dict(n_kv_heads=Hkv, group_size=G, is_causal=causal, sm_scale=sm, seq_lens=sl)
    return q, (kp, ks, vp, vs), before, ref, kw, S


def _check_weights(got, before, ref, S, rows):
    assert torch.equal(got[:, :, S:], before[:, :, S:])
    err = (got[:, :, :S].double() - before[:, :, :S].double() - ref.weights).abs()
    tol = ref.weight_tolerance(rows, before[:, :, :S].double())
    assert bool((err <= tol).all()), f"error {float(err.max()):.3g}, {float((err / tol).max()):.2f} of its bound"
    idle = ref.weights == 0
    assert torch.equal(got[:, :, :S][idle], before[:, :, :S][idle])


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s).replace(" ", ""))
def test_weights_and_attention_match_64_bits(shape):
    q, cache, before, ref, kw, S = _case(shape)
    dt = q.dtype
    rows = q.shape[1] // kw["n_kv_heads"] * q.shape[2]
    w = before.clone()
    ops.add_key_weights(q, cache[0], cache[1], w, **kw)
    _check_weights(w, before, ref, S, rows)
    w = before.clone()
    out = ops.attention_with_key_weights(q, *cache, w, **kw)
    _check_weights(w, before, ref, S, rows)
    # attention: long blocks of 16-bit queries may take the prefill kernels, which round keys, values and weights to the
    # queries' type; a key off by half a step moves a score by at most that much of its reach
    exact = dt == torch.float32 or cache[1].dtype == torch.float32
    half = 0.0 if exact else torch.finfo(dt).eps / 2
    tol = ref.tolerance(dt, half) + 4 * half * ref.reach * ref.spread
    assert bool(((out.double() - ref.out).abs() <= tol).all())


def test_each_row_adds_one():
    """The sums of a call over the keys are the number of rows that attend any."""
    for shape in SHAPES[:10]:
        q, cache, before, ref, kw, S = _case(shape)
        w = torch.zeros_like(before)
        ops.add_key_weights(q, cache[0], cache[1], w, **kw)
        r = q.shape[1] // kw["n_kv_heads"]
        lens = kw["seq_lens"].tolist() if kw["seq_lens"] is not None else [S] * q.shape[0]
        for b, n in enumerate(lens):
            rows = r * min(q.shape[2], n) if kw["is_causal"] else (r * q.shape[2] if n else 0)
            # every row's weights sum to 1 within 4 d and their sums' roundings
            tol = rows * (4 * ref.score_error() + 2 * (S + rows + 16) * 2.0 ** -24)
            assert float((w[b].double().sum(-1) - rows).abs().max()) <= tol + 1e-12


@pytest.mark.parametrize("shape", [SHAPES[1], SHAPES[2], SHAPES[9], SHAPES[11]], ids=str)
def test_equal_calls_give_equal_bits_and_calls_add_up(shape):
    q, cache, before, ref, kw, S = _case(shape)
    a, b = before.clone(), before.clone()
    for w in (a, b):
        for _ in range(3):
            ops.attention_with_key_weights(q, *cache, w, **kw)
    assert torch.equal(a, b)
    rows = q.shape[1] // kw["n_kv_heads"] * q.shape[2]
    err = (a[:, :, :S].double() - before[:, :, :S] - 3 * ref.weights).abs()
    assert bool((err <= 3 * ref.weight_tolerance(rows, before[:, :, :S].double() + 2 * ref.weights)).all())


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[9], SHAPES[8]], ids=str)
def test_strided_sums_and_caches(shape):
    """Sums that are a slice of a larger buffer, every second entry, and a cache that is a narrowed, padded buffer."""
    q, cache, before, ref, kw, S = _case(shape)
    B, H = before.shape[:2]
    wide = torch.full((H, B, 2 * before.shape[2] + 1), 3.0, device=DEV)
    w = wide.transpose(0, 1)[:, :, 1::2]
    w.copy_(before)
    big = []
    for t in cache:
        buf = torch.zeros(B, H, S + 9, t.shape[3] + (t.shape[3] % 2 + 1), dtype=t.dtype, device=DEV)
        buf[:, :, 4:4 + S, :t.shape[3]] = t
        big.append(buf[:, :, 4:4 + S, :t.shape[3]])
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    ops.attention_with_key_weights(qt, *big, w, **kw)
    _check_weights(w.contiguous(), before, ref, S, q.shape[1] // H * q.shape[2])
    assert bool((wide[:, :, 0::2] == 3).all())


def test_what_lies_past_the_length_does_not_matter():
    for sq in (1, 40):
        q, cache, before, ref, kw, S = _case(("bf16", "bf16", 2, 8, 2, 128, 32, [130, 77], sq, sq > 1), 4)
        w1, w2 = before.clone(), before.clone()
        out1 = ops.attention_with_key_weights(q, *cache, w1, **kw)
        for b, n in enumerate((130, 77)):
            cache[1][b, :, n:], cache[3][b, :, n:] = math.nan, math.inf
        out2 = ops.attention_with_key_weights(q, *cache, w2, **kw)
        assert torch.equal(out1, out2) and torch.equal(w1, w2)


def test_large_scores_leave_one_key():
    """Scores so far apart that one key takes everything, and so large that 2^s overflows fp32."""
    for q_dt in ("bf16", "f32"):
        B, Hq, Hkv, D, G, S = 1, 8, 2, 128, 32, 300
        g = torch.Generator().manual_seed(3)
        kp, ks = random_cache(B, Hkv, S, D, G, DT[q_dt], g, DEV)
        q = torch.randn(B, Hq, 1, D, generator=g).to(DT[q_dt]).to(DEV) * 100
        w = torch.zeros(B, Hkv, S, device=DEV)
        ops.add_key_weights(q, kp, ks, w, n_kv_heads=Hkv, group_size=G, is_causal=False, sm_scale=1.0)
        k = values(kp, ks, G, D)
        best = torch.matmul(q.double().reshape(Hkv, 4, D), k[0].transpose(-1, -2).contiguous())
        for h in range(Hkv):
            s = best[h].sort(-1, descending=True)
            sure = s.values[:, 0] - s.values[:, 1] > 40
            assert sure.any()
            count = torch.zeros(S, device=DEV)
            for r in range(4):
                if sure[r]:
                    count[s.indices[r, 0]] += 1
            assert bool((w[0, h] >= count * (1 - 1e-6)).all()) and abs(float(w[0, h].sum()) - 4) < 1e-3


def test_graphs_replay_what_runs_eagerly():
    for shape in (SHAPES[0], SHAPES[9]):
        q, cache, before, ref, kw, S = _case(shape)
        w = before.clone()
        graph = torch.cuda.CUDAGraph()
        ops.attention_with_key_weights(q, *cache, w, **kw)
        with torch.cuda.graph(graph):
            out = ops.attention_with_key_weights(q, *cache, w, **kw)
        for _ in range(3):
            q.copy_(torch.randn(q.shape, device=DEV).to(q.dtype))
            w.copy_(before)
            graph.replay()
            got, sums = out.clone(), w.clone()
            w.copy_(before)
            want = ops.attention_with_key_weights(q, *cache, w, **kw)
            torch.cuda.synchronize()
            assert torch.equal(got, want) and torch.equal(sums, w)
