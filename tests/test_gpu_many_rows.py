"""GPU: trees and weighed blocks of many rows per KV head (the kernels whose workgroups share decoded tiles), against the
64-bit restatement: wide trees over ragged, paged, short and empty sequences, scales that fp16 operands cannot hold, and
infinities. Tolerances as in _block_ref."""

from __future__ import annotations

import math

import pytest
import torch

from _block_ref import Reference, allowed, random_cache, random_tree, values
from kvint4 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
STEP = 2.0 ** -11  # half a step of the fp16 weights and values


def _check(out, ref, dt):
    err, tol = (out.double() - ref.out).abs(), ref.tolerance(dt, STEP)
    assert bool((err <= tol).all()), f"error {float(err.max()):.3g}, {float((err / tol).max()):.2f} of its bound"


TREES = [
    # q, scales, B, Hq, Hkv, D, G, lens, T
    ("bf16", "bf16", 1, 8, 1, 128, 32, [900], 9),       # 72 rows
    ("bf16", "bf16", 1, 16, 2, 64, 32, [70], 16),       # 128 rows, a tree across two tiles
    ("bf16", "bf16", 3, 8, 2, 128, 64, [64, 330, 1], 65),
    ("f16", "f16", 2, 8, 2, 128, 32, [500, 129], 41),   # 164 rows
    ("f16", "f16", 1, 4, 1, 64, 64, [1000], 100),
    ("f16", "bf16", 1, 16, 1, 128, 128, [300], 20),     # 320 rows
    ("bf16", "f16", 1, 8, 1, 128, 64, [2500], 33),
    ("bf16", "bf16", 1, 2, 2, 128, 32, [200], 200),     # nothing but the tree
    ("bf16", "bf16", 2, 4, 1, 64, 64, [30, 0], 90),     # shorter than the tree, and empty
    ("bf16", "bf16", 1, 4, 4, 128, 32, [5000], 129),
]


def _tree(case, page=0):
    q_dt, s_dt, B, Hq, Hkv, D, G, lens, T = case
    g = torch.Generator().manual_seed(sum(map(ord, str(case))))
    S = max(max(lens), 1) + 2
    kp, ks = random_cache(B, Hkv, S, D, G, DT[s_dt], g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, DT[s_dt], g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).to(DT[q_dt]).to(DEV)
    mask = random_tree(T, g, B)
    return q, (kp, ks, vp, vs), mask, lens, S, dict(n_kv_heads=Hkv, group_size=G, sm_scale=D ** -0.5)


def _ref(q, cache, mask, lens, S, kw):
    G, D = kw["group_size"], q.shape[-1]
    keys = allowed("tree", lens, q.shape[2], S, mask, DEV)
    return Reference(q, values(*cache[:2], G, D), values(*cache[2:], G, D), keys, kw["sm_scale"])


@pytest.mark.parametrize("case", TREES, ids=lambda s: "-".join(str(x) for x in s).replace(" ", ""))
def test_wide_trees(case):
    q, cache, mask, lens, S, kw = _tree(case)
    mask[:, q.shape[2] // 2] = False  # a row that attends the prefix alone
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention(q, *cache, mask.to(DEV), seq_lens=sl, **kw)
    ref = _ref(q, cache, mask, lens, S, kw)
    _check(out, ref, q.dtype)
    empty = (ref.p.sum(-1) == 0)
    assert bool((out[empty] == 0).all())
    assert torch.equal(out, ops.tree_attention(q, *cache, mask.to(DEV), seq_lens=sl, **kw))


@pytest.mark.parametrize("page", [64, 128])
@pytest.mark.parametrize("case", [TREES[2], TREES[3], TREES[8]], ids=str)
def test_wide_trees_in_pages(case, page):
    """The pages of the same rows, shuffled: the same bits as the contiguous cache; a page without a block is not attended."""
    q, cache, mask, lens, S, kw = _tree(case)
    B, Hkv = q.shape[0], kw["n_kv_heads"]
    n_pages = -(-S // page)
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(B * n_pages + 1, generator=g)[:B * n_pages].reshape(B, n_pages)
    pools = []
    for t in cache:
        pool = torch.zeros(Hkv, (B * n_pages + 1) * page, t.shape[-1], dtype=t.dtype, device=DEV)
        for b in range(B):
            rows = (table[b].repeat_interleave(page) * page + torch.arange(page).repeat(n_pages))[:S].to(DEV)
            pool[:, rows] = t[b]
        pools.append(pool)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = ops.tree_attention(q, *cache, mask.to(DEV), seq_lens=sl, **kw)
    pt = ops.PageTable(table.int().to(DEV), page, B * n_pages + 1)
    got = ops.tree_attention_paged(q, *pools, pt, mask.to(DEV), seq_lens=sl, **kw)
    if S == n_pages * page or max(lens) <= S:
        _check(got, _ref(q, cache, mask, lens, S, kw), q.dtype)
    table[0, 0] = -1
    pt = ops.PageTable(table.int().to(DEV), page, B * n_pages + 1)
    got = ops.tree_attention_paged(q, *pools, pt, mask.to(DEV), seq_lens=sl, **kw)
    keys = allowed("tree", lens, q.shape[2], S, mask, DEV)
    keys[0, :, :page] = False
    G, D = kw["group_size"], q.shape[-1]
    _check(got, Reference(q, values(*cache[:2], G, D), values(*cache[2:], G, D), keys, kw["sm_scale"]), q.dtype)
    assert torch.isfinite(want.float()).all()


# powers of two of the scales of (the first tile, keys 100 .. 139, one group of keys 200 .. 219)
FAR = {"small among large": (0, -22, -40), "large after small": (-30, 0, 8), "beyond fp16": (20, -4, 30), "tiny": (-70, -90, -60)}


@pytest.mark.parametrize("far", FAR, ids=str)
@pytest.mark.parametrize("which", ["keys", "values"])
def test_scales_far_apart(far, which):
    """bf16 scales that no common power of two brings into fp16: those keys' scores, and those values, in fp32."""
    q, cache, mask, lens, S, kw = _tree(("bf16", "bf16", 1, 8, 2, 128, 32, [400], 33))
    a, b, c = FAR[far]
    s = cache[1 if which == "keys" else 3]
    f = s.float() * 2.0 ** a
    f[:, :, 100:140] = s[:, :, 100:140].float() * 2.0 ** b
    f[:, :, 200:220, 1] = s[:, :, 200:220, 1].float() * 2.0 ** c
    s.copy_(f)
    kw["sm_scale"] = 2.0 ** -max(a, b, c, 0) * 0.1 if which == "keys" else 0.1
    out = ops.tree_attention(q, *cache, mask.to(DEV), **kw)
    _check(out, _ref(q, cache, mask, [S], S, kw), q.dtype)


@pytest.mark.parametrize("case", [TREES[2], TREES[3]], ids=str)
def test_infinities_stay_where_they_are_attended(case):
    q, cache, mask, lens, S, kw = _tree(case)
    ref = _ref(q, cache, mask, lens, S, kw)
    T = q.shape[2]
    bad = T - 1  # the last draft, that only its own row attends
    mask[:, :, bad] = False
    mask[:, bad, bad] = True
    ref = _ref(q, cache, mask, lens, S, kw)
    for b, n in enumerate(lens):
        for t, v in zip(cache[1::2], (math.nan, math.inf)):
            t[b, :, n:] = v
            if n:
                t[b, :, n - 1] = v
    q[:, :, 2, 5] = math.inf  # and a row of its own that is not finite
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention(q, *cache, mask.to(DEV), seq_lens=sl, **kw)
    rows = [i for i in range(T) if i not in (2, bad)]
    err, tol = (out.double() - ref.out).abs()[:, :, rows], ref.tolerance(q.dtype, STEP)[:, :, rows]
    assert bool((err <= tol).all())


@pytest.mark.parametrize("sm", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("s_dt", ["bf16", "f16"])
def test_scales_of_the_scores(sm, s_dt):
    q, cache, mask, lens, S, kw = _tree((s_dt, s_dt, 1, 8, 2, 128, 64, [333], 37))
    kw["sm_scale"] = sm
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention(q, *cache, mask.to(DEV), seq_lens=sl, **kw)
    _check(out, _ref(q, cache, mask, lens, S, kw), q.dtype)


@pytest.mark.parametrize("s_dt,D,causal,Sq,S", [("bf16", 128, True, 260, 700), ("f16", 128, True, 129, 129),
                                                ("bf16", 64, False, 70, 520), ("f16", 64, False, 33, 64),
                                                ("bf16", 128, True, 1200, 1200)])
def test_weighed_blocks(s_dt, D, causal, Sq, S):
    """Attention with its weights, and the weights alone: both within the bounds, with scales far apart and a key that is
    not finite at the end, which the causal mask hides from all rows but the last."""
    g = torch.Generator().manual_seed(Sq)
    B, Hq, Hkv, G, dt = 1, 8, 2, 32, DT[s_dt]
    cache = [t for _ in range(2) for t in random_cache(B, Hkv, S, D, G, dt, g, DEV)]
    cache[1][:, :, 5:9] *= 2.0 ** -6
    cache[1][:, :, 9, 0] = 0.0
    q = torch.randn(B, Hq, Sq, D, generator=g).to(dt).to(DEV)
    kw = dict(n_kv_heads=Hkv, group_size=G, is_causal=causal, sm_scale=D ** -0.5)
    ref = Reference(q, values(*cache[:2], G, D), values(*cache[2:], G, D),
                    allowed("causal" if causal else "none", [S], Sq, S, None, DEV), kw["sm_scale"])
    before = torch.rand(B, Hkv, S, generator=g).to(DEV)
    for with_out in (False, True):
        w = before.clone()
        if with_out:
            out = ops.attention_with_key_weights(q, *cache, w, **kw)
            _check(out, ref, dt)
        else:
            ops.add_key_weights(q, cache[0], cache[1], w, **kw)
        err = (w.double() - before.double() - ref.weights).abs()
        assert bool((err <= ref.weight_tolerance(Hq // Hkv * Sq, before.double())).all())
    if causal:  # the last key's scale is not a number: its score weighs nothing, and other keys keep theirs
        cache[1][:, :, -1] = math.nan
        keys = allowed("causal", [S], Sq, S, None, DEV)
        keys[:, :, -1] = False
        k = values(*cache[:2], G, D)
        k[:, :, -1] = 0.0
        ref = Reference(q, k, values(*cache[2:], G, D), keys, kw["sm_scale"])
        for with_out in (False, True):
            w = before.clone()
            if with_out:
                out = ops.attention_with_key_weights(q, *cache, w, **kw)
                _check(out, ref, dt)
            else:
                ops.add_key_weights(q, cache[0], cache[1], w, **kw)
            err = (w.double() - before.double() - ref.weights).abs()
            assert bool((err <= ref.weight_tolerance(Hq // Hkv * Sq, before.double())).all())


def test_two_graphs_of_wide_blocks_share_no_workspace():
    """Two captured calls replayed in turn, with eager ones between, give the eager bits."""
    a = _tree(TREES[9])
    b = _tree(TREES[3])
    runs = []
    for q, cache, mask, lens, S, kw in (a, b):
        m, sl = mask.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
        out = torch.empty_like(q)
        run = lambda q=q, cache=cache, m=m, sl=sl, kw=kw, out=out: ops.tree_attention(q, *cache, m, seq_lens=sl, out=out, **kw)
        runs.append((run, out, run().clone()))
    torch.cuda.synchronize()
    graphs = []
    for run, out, want in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append(g)
    for _ in range(3):
        for (run, out, want), g in zip(runs, graphs):
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            out.zero_()
            run()
            assert torch.equal(out, want)


@pytest.mark.parametrize("s_dt", ["bf16", "f16"])
def test_rows_that_are_not_finite_leave_the_sums_of_others(s_dt):
    """A query of infinities and one of NaN: their blocks' other rows, and the weights of all, stay finite and bounded."""
    g = torch.Generator().manual_seed(9)
    B, Hq, Hkv, D, G, Sq, S, dt = 1, 4, 1, 128, 32, 40, 300, DT[s_dt]
    cache = [t for _ in range(2) for t in random_cache(B, Hkv, S, D, G, dt, g, DEV)]
    q = torch.randn(B, Hq, Sq, D, generator=g).to(dt).to(DEV)
    kw = dict(n_kv_heads=Hkv, group_size=G, is_causal=False, sm_scale=D ** -0.5)
    ref = Reference(q, values(*cache[:2], G, D), values(*cache[2:], G, D),
                    allowed("none", [S], Sq, S, None, DEV), kw["sm_scale"])
    q[:, 1, 7, 3] = math.inf
    q[:, 2, 30] = math.nan
    rows = [i for i in range(Sq) if i not in (7, 30)]
    fine = ref.p[:, :, rows].sum((1, 2))  # [B, S]: the finite rows' weights
    fine += ref.p[:, [0, 2, 3]][:, :, 7].sum(1) + ref.p[:, [0, 1, 3]][:, :, 30].sum(1)
    for with_out in (False, True):
        w = torch.zeros(B, Hkv, S, device=DEV)
        if with_out:
            out = ops.attention_with_key_weights(q, *cache, w, **kw)
            err, tol = (out.double() - ref.out).abs()[:, :, rows], ref.tolerance(dt, STEP)[:, :, rows]
            assert bool((err <= tol).all())
        else:
            ops.add_key_weights(q, cache[0], cache[1], w, **kw)
        assert torch.isfinite(w).all()
        more = w.double()[:, 0] - fine  # what the row of infinities adds: at most 1 in all, the row of NaN nothing
        slack = ref.weight_tolerance(Hq * Sq, torch.zeros_like(ref.weights))[:, 0]
        assert bool((more >= -slack).all()) and bool((more.sum(-1) <= 1 + slack.sum(-1) + 1e-6).all())


@pytest.mark.parametrize("far", FAR, ids=str)
def test_weights_of_scales_far_apart(far):
    g = torch.Generator().manual_seed(12)
    B, Hq, Hkv, D, G, Sq, S = 1, 8, 2, 128, 32, 50, 400
    cache = [t for _ in range(2) for t in random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)]
    q = torch.randn(B, Hq, Sq, D, generator=g).bfloat16().to(DEV)
    a, b, c = FAR[far]
    f = cache[1].float() * 2.0 ** a
    f[:, :, 100:140] = cache[1][:, :, 100:140].float() * 2.0 ** b
    f[:, :, 200:220, 1] = cache[1][:, :, 200:220, 1].float() * 2.0 ** c
    cache[1].copy_(f)
    kw = dict(n_kv_heads=Hkv, group_size=G, is_causal=True, sm_scale=2.0 ** -max(a, b, c, 0) * 0.1)
    ref = Reference(q, values(*cache[:2], G, D), values(*cache[2:], G, D), allowed("causal", [S], Sq, S, None, DEV),
                    kw["sm_scale"])
    for with_out in (False, True):
        w = torch.zeros(B, Hkv, S, device=DEV)
        if with_out:
            _check(ops.attention_with_key_weights(q, *cache, w, **kw), ref, q.dtype)
        else:
            ops.add_key_weights(q, cache[0], cache[1], w, **kw)
        err = (w.double() - ref.weights).abs()
        assert bool((err <= ref.weight_tolerance(Hq // Hkv * Sq, torch.zeros_like(ref.weights))).all())
