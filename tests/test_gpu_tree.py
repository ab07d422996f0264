"""GPU: attention of trees of drafted tokens against a 64-bit restatement: every dtype and head layout, odd head dims and
groups, one draft to many, lengths from the block itself on, masks that leave rows empty, pages, strides, and what a
draft that is not attended may hold. Tolerances are derived in _block_ref.Reference.tolerance."""

from __future__ import annotations

import math

import pytest
import torch

from _block_ref import Reference, allowed, random_cache, random_tree, values
from kvint4 import _native as nat, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _step(q_dt, s_dt):
    """Half a step of the weights and values of the 16-bit kernel (fp16 operands); the exact kernel rounds neither."""
    return 0.0 if q_dt == "f32" or s_dt == "f32" else 2.0 ** -11


def _check(out, ref, dt, step):
    err = (out.double() - ref.out).abs()
    tol = ref.tolerance(dt, step)
    assert torch.isfinite(out.float()).all()
    assert bool((err <= tol).all()), f"error {float(err.max()):.3g}, {float((err / tol).max()):.2f} of its bound"


SHAPES = [
    # q, scales, B, Hq, Hkv, D, G, lens, T
    ("bf16", "bf16", 1, 32, 8, 128, 32, [517], 8),
    ("bf16", "bf16", 1, 8, 8, 128, 32, [64], 1),
    ("bf16", "bf16", 2, 8, 2, 128, 32, [1, 3], 1),
    ("bf16", "bf16", 3, 8, 2, 128, 64, [70, 200, 129], 17),
    ("f16", "f16", 2, 16, 2, 128, 128, [333, 90], 33),
    ("f16", "f16", 2, 25, 25, 64, 32, [300, 77], 13),
    ("bf16", "bf16", 1, 4, 1, 64, 64, [1025], 64),
    ("bf16", "bf16", 1, 2, 2, 64, 32, [128], 128),
    ("bf16", "f16", 1, 4, 2, 128, 32, [400], 9),
    ("f16", "bf16", 1, 4, 2, 128, 32, [400], 9),
    ("f16", "f16", 1, 64, 1, 128, 32, [260], 5),
    ("f16", "f16", 1, 12, 4, 64, 32, [100], 6),
    ("bf16", "bf16", 1, 20, 4, 128, 32, [3000], 27),
    ("bf16", "bf16", 1, 4, 2, 128, 32, [9000], 31),
    ("bf16", "bf16", 1, 8, 2, 96, 32, [150], 7),
    ("f16", "f16", 1, 3, 3, 80, 32, [150], 7),
    ("f32", "f16", 1, 12, 12, 64, 32, [600], 8),
    ("f32", "f32", 2, 4, 2, 128, 32, [257, 30], 5),
    ("bf16", "f32", 1, 4, 2, 64, 32, [120], 5),
    ("f32", "bf16", 1, 2, 1, 33, 7, [80], 9),
    ("bf16", "bf16", 1, 4, 1, 37, 5, [90], 4),
    ("f16", "f16", 1, 2, 2, 256, 64, [130], 3),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s).replace(" ", ""))
def test_tree_matches_64_bits(shape):
    q_dt, s_dt, B, Hq, Hkv, D, G, lens, T = shape
    g = torch.Generator().manual_seed(sum(map(ord, str(shape))))
    S = max(lens) + 3
    kp, ks = random_cache(B, Hkv, S, D, G, DT[s_dt], g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, DT[s_dt], g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).to(DT[q_dt]).to(DEV)
    mask = random_tree(T, g, B)
    sm = D ** -0.5
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention(q, kp, ks, vp, vs, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=sm, seq_lens=sl)
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), allowed("tree", lens, T, S, mask, DEV), sm)
    _check(out, ref, DT[q_dt], _step(q_dt, s_dt))


@pytest.mark.parametrize("q_dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens,T", [([6, 21, 200], 21), ([0, 1, 64], 4), ([3, 4, 5], 5)])
def test_rows_and_sequences_without_keys(q_dt, lens, T):
    """Rows whose mask is empty over an empty prefix give zeros; sequences shorter than the block hold its last rows."""
    g = torch.Generator().manual_seed(5)
    B, Hq, Hkv, D, G, S = len(lens), 8, 2, 128, 32, max(lens) + 1
    dt = DT[q_dt]
    kp, ks = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).to(dt).to(DEV)
    mask = random_tree(T, g)
    mask[T // 2] = False
    mask[:, 0] = False
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention(q, kp, ks, vp, vs, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=0.1, seq_lens=sl)
    keys = allowed("tree", lens, T, S, mask, DEV)
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), keys, 0.1)
    _check(out, ref, dt, _step(q_dt, q_dt))
    empty = ~keys.any(-1)
    assert empty.any() and bool((out.transpose(1, 2)[empty] == 0).all())


@pytest.mark.parametrize("q_dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_attended_does_not_matter(q_dt, D):
    """Rows past the lengths, and drafts outside a row's path, hold infinities and NaN; only their own rows see them."""
    g = torch.Generator().manual_seed(6)
    B, Hq, Hkv, G, T, lens = 2, 8, 2, 32, 12, [140, 77]
    S, dt = 150, DT[q_dt]
    kp, ks = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).to(dt).to(DEV)
    mask = random_tree(T, g)
    bad = [3, 7]
    keep = [i for i in range(T) if not mask[i, bad].any()]
    assert len(keep) >= 2
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), allowed("tree", lens, T, S, mask, DEV), 0.1)
    for b, n in enumerate(lens):
        ks[b, :, n:], vs[b, :, n:] = math.nan, math.inf
        ks[b, :, n - T + bad[0]], vs[b, :, n - T + bad[0]] = math.inf, math.nan
        ks[b, :, n - T + bad[1], 0], vs[b, :, n - T + bad[1], 1] = math.nan, -math.inf
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention(q, kp, ks, vp, vs, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=0.1, seq_lens=sl)
    err, tol = (out.double() - ref.out).abs()[:, :, keep], ref.tolerance(dt, _step(q_dt, q_dt))[:, :, keep]
    assert bool((err <= tol).all())  # (a NaN or an infinity is not)


@pytest.mark.parametrize("q_dt", ["bf16", "f16", "f32"])
def test_infinite_values_reach_the_rows_that_attend_them(q_dt):
    """A value of infinity (its scale overflowed) makes the attending rows' outputs infinite or NaN in its dims only."""
    g = torch.Generator().manual_seed(16)
    B, Hq, Hkv, D, G, T, S, dt = 1, 8, 2, 128, 32, 5, 150, DT[q_dt]
    kp, ks = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).to(dt).to(DEV)
    mask = torch.eye(T, dtype=torch.bool)
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), allowed("tree", [S], T, S, mask, DEV), 0.1)
    vs[0, :, S - T + 2, 1] = math.inf  # draft 2's own value, dims 32 .. 63
    out = ops.tree_attention(q, kp, ks, vp, vs, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=0.1)
    fine = torch.isfinite(out.float())
    assert not fine[:, :, 2, 32:64].any()
    fine[:, :, 2, 32:64] = True
    assert fine.all()
    err, tol = (out.double() - ref.out).abs(), ref.tolerance(dt, _step(q_dt, q_dt))
    ok = err <= tol
    ok[:, :, 2, 32:64] = True
    assert ok.all()


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("q_dt,D", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_paged_equals_64_bits(page, q_dt, D):
    g = torch.Generator().manual_seed(7)
    B, Hq, Hkv, G, T, lens = 3, 8, 2, 32, 11, [page + 5, 4 * page, 11]
    dt, sm = DT[q_dt], D ** -0.5
    need = [-(-n // page) for n in lens]
    blocks = sum(need) + 2
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
    order = torch.randperm(blocks, generator=g).int()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    kp, ks = (t[0] for t in random_cache(1, Hkv, blocks * page, D, G, dt, g, DEV))
    vp, vs = (t[0] for t in random_cache(1, Hkv, blocks * page, D, G, dt, g, DEV))
    q = torch.randn(B, Hq, T, D, generator=g).to(dt).to(DEV)
    mask = random_tree(T, g, B)
    table[1, 1] = -1        # a page without a block: not attended
    table[1, 2] = blocks    # nor one outside the pool
    pt = ops.PageTable(table.to(DEV), page, blocks)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.tree_attention_paged(q, kp, ks, vp, vs, pt, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=sm,
                                   seq_lens=sl)
    S = max(lens)
    t = torch.arange(S)
    page_of = table[:, t // page].long()
    rows = (page_of.clamp(0, blocks - 1) * page + t % page).to(DEV)
    keys = allowed("tree", lens, T, S, mask, DEV) & ((page_of >= 0) & (page_of < blocks))[:, None].to(DEV)
    k, v = (values(p[:, rows].transpose(0, 1), s[:, rows].transpose(0, 1), G, D) for p, s in ((kp, ks), (vp, vs)))
    ref = Reference(q, k, v, keys, sm)
    _check(out, ref, dt, _step(q_dt, q_dt))
    # one length for all, without device lengths
    n = 2 * page - 3
    if n >= T:
        table[1, 1], table[2, :2] = order[-1], order[-2:]
        pt = ops.PageTable(table.to(DEV), page, blocks)
        out = ops.tree_attention_paged(q, kp, ks, vp, vs, pt, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=sm,
                                       seq_len=n)
        t = torch.arange(n)
        rows = (table[:, t // page].long() * page + t % page).to(DEV)
        k, v = (values(p[:, rows].transpose(0, 1), s[:, rows].transpose(0, 1), G, D) for p, s in ((kp, ks), (vp, vs)))
        _check(out, Reference(q, k, v, allowed("tree", [n] * B, T, n, mask, DEV), sm), dt, _step(q_dt, q_dt))


@pytest.mark.parametrize("q_dt,D", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_strides_and_one_mask_for_the_batch(q_dt, D):
    """Queries and outputs [B, T, H, D] seen as [B, H, T, D], cache rows with padding at odd addresses, a mask that is a
    transposed view and shared: the same as the plain layout, within the bound."""
    g = torch.Generator().manual_seed(8)
    B, Hq, Hkv, G, T, S = 2, 8, 4, 32, 10, 203
    dt, sm = DT[q_dt], D ** -0.5
    q = torch.randn(B, T, Hq, D + 1, generator=g).to(dt).to(DEV)[..., 1:].transpose(1, 2)
    kp, ks = random_cache(B, Hkv, S, D, G, dt, g, DEV, pad=3)
    vp, vs = random_cache(B, Hkv, S, D, G, dt, g, DEV, pad=5)
    mask = random_tree(T, g)
    mt = mask.T.contiguous().to(DEV).T
    out = torch.full((B, T, Hq, D + 3), 7.0, dtype=dt, device=DEV)
    view = out[..., 3:].transpose(1, 2)
    got = ops.tree_attention(q, kp, ks, vp, vs, mt, n_kv_heads=Hkv, group_size=G, sm_scale=sm, out=view)
    assert got.data_ptr() == view.data_ptr() and bool((out[..., :3] == 7).all())
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), allowed("tree", [S] * B, T, S, mask, DEV), sm)
    _check(got, ref, dt, _step(q_dt, q_dt))


@pytest.mark.parametrize("sm", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("q_dt", ["bf16", "f32"])
def test_scales_of_the_scores(sm, q_dt):
    """A zero scale weighs every key alike, a negative one turns the order, a large one leaves few keys."""
    g = torch.Generator().manual_seed(9)
    B, Hq, Hkv, D, G, T, S, dt = 1, 8, 2, 128, 32, 9, 700, DT[q_dt]
    kp, ks = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, dt, g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).to(dt).to(DEV)
    mask = random_tree(T, g)
    out = ops.tree_attention(q, kp, ks, vp, vs, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=sm)
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), allowed("tree", [S], T, S, mask, DEV), sm)
    _check(out, ref, dt, _step(q_dt, q_dt))


@pytest.mark.parametrize("big", [2.0 ** 20, 2.0 ** 100, 2.0 ** -20, 2.0 ** -60])
def test_value_scales_outside_fp16(big):
    """Value scales that fp16 operands cannot hold (bf16 caches): the rows' outputs keep their relative precision."""
    g = torch.Generator().manual_seed(10)
    B, Hq, Hkv, D, G, T, S = 1, 8, 2, 128, 32, 9, 300
    kp, ks = random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)
    vs = (vs.float() * big).bfloat16()
    vs[:, :, 100:160] = (vs[:, :, 100:160].float() / big).bfloat16()  # a tile of both kinds
    q = torch.randn(B, Hq, T, D, generator=g).bfloat16().to(DEV)
    mask = random_tree(T, g)
    out = ops.tree_attention(q, kp, ks, vp, vs, mask.to(DEV), n_kv_heads=Hkv, group_size=G, sm_scale=0.088)
    ref = Reference(q, values(kp, ks, G, D), values(vp, vs, G, D), allowed("tree", [S], T, S, mask, DEV), 0.088)
    # (fp16 operands take the scales times a power of two, and keys far from the others' scale in fp32: half a step 2^-11;
    # weights under 2^-14 are off by 2^-25, which the bound counts against the largest attended value)
    _check(out, ref, torch.bfloat16, 2.0 ** -11)


def test_matches_a_chain_of_single_steps():
    """A tree that is a chain gives what decoding its tokens one by one gives, within both routes' roundings."""
    g = torch.Generator().manual_seed(11)
    B, Hq, Hkv, D, G, T, S = 1, 32, 8, 128, 32, 6, 400
    kp, ks = random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).bfloat16().to(DEV)
    mask = torch.ones(T, T, dtype=torch.bool).tril().to(DEV)
    out = ops.tree_attention(q, kp, ks, vp, vs, mask, n_kv_heads=Hkv, group_size=G, sm_scale=0.088)
    for i in range(T):
        n = S - T + i + 1
        one = ops.fused_decode_attention(q[:, :, i:i + 1], kp[:, :, :n], ks[:, :, :n], vp[:, :, :n], vs[:, :, :n],
                                         n_kv_heads=Hkv, group_size=G, is_causal=False, sm_scale=0.088)
        # outputs of magnitude under 1: two bf16 roundings and the single step's bf16 weights (spread under 2)
        assert float((one.float() - out[:, :, i:i + 1].float()).abs().max()) <= 2 * 2.0 ** -8 + 2 * 2.0 ** -8


def test_another_stream_and_graph_replays():
    """On a side stream, and captured into a graph replayed on new inputs with eager work between, as eagerly."""
    g = torch.Generator().manual_seed(12)
    B, Hq, Hkv, D, G, T, S = 1, 32, 8, 128, 32, 16, 3000
    kp, ks = random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)
    vp, vs = random_cache(B, Hkv, S, D, G, torch.bfloat16, g, DEV)
    q = torch.randn(B, Hq, T, D, generator=g).bfloat16().to(DEV)
    mask = random_tree(T, g).to(DEV)
    run = lambda: ops.tree_attention(q, kp, ks, vp, vs, mask, n_kv_heads=Hkv, group_size=G, sm_scale=0.088)  # noqa: E731
    eager = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, run()))
    for k in range(4):
        q.copy_(torch.randn(B, Hq, T, D, generator=g).bfloat16())
        for graph, got in graphs:
            got.zero_()
            graph.replay()
        want = run()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert torch.equal(got, want), k


def test_empty_calls():
    z = torch.zeros
    for B, T in ((0, 4), (2, 0)):
        q = z(B, 8, T, 128, dtype=torch.bfloat16, device=DEV)
        c, s = z(B, 2, 5, 64, dtype=torch.uint8, device=DEV), z(B, 2, 5, 4, dtype=torch.bfloat16, device=DEV)
        m = z(T, T, dtype=torch.bool, device=DEV)
        out = ops.tree_attention(q, c, s, c, s, m, n_kv_heads=2, group_size=32, sm_scale=1.0)
        assert out.shape == q.shape
    q = torch.ones(1, 8, 3, 128, dtype=torch.bfloat16, device=DEV)
    c, s = z(1, 2, 0, 64, dtype=torch.uint8, device=DEV), z(1, 2, 0, 4, dtype=torch.bfloat16, device=DEV)
    m = torch.ones(3, 3, dtype=torch.bool, device=DEV)
    out = ops.tree_attention(q, c, s, c, s, m, n_kv_heads=2, group_size=32, sm_scale=1.0)
    assert bool((out == 0).all())


def test_head_dims_past_256_are_refused():
    q = torch.zeros(1, 1, 1, 288, dtype=torch.bfloat16, device=DEV)
    c = torch.zeros(1, 1, 5, 144, dtype=torch.uint8, device=DEV)
    s = torch.zeros(1, 1, 5, 9, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(nat.KVQUnsupported):
        ops.tree_attention(q, c, s, c, s, torch.ones(1, 1, dtype=torch.bool, device=DEV), n_kv_heads=1, group_size=32,
                           sm_scale=1.0)
