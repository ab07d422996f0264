"""GPU: the rows an eviction keeps and their moves, exactly: ties, NaN and signed zeros, every kind of protected row,
lengths around the budget, ragged batches, strides; rows moved into other buffers, in place and through pages."""

from __future__ import annotations

import math

import pytest
import torch

from kvint4 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _want(w, n_keep, sink, recent, lens):
    """Plain selection, by a stable sort of (NaN first, then falling weight, then row)."""
    B, H, _ = w.shape
    out = torch.full((B, H, n_keep), -1, dtype=torch.int32)
    for b in range(B):
        n = lens[b]
        for h in range(H):
            if n <= n_keep:
                out[b, h, :n] = torch.arange(n)
                continue
            row = w[b, h, :n].tolist()
            mid = sorted(range(sink, n - recent), key=lambda j: (0, 0.0, j) if math.isnan(row[j]) else (1, -row[j], j))
            rows = sorted([*range(sink), *range(n - recent, n), *mid[:n_keep - sink - recent]])
            out[b, h] = torch.tensor(rows)
    return out


def _weights(kind, shape, g):
    w = torch.exp(2 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, shape, generator=g).float()
    elif kind == "equal":
        w = torch.full(shape, 0.25)
    elif kind == "zeros":
        w = torch.where(torch.rand(shape, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "odd":
        w = torch.randn(shape, generator=g) * 10.0 ** torch.randint(-38, 38, shape, generator=g)
        w[torch.rand(shape, generator=g) < 0.05] = math.nan
        w[torch.rand(shape, generator=g) < 0.05] = math.inf
        w[torch.rand(shape, generator=g) < 0.05] = -math.inf
        w[torch.rand(shape, generator=g) < 0.05] = -math.nan
        w[torch.rand(shape, generator=g) < 0.05] = 1e-42
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "zeros", "odd"])
@pytest.mark.parametrize("B,H,S,keep,sink,recent", [
    (1, 8, 1000, 300, 4, 64), (2, 3, 1024, 1023, 0, 0), (1, 2, 1025, 1, 0, 0), (1, 2, 1025, 1, 1, 0), (1, 2, 70, 64, 32, 32),
    (3, 1, 5000, 4000, 10, 2000), (1, 1, 2, 1, 0, 1), (2, 2, 64, 64, 0, 0), (1, 2, 40, 64, 3, 9), (1, 2, 9000, 17, 0, 16),
    (1, 1, 20000, 9999, 1, 0), (1, 1, 70000, 30000, 4, 500)])
def test_selection_is_exact(kind, B, H, S, keep, sink, recent):
    g = torch.Generator().manual_seed(S + keep)
    w = _weights(kind, (B, H, S), g)
    got = ops.select_keys(w.to(DEV), keep, recent=recent, sink=sink)
    assert torch.equal(got.cpu(), _want(w, keep, sink, recent, [S] * B))


@pytest.mark.parametrize("lens", [[0, 1, 99, 100, 101, 640], [640, 500, 110, 1000, -3, 100]])
def test_ragged_selection(lens):
    g = torch.Generator().manual_seed(1)
    w = _weights("ties", (6, 3, 640), g)
    sl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    got = ops.select_keys(w.to(DEV), 100, recent=20, sink=5, seq_lens=sl)
    clamped = [min(max(n, 0), 640) for n in lens]
    assert torch.equal(got.cpu(), _want(w, 100, 5, 20, clamped))
    one = ops.select_keys(w.to(DEV), 100, recent=20, sink=5, seq_len=333)
    assert torch.equal(one.cpu(), _want(w, 100, 5, 20, [333] * 6))


def test_strided_weights():
    g = torch.Generator().manual_seed(2)
    w = _weights("spread", (3, 700, 2), g).to(DEV).permute(0, 2, 1)[:, :, 1:601]
    got = ops.select_keys(w, 77, recent=7, sink=2)
    assert torch.equal(got.cpu(), _want(w.cpu(), 77, 2, 7, [600] * 3))


def _tensors(B, H, S, g, widths=((64, torch.uint8), (4, torch.bfloat16), (33, torch.uint8), (3, torch.float32))):
    out = []
    for w, dt in widths:
        t = torch.randint(0, 256, (B, H, S, w), generator=g)
        out.append(t.to(dt).to(DEV))
    out.append(torch.randn(B, H, S, generator=g).to(DEV))
    return out


def _moved(tensors, dst, index, first):
    out = [d.clone() for d in dst]
    B, H, S = tensors[0].shape[:3]
    index = index.expand(B, H, -1).tolist()
    for b in range(B):
        f = first if isinstance(first, int) else first[b]
        for h in range(H):
            for i, j in enumerate(index[b][h]):
                if 0 <= j < S and 0 <= f + i < dst[0].shape[2]:
                    for t, o in zip(tensors, out):
                        o[b, h, f + i] = t[b, h, j]
    return out


@pytest.mark.parametrize("first", [0, 3, "tensor"])
@pytest.mark.parametrize("shared", [(False, False), (True, True), (True, False)])
def test_rows_move_into_other_buffers(first, shared):
    g = torch.Generator().manual_seed(3)
    B, H, S, n, rows = 2, 3, 90, 41, 50
    src, dst = _tensors(B, H, S, g), _tensors(B, H, rows, g)
    index = torch.randint(-2, S + 3, (1 if shared[0] else B, 1 if shared[1] else H, n), generator=g).int()
    index[..., 5] = index[..., 6]
    f = [-2, 20] if first == "tensor" else first
    arg = torch.tensor(f, dtype=torch.int32, device=DEV) if first == "tensor" else first
    want = _moved([t.cpu() for t in src], [t.cpu() for t in dst], index, f)
    kept = [t.clone() for t in src]
    ops.move_rows(src, index.to(DEV), out=dst, first=arg)
    for a, b in zip(dst, want):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(src, kept):
        assert torch.equal(a, b)


def test_rows_move_between_strided_views():
    g = torch.Generator().manual_seed(4)
    B, H, S, n = 2, 2, 60, 30
    big = torch.randint(0, 256, (H, S, B, 70), generator=g, dtype=torch.uint8).to(DEV)
    src = big.permute(2, 0, 1, 3)[..., 3:67]
    out = torch.zeros(B, H, n, 71, dtype=torch.uint8, device=DEV)
    index = torch.randint(0, S, (B, H, n), generator=g).int()
    ops.move_rows([src], index.to(DEV), out=[out[..., 5:69]])
    want = _moved([src.cpu()], [torch.zeros(B, H, n, 64, dtype=torch.uint8)], index, 0)[0]
    assert torch.equal(out[..., 5:69].cpu(), want) and bool((out[..., :5] == 0).all()) and bool((out[..., 69:] == 0).all())


def test_in_place_moves_take_any_index():
    """Forward, backward and crossing moves, the same row twice, a row onto itself."""
    g = torch.Generator().manual_seed(5)
    B, H, S = 2, 2, 500
    for index in (torch.arange(100, 140), torch.arange(0, 40), torch.tensor([41, 40, 7, 7, 44, -1, 600, 46]),
                  torch.randperm(400, generator=g)):
        t = _tensors(B, H, S, g)
        index = index.int().reshape(1, 1, -1).expand(B, 1, -1).contiguous()
        want = _moved([x.cpu() for x in t], [x.cpu() for x in t], index, 40)
        ops.move_rows(t, index.to(DEV), first=40)
        for a, b in zip(t, want):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("page", [1, 16, 64])
def test_moves_through_pages(page):
    g = torch.Generator().manual_seed(6)
    B, H, S = 2, 3, 200
    need = -(-S // page)
    blocks = B * need + 1
    table = torch.randperm(blocks, generator=g)[:B * need].reshape(B, need).int()
    table[1, 100 // page] = -1
    pools = [torch.randint(0, 256, (H, blocks * page, w), generator=g).to(dt).to(DEV)
             for w, dt in ((64, torch.uint8), (4, torch.float16), (64, torch.uint8), (4, torch.float16))]
    pt = ops.PageTable(table.to(DEV), page, blocks)
    index = torch.tensor([[[150, 151, 160, 199]], [[150, 100, 152, 300]]], dtype=torch.int32)
    first = [149, 98]
    want = [p.cpu().clone() for p in pools]
    row = lambda b, j: None if not 0 <= j < need * page or table[b, j // page] < 0 else \
        int(table[b, j // page]) * page + j % page  # noqa: E731
    old = [p.clone() for p in want]
    for b in range(B):
        for i, j in enumerate(index[b, 0].tolist()):
            s, d = row(b, j), row(b, first[b] + i)
            if s is not None and d is not None:
                for o, p in zip(want, old):
                    o[:, d] = p[:, s]
    ops.move_rows_paged(pools, pt, index.to(DEV), first=torch.tensor(first, dtype=torch.int32, device=DEV))
    for a, b in zip(pools, want):
        assert torch.equal(a.cpu(), b)


def test_select_then_move_keeps_what_attention_needs():
    """The two together, as an eviction: the kept rows are the source's, bit for bit, on a side stream and in a graph."""
    g = torch.Generator().manual_seed(7)
    B, H, S, keep = 2, 4, 3000, 700
    src = _tensors(B, H, S, g)[:4] + [torch.rand(B, H, S, generator=g).to(DEV)]
    dst = [torch.zeros(B, H, keep, *t.shape[3:], dtype=t.dtype, device=DEV) for t in src]

    def evict():
        index = ops.select_keys(src[4], keep, recent=50, sink=4)
        ops.move_rows(src, index, out=dst)
        return index

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        index = evict()
    torch.cuda.current_stream().wait_stream(side)
    rows = index.long()
    for t, d in zip(src, dst):
        at = rows[..., None].expand(B, H, keep, t.shape[3]) if t.dim() == 4 else rows
        assert torch.equal(t.gather(2, at), d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = evict()
    for _ in range(3):
        src[4].copy_(torch.rand(B, H, S, device=DEV))
        graph.replay()
        got = [kept.clone(), *(d.clone() for d in dst)]
        want = evict()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and all(torch.equal(a, b) for a, b in zip(got[1:], dst))
