"""GPU: what the operators of trees, key weights and eviction refuse on device tensors, before any launch: shapes, dtypes,
strides, lengths and places that the kernels do not take."""

from __future__ import annotations

import pytest
import torch

from kvint4 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype, device=DEV)


def _args(**kw):
    a = dict(q=_z(2, 8, 4, 128), kp=_z(2, 2, 9, 64, dtype=torch.uint8), ks=_z(2, 2, 9, 4),
             vp=_z(2, 2, 9, 64, dtype=torch.uint8), vs=_z(2, 2, 9, 4))
    a.update(kw)
    return list(a.values())


KW = dict(n_kv_heads=2, group_size=32, sm_scale=1.0)
BAD_CACHE = [
    dict(q="q64"), dict(kp="short"),
    dict(ks="f64"), dict(vp="heads"), dict(vs="batch"), dict(kp="narrow"), dict(vs="dtype"), dict(kp="stride"), dict(q="3d"),
]


def _bad(name):
    return {"q64": lambda: _z(2, 8, 4, 128, dtype=torch.float64), "short": lambda: _z(2, 2, 8, 64, dtype=torch.uint8), "f64": lambda: _z(2, 2, 9, 4, dtype=torch.float64),
            "heads": lambda: _z(2, 3, 9, 64, dtype=torch.uint8), "batch": lambda: _z(1, 2, 9, 4),
            "narrow": lambda: _z(2, 2, 9, 63, dtype=torch.uint8), "dtype": lambda: _z(2, 2, 9, 4, dtype=torch.float16),
            "stride": lambda: _z(2, 2, 9, 128, dtype=torch.uint8)[..., ::2], "3d": lambda: _z(8, 4, 128)}[name]()


@pytest.mark.parametrize("bad", BAD_CACHE, ids=lambda d: "-".join(f"{k}-{v}" if isinstance(v, str) else k for k, v in d.items()))
def test_cache_arguments(bad):
    a = _args(**{k: _bad(v) if isinstance(v, str) else v for k, v in bad.items()})
    with pytest.raises(ValueError):
        ops.tree_attention(*a, torch.ones(4, 4, dtype=torch.bool, device=DEV), **KW)
    with pytest.raises(ValueError):
        ops.attention_with_key_weights(*a, _z(2, 2, 9, dtype=torch.float32), is_causal=True, **KW)


@pytest.mark.parametrize("mask", [torch.ones(4, 4), torch.ones(3, 4, dtype=torch.bool), torch.ones(3, 4, 4, dtype=torch.bool),
                                  torch.ones(4, 4, dtype=torch.uint8)], ids=["float", "3x4", "batch", "uint8"])
def test_tree_masks(mask):
    with pytest.raises(ValueError, match="tree_mask"):
        ops.tree_attention(*_args(), mask.to(DEV), **KW)


def test_heads_groups_lengths_and_outputs():
    m = torch.ones(4, 4, dtype=torch.bool, device=DEV)
    for kw in (dict(n_kv_heads=3), dict(n_kv_heads=0), dict(group_size=0)):
        with pytest.raises(ValueError):
            ops.tree_attention(*_args(), m, **{**KW, **kw})
    for sl in (torch.ones(2, dtype=torch.int64, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV),
               torch.ones(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="seq_lens"):
            ops.tree_attention(*_args(), m, seq_lens=sl, **KW)
    for out in (_z(2, 8, 4, 64), _z(2, 8, 4, 128, dtype=torch.float32)):
        with pytest.raises(ValueError, match="out"):
            ops.tree_attention(*_args(), m, out=out, **KW)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_attention(*_args(vs=torch.zeros(2, 2, 9, 4, dtype=torch.bfloat16)), m, **KW)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_attention(*_args(), m.cpu(), **KW)


def test_pages():
    q, m = _z(2, 8, 4, 128), torch.ones(4, 4, dtype=torch.bool, device=DEV)
    pool, sc = _z(2, 192, 64, dtype=torch.uint8), _z(2, 192, 4)
    pt = ops.PageTable(torch.zeros(2, 2, dtype=torch.int32, device=DEV), 64, 3)
    kw = dict(**KW, seq_len=100)
    ops.tree_attention_paged(q, pool, sc, pool, sc, pt, m, **kw)
    with pytest.raises(ValueError):
        ops.tree_attention_paged(q, pool[:, :128], sc, pool, sc, pt, m, **kw)
    with pytest.raises(ValueError, match="share"):
        ops.tree_attention_paged(q, pool, sc, pool, sc.half(), pt, m, **kw)
    with pytest.raises(ValueError, match="seq_len"):
        ops.tree_attention_paged(q, pool, sc, pool, sc, pt, m, **KW)
    with pytest.raises(ValueError, match="seq_len"):
        ops.tree_attention_paged(q, pool, sc, pool, sc, pt, m, **KW, seq_len=129)
    with pytest.raises(ValueError, match="rows"):
        ops.tree_attention_paged(_z(3, 8, 4, 128), pool, sc, pool, sc, pt, m, **kw)


@pytest.mark.parametrize("w", ["half", "2d", "short", "heads", "broadcast"])
def test_key_weight_tensors(w):
    bad = {"half": _z(2, 2, 9), "2d": _z(2, 18, dtype=torch.float32), "short": _z(2, 2, 8, dtype=torch.float32),
           "heads": _z(2, 1, 9, dtype=torch.float32), "broadcast": _z(2, 1, 9, dtype=torch.float32).expand(2, 2, 9)}[w]
    q, kp, ks, vp, vs = _args()
    with pytest.raises(ValueError, match="key_weights"):
        ops.add_key_weights(q, kp, ks, bad, is_causal=True, **KW)
    with pytest.raises(ValueError, match="key_weights"):
        ops.attention_with_key_weights(q, kp, ks, vp, vs, bad, is_causal=True, **KW)


def test_selection():
    w = _z(2, 3, 50, dtype=torch.float32)
    for kw in (dict(n_keep=5, recent=6), dict(n_keep=5, recent=3, sink=3), dict(n_keep=-1), dict(n_keep=5, sink=-1),
               dict(n_keep=5, seq_len=51), dict(n_keep=5, seq_len=4, seq_lens=torch.ones(2, dtype=torch.int32, device=DEV)),
               dict(n_keep=5, seq_lens=torch.ones(3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            ops.select_keys(w, **kw)
    with pytest.raises(ValueError):
        ops.select_keys(w.half(), 5)
    with pytest.raises(ValueError):
        ops.select_keys(w[0], 5)
    assert ops.select_keys(w, 0).shape == (2, 3, 0)


def test_moves():
    t, i = _z(2, 3, 50, 8), torch.zeros(2, 3, 4, dtype=torch.int32, device=DEV)
    out = _z(2, 3, 10, 8)
    ops.move_rows([t], i, out=[out])
    for bad in (dict(index=i.long()), dict(index=i[0]), dict(index=_z(3, 3, 4, dtype=torch.int32)), dict(index=i.cpu()),
                dict(out=[_z(2, 3, 10, 9)]), dict(out=[_z(2, 3, 10, 8, dtype=torch.float16)]), dict(out=[]),
                dict(out=[_z(2, 3, 10)]), dict(first=-1), dict(first=torch.zeros(3, dtype=torch.int32, device=DEV)),
                dict(tensors=[]), dict(tensors=[t] * 6), dict(tensors=[t[0, 0]]), dict(tensors=[t, _z(2, 3, 49, 8)], out=None),
                dict(tensors=[_z(2, 3, 50, 16)[..., ::2]], out=None)):
        a = dict(tensors=[t], index=i, out=[out], first=0)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.move_rows(a["tensors"], a["index"], out=a["out"], first=a["first"])
    with pytest.raises(ValueError, match="overlaps"):
        ops.move_rows([t], i, out=[t[:, :, 5:15]])
    with pytest.raises(ValueError, match="in place"):
        ops.move_rows([_z(1, 1, 9000, 8)], torch.zeros(1, 1, 4097, dtype=torch.int32, device=DEV))
