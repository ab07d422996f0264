"""What tree attention, key weights and eviction refuse, without a GPU: the C entry points' own checks (no launch), and
the operators' on host tensors and wrong shapes."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kvint4 import _native as nat, ops

A = nat.i64_array
S4, S3, S2 = A([0, 0, 0, 1]), A([0, 0, 64]), A([0, 64])
SC3 = A([0, 0, 4])
B16, F32 = nat.KVQ_BF16, nat.KVQ_F32
PTR = ctypes.c_void_p(4096)  # never read: the checks come first


def _tree(**kw):
    a = dict(q=PTR, qd=B16, qs=S4, kp=PTR, kps=S3, ks=PTR, kss=SC3, vp=PTR, vps=S3, vs=PTR, vss=SC3, sd=B16, m=PTR,
             ms=A([0, 1, 1]), o=PTR, os=S4, B=1, Hq=8, Hkv=2, T=4, D=128, G=32, sl=None, Sk=16, sm=1.0, ws=None, wb=0)
    a.update(kw)
    return nat.lib().kvq_tree_attn(*a.values(), None)


@pytest.mark.parametrize("bad,code,says", [
    (dict(qd=7), nat.KVQ_EINVAL, "dtype"), (dict(Hq=7), nat.KVQ_EINVAL, "multiple"), (dict(T=-1), nat.KVQ_EINVAL, "shape"),
    (dict(G=0), nat.KVQ_EINVAL, "shape"), (dict(D=257), nat.KVQ_EUNSUP, "256"), (dict(q=None), nat.KVQ_EINVAL, "null"),
    (dict(m=None), nat.KVQ_EINVAL, "null"), (dict(o=None), nat.KVQ_EINVAL, "null"), (dict(vp=None), nat.KVQ_EINVAL, "null"),
    (dict(kps=A([0, 0, 63])), nat.KVQ_EINVAL, "narrower"), (dict(vss=A([0, 0, 3])), nat.KVQ_EINVAL, "narrower"),
    (dict(ms=None), nat.KVQ_EINVAL, "stride"), (dict(Sk=1 << 31), nat.KVQ_EINVAL, "large"),
])
def test_tree_arguments(bad, code, says):
    assert _tree(**bad) == code and says in nat.last_error()


def test_tree_calls_without_rows_launch_nothing():
    assert _tree(B=0, q=None, kp=None, ks=None, vp=None, vs=None, m=None, o=None) == nat.KVQ_OK
    assert _tree(T=0, q=None, m=None, o=None) == nat.KVQ_OK
    assert nat.lib().kvq_tree_attn_workspace_bytes(0, 8, 2, 4, 128, 32, 16, B16, B16) == 0
    assert nat.lib().kvq_tree_attn_workspace_bytes(1, 7, 2, 4, 128, 32, 16, B16, B16) == nat.KVQ_EINVAL
    assert nat.lib().kvq_tree_attn_workspace_bytes(1, 8, 2, 4, 128, 32, 16, 9, B16) == nat.KVQ_EINVAL


def _paged(**kw):
    a = dict(q=PTR, qd=B16, qs=S4, kp=PTR, kps=S2, ks=PTR, kss=A([0, 4]), vp=PTR, vps=S2, vs=PTR, vss=A([0, 4]), sd=B16,
             bt=PTR, stride=2, cols=2, blocks=3, page=64, m=PTR, ms=A([0, 1, 1]), o=PTR, os=S4, B=1, Hq=8, Hkv=2, T=4,
             D=128, G=32, sl=None, Sk=100, sm=1.0, ws=None, wb=0)
    a.update(kw)
    return nat.lib().kvq_tree_attn_paged(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(page=48), dict(page=0), dict(Sk=129), dict(bt=None), dict(stride=1), dict(blocks=-1)])
def test_paged_tree_arguments(bad):
    assert _paged(**bad) == nat.KVQ_EINVAL


def test_key_weight_arguments():
    lib = nat.lib()
    need = lib.kvq_key_weights_workspace_bytes(1, 8, 2, 4, 128, 32, 16, B16, B16, 0)
    assert need > 0
    assert lib.kvq_key_weights_workspace_bytes(1, 7, 2, 4, 128, 32, 16, B16, B16, 0) == nat.KVQ_EINVAL

    def call(**kw):
        a = dict(q=PTR, qd=B16, qs=S4, kp=PTR, kps=S3, ks=PTR, kss=SC3, sd=B16, w=PTR, wst=A([0, 0, 1]), B=1, Hq=8,
                 Hkv=2, Sq=4, D=128, G=32, sl=None, Sk=16, causal=1, sm=1.0, ws=PTR, wb=need)
        a.update(kw)
        return lib.kvq_add_key_weights(*a.values(), None)

    assert call(ws=None) == nat.KVQ_ESPACE and "workspace" in nat.last_error()
    assert call(wb=need - 1) == nat.KVQ_ESPACE
    assert call(ws=ctypes.c_void_p(4100)) == nat.KVQ_ESPACE
    assert call(w=None) == nat.KVQ_EINVAL and call(wst=None) == nat.KVQ_EINVAL and call(D=300) == nat.KVQ_EUNSUP
    assert call(B=0, ws=None) == nat.KVQ_OK and call(Sq=0, ws=None) == nat.KVQ_OK


def test_select_arguments():
    def call(B=1, H=2, S=100, keep=10, sink=0, recent=0, w=PTR, index=PTR, st=A([0, 0, 1])):
        return nat.lib().kvq_select_keys(w, st, B, H, S, None, keep, sink, recent, index, None)

    assert call(keep=10, sink=6, recent=5) == nat.KVQ_EINVAL and "hold" in nat.last_error()
    assert call(sink=-1) == nat.KVQ_EINVAL and call(keep=-1) == nat.KVQ_EINVAL and call(recent=1 << 62, keep=5) == nat.KVQ_EINVAL
    assert call(S=-1) == nat.KVQ_EINVAL and call(w=None) == nat.KVQ_EINVAL and call(index=None) == nat.KVQ_EINVAL
    assert call(st=None) == nat.KVQ_EINVAL
    assert call(keep=0, index=None) == nat.KVQ_OK and call(B=0, w=None, index=None) == nat.KVQ_OK


def test_move_arguments():
    one = (ctypes.c_void_p * 1)(4096)

    def call(k=1, src=one, dst=one, width=64, B=1, H=2, S=100, n=10, rows=100, in_place=0, index=PTR):
        w = A([width] * max(k, 1))
        st = A([0, 0, 64] * max(k, 1))
        return nat.lib().kvq_move_rows(k, src, st, dst, st, w, index, A([0, 0, 1]), B, H, S, n, rows, None, 0, in_place,
                                       None)

    assert call(k=0) == nat.KVQ_EINVAL and call(k=6) == nat.KVQ_EINVAL and call(width=0) == nat.KVQ_EINVAL
    assert call(S=-1) == nat.KVQ_EINVAL and call(index=None) == nat.KVQ_EINVAL and call(B=40000) == nat.KVQ_EINVAL
    assert call(n=1025, in_place=1) == nat.KVQ_EINVAL and "in place" in nat.last_error()
    assert call(src=(ctypes.c_void_p * 1)(None)) == nat.KVQ_EINVAL
    assert call(n=0, index=None) == nat.KVQ_OK and call(B=0, index=None) == nat.KVQ_OK


# -- the operators ------------------------------------------------------------

Q = torch.zeros(2, 8, 4, 128, dtype=torch.bfloat16)
C, SC = torch.zeros(2, 2, 9, 64, dtype=torch.uint8), torch.zeros(2, 2, 9, 4, dtype=torch.bfloat16)
M = torch.ones(4, 4, dtype=torch.bool)
KW = dict(n_kv_heads=2, group_size=32, sm_scale=1.0)


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_attention(Q, C, SC, C, SC, M, **KW)
    with pytest.raises(ValueError, match="GPU"):
        ops.add_key_weights(Q, C, SC, torch.zeros(2, 2, 9), is_causal=True, **KW)
    with pytest.raises(ValueError, match="GPU"):
        ops.attention_with_key_weights(Q, C, SC, C, SC, torch.zeros(2, 2, 9), is_causal=True, **KW)
    with pytest.raises(ValueError, match="GPU"):
        ops.select_keys(torch.zeros(1, 1, 5), 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.move_rows([C], torch.zeros(1, 1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        ops.move_rows_paged([C[0]], type("T", (), {"table": torch.zeros(1, 1), "num_blocks": 1, "page_size": 9})(),
                            torch.zeros(1, 1, 2, dtype=torch.int32))


@pytest.mark.parametrize("name,places,n", [
    ("tree_attn", (0, 2, 3, 4, 5, 7, 8), 21), ("tree_attn_paged", (0, 2, 3, 4, 5, 8, 9), 22),
    ("attn_key_weights", (0, 2, 3, 4, 5, 7, 8), 22), ("add_key_weights", (0, 2, 3, 5), 19), ("select_keys", (0, 8), 10)])
def test_the_host_module_refuses_host_tensors(name, places, n):
    fn, t = getattr(nat.host(), name), torch.zeros(1, 1, 1, 1)
    for at in places:
        args = [None if i in places else 0 for i in range(n)]
        if name == "tree_attn_paged":
            args[7] = (None, 0, 0, 0, 0)
        args[at] = t
        with pytest.raises(ValueError, match="host memory"):
            fn(*args)
    with pytest.raises(TypeError):
        fn(*([0] * (n - 1)))


def test_the_host_module_refuses_host_tensors_in_tuples():
    t = torch.zeros(1, 1, 1, 1)
    with pytest.raises(ValueError, match="host memory"):
        nat.host().move_rows((t,), (t,), (1,), (1,), None, 1, 1, 1, 1, 1, None, 0, 0, None)
    with pytest.raises(ValueError, match="tuples"):
        nat.host().move_rows([t], [t], (1,), (1,), None, 1, 1, 1, 1, 1, None, 0, 0, None)
    with pytest.raises(ValueError, match="host memory"):
        nat.host().move_rows_paged((t,), (1,), (1,), (None, 0, 0, 0, 1), None, 1, 1, 1, None, 0, None)
    with pytest.raises(ValueError, match="tuples"):
        nat.host().move_rows_paged((t,) * 6, (1,) * 6, (1,) * 6, (None, 0, 0, 0, 1), None, 1, 1, 1, None, 0, None)
