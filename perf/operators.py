"""Tree attention, key weights and eviction over the INT4 cache, as measurable cases.

A case is a dict of plain values. Its ``op`` names the operator:

  tree     attention of a tree of drafted tokens: the block's rows are the last
           ``T`` of each sequence's cached rows, and a mask says which of them
           each query attends (``ops.tree_attention``, ``ops.tree_attention_paged``)
  weights  attention that adds each key's softmax weight, over the query heads
           of its KV head and the block's rows, to the cache's running sum
           (``ops.attention_with_key_weights``): one decode token, a prompt, a chunk
  evict    the rows that an eviction keeps, and their codes, scales and weights
           gathered into smaller buffers (``ops.select_keys``, ``ops.move_rows``)

With ``own`` false ``run`` computes the same in elementary torch operations in
32 bits; ``exact`` does in 64 bits. Shapes are those of the repository's own
benchmark workloads (GPT-2 small and XL, Llama-3.1-8B, the 70B shape) and of
the ranges around them. Keys carry eight outlier channels, as trained models'
keys do.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # the smallest call: GPT-2 small in fp32, a tree of 8 drafts over a short context (latency)
        dict(name="tree-gpt2-f32-t8", op="tree", dtype="f32", B=1, Hq=12, Hkv=12, D=64, G=32, S=1000, T=8,
             ragged=False, page=0),
        # the ordinary speculative step: Llama-3.1-8B, 64 drafts at 16K context
        dict(name="tree-llama8b-16k-t64", op="tree", dtype="bf16", B=1, Hq=32, Hkv=8, D=128, G=32, S=16384, T=64,
             ragged=False, page=0),
        # serving: the 70B shape, eight sequences of different lengths in pages, a small odd tree
        dict(name="tree-70b-paged-b8-t13", op="tree", dtype="bf16", B=8, Hq=64, Hkv=8, D=128, G=32, S=8192, T=13,
             ragged=True, page=64),
        # a wide tree of odd size over a long context, fp16
        dict(name="tree-f16-30k-t101", op="tree", dtype="f16", B=2, Hq=32, Hkv=8, D=128, G=64, S=30001, T=101,
             ragged=False, page=0),
        # one decode token of a layer at 16K context, every step of a cache that evicts
        dict(name="weights-llama8b-16k", op="weights", dtype="bf16", B=1, Hq=32, Hkv=8, D=128, G=32, S=16385, Sq=1,
             ragged=False),
        # GPT-2 XL, 16 short sequences of different lengths, one token each
        dict(name="weights-gpt2xl-ragged-b16", op="weights", dtype="f16", B=16, Hq=25, Hkv=25, D=64, G=32, S=1024,
             Sq=1, ragged=True),
        # the 70B shape, batch 8 at 32K context, one token each (the most bytes)
        dict(name="weights-70b-b8-32k", op="weights", dtype="bf16", B=8, Hq=64, Hkv=8, D=128, G=32, S=32768, Sq=1,
             ragged=False),
        # a whole prompt: every row's weights before the first eviction (the largest)
        dict(name="weights-prompt-4k", op="weights", dtype="bf16", B=1, Hq=32, Hkv=8, D=128, G=32, S=4096, Sq=4096,
             ragged=False),
        # a prompt chunk of odd length after odd cached tokens
        dict(name="weights-chunk-odd-f16", op="weights", dtype="f16", B=1, Hq=32, Hkv=8, D=128, G=32, S=9001, Sq=777,
             ragged=False),
        # a 16K prompt cut to 2K rows a head after its prefill
        dict(name="evict-llama8b-16k-2k", op="evict", dtype="bf16", B=1, Hkv=8, D=128, G=32, S=16384, keep=2048,
             recent=256, sink=4, ragged=False),
        # many short sequences over their budget by a few decode steps
        dict(name="evict-gpt2xl-b16", op="evict", dtype="f16", B=16, Hkv=25, D=64, G=32, S=1100, keep=1000, recent=100,
             sink=1, ragged=True),
        # the 70B shape, eight 32K sequences cut to a quarter (the most rows moved)
        dict(name="evict-70b-b8-32k", op="evict", dtype="bf16", B=8, Hkv=8, D=128, G=32, S=32768, keep=8192,
             recent=1024, sink=4, ragged=False),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "weights", "evict"])
    gpt2 = rng.random() < 0.25
    if gpt2:
        Hkv = rng.choice([12, 25])
        Hq, D, G, dtype = Hkv, 64, 32, rng.choice(["f32", "f16"]) if op == "tree" else "f16"
    else:
        Hkv = rng.choice([1, 2, 4, 8])
        Hq, D, G, dtype = Hkv * rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128]), rng.choice([32, 32, 64]), \
            rng.choice(["bf16", "bf16", "f16"])
    if op == "tree":
        T = _log(rng, 1, 16 if dtype == "f32" else 128)
        B = _log(rng, 1, 16)
        most = 1023 if gpt2 else min(30000, (1 << 21) // (B * T))
        page = rng.choice([0, 0, 64, 128]) if dtype != "f32" else 0
        return dict(op=op, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, G=G, S=max(T, _log(rng, 64, max(64, most))), T=T,
                    ragged=B > 1 and rng.random() < 0.5, page=page)
    if op == "weights":
        if rng.random() < 0.5:
            B = _log(rng, 1, 16)
            return dict(op=op, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, G=G,
                        S=_log(rng, 32, 1023 if gpt2 else min(32768, 262144 // B)), Sq=1,
                        ragged=B > 1 and rng.random() < 0.5)
        B = rng.randint(1, 2)
        S = _log(rng, 64, 1023 if gpt2 else min(9000, int(4096 * math.sqrt(32 / (B * Hq)))))
        return dict(op=op, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, G=G, S=S,
                    Sq=S if rng.random() < 0.5 else _log(rng, 2, S), ragged=False)
    B = _log(rng, 1, 16)
    S = _log(rng, 64, 1023 if gpt2 else min(32768, 262144 // B))
    keep = _log(rng, 8, S if B * S < 100000 else S // 2)
    recent = rng.randint(0, keep // 2)
    return dict(op=op, dtype=dtype, B=B, Hkv=Hkv, D=D, G=G, S=S, keep=keep, recent=recent,
                sink=rng.randint(0, min(8, keep - recent)), ragged=B > 1 and rng.random() < 0.5)


def _scale_size(case):
    return 4 if case["dtype"] == "f32" else 2


def _lengths(case, seed):
    """The sequences' lengths (host): all S, or spread from a quarter of it."""
    if not case["ragged"]:
        return [case["S"]] * case["B"]
    g = torch.Generator().manual_seed(seed)
    least = max(case["S"] // 4, case.get("T", 1))
    lens = torch.randint(least, case["S"] + 1, (case["B"],), generator=g).tolist()
    lens[0] = case["S"]
    return lens


def work(case):
    B, Hkv, D, G, S = (case[k] for k in ("B", "Hkv", "D", "G", "S"))
    # the lengths of a ragged batch are spread evenly from S / 4: 5/8 of S on average, and the first is S
    total = (S + (B - 1) * 0.625 * S) if case["ragged"] else B * S
    row = D // 2 + D // G * _scale_size(case)  # bytes of one key's (or value's) codes and scales
    if case["op"] == "evict":
        kept = B * min(case["keep"], S) * Hkv
        return {"bytes": 4 * total * Hkv + kept * (2 * (2 * row + 4) + 4), "flops": total * Hkv}
    Sq, Hq = case.get("T") or case["Sq"], case["Hq"]
    io = 2 * B * Hq * Sq * D * (4 if case["dtype"] == "f32" else 2)
    pairs = Hq * Sq * (total - (B * (Sq - 1) / 2 if Sq > 1 else 0))
    if case["op"] == "tree":
        return {"bytes": 2 * row * Hkv * total + io + B * Sq * Sq, "flops": 4 * D * Hq * Sq * total}
    return {"bytes": (2 * row + 8) * Hkv * total + io, "flops": 4 * D * pairs}


def _quantized(x, G):
    """(codes, scales) of x [..., D] in the cache's layout: two 4-bit codes + 8 a byte, a scale for each group of G."""
    y = x.float().unflatten(-1, (-1, G))
    top = y.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / 7, torch.ones_like(top))
    n = ((y / scale).round().clamp(-8, 7) + 8).to(torch.uint8).flatten(-2)
    return n[..., 0::2] | (n[..., 1::2] << 4), scale[..., 0].to(x.dtype)


def _cache(case, g, rows):
    """K and V codes and scales of `rows` = (leading sizes) random rows."""
    dt, D, G = DT[case["dtype"]], case["D"], case["G"]
    k = torch.randn(*rows, D, device="cuda", generator=g)
    k[..., torch.randperm(D, device="cuda", generator=g)[:8]] *= 4
    v = torch.randn(*rows, D, device="cuda", generator=g)
    return (*_quantized(k.to(dt), G), *_quantized(v.to(dt), G))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, Hkv, D, S = case["B"], case["Hkv"], case["D"], case["S"]
    lens = _lengths(case, seed)
    st = dict(case=case, lens_host=lens,
              lens=torch.tensor(lens, dtype=torch.int32, device="cuda") if case["ragged"] else None)
    if case["op"] == "tree" and case["page"]:
        # pools of pages in a random order, a table of block ids for each sequence
        P = case["page"]
        need = [-(-n // P) for n in lens]
        order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        table = torch.full((B, max(need)), -1, dtype=torch.int32)
        for b, part in enumerate(order.split(need)):
            table[b, :need[b]] = part
        st["cache"] = _cache(case, g, (Hkv, sum(need) * P))
        st["table"] = table.cuda()
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    else:
        st["cache"] = _cache(case, g, (B, Hkv, S))
    if case["op"] == "evict":
        # a heavy-tailed sum of weights, a tenth of the keys never attended to within fp32
        w = torch.exp(2 * torch.randn(B, Hkv, S, device="cuda", generator=g) - 4)
        st["weights"] = w * (torch.rand(B, Hkv, S, device="cuda", generator=g) > 0.1)
        keep = case["keep"]
        st["kept"] = [torch.zeros(B, Hkv, keep, t.shape[-1], dtype=t.dtype, device="cuda") for t in st["cache"]]
        st["kept_weights"] = torch.zeros(B, Hkv, keep, device="cuda")
        return st
    Sq = case.get("T") or case["Sq"]
    st["q"] = torch.randn(B, case["Hq"], Sq, D, device="cuda", generator=g).to(DT[case["dtype"]])
    if case["op"] == "tree":
        # random trees: node t's parent is a node before it or the cache; a node attends itself and its ancestors
        T, host = case["T"], torch.Generator().manual_seed(seed)
        parent = (torch.rand(B, T, generator=host) * (torch.arange(T) + 1)).long() - 1
        mask = torch.zeros(B, T, T, dtype=torch.bool)
        for t in range(T):
            up = parent[:, t]
            mask[:, t] = (up >= 0)[:, None] & mask[torch.arange(B), up.clamp(min=0)]
            mask[:, t, t] = True
        st["mask"] = mask.cuda()
    else:
        # nothing before a whole prompt, else what some thirty tokens left
        st["weights"] = torch.rand(B, Hkv, S, device="cuda", generator=g) * (32 / S if Sq < S else 0)
    return st


# -- the plain forms ----------------------------------------------------------


def _values(codes, scales):
    """fp32 values of packed codes."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return (n.unflatten(-1, (scales.shape[-1], -1)) * scales.float()[..., None]).flatten(-2)


def _paged_rows(st):
    """[B, Hkv, S, .] copies of the pools' rows through the table."""
    P, S = st["case"]["page"], st["case"]["S"]
    t = torch.arange(S, device="cuda")
    rows = st["table"].long().clamp(min=0)[:, t // P] * P + t % P
    return [p[:, rows].transpose(0, 1) for p in st["cache"]]


def _sm_scale(case):
    return case["D"] ** -0.5


def _softmax(st, q, k, allowed):
    """Softmax weights [B, Hkv, rows, S] of the query rows of each KV head over the keys that `allowed` admits."""
    s = torch.matmul(q, k.transpose(-1, -2)) * _sm_scale(st["case"])
    s = torch.where(allowed, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _plain(st):
    case = st["case"]
    B, Hkv, D, S = case["B"], case["Hkv"], case["D"], case["S"]
    lens = st["lens"].long() if st["lens"] is not None else torch.full((B,), S, device="cuda")
    at = torch.arange(S, device="cuda")
    if case["op"] == "evict":
        return _plain_evict(st, lens, at)
    kp, ks, vp, vs = _paged_rows(st) if case.get("page") else st["cache"]
    Sq = case.get("T") or case["Sq"]
    r = case["Hq"] // Hkv
    q = st["q"].float().reshape(B, Hkv, r * Sq, D)
    back = at - (lens[:, None] - Sq)  # [B, S]: a key's place in the block (negative: before it)
    rows = torch.arange(Sq, device="cuda")
    if case["op"] == "tree":
        inside = torch.gather(st["mask"], 2, back.clamp(0, Sq - 1)[:, None].expand(B, Sq, S))
        allowed = (back < 0)[:, None] | ((back < Sq)[:, None] & inside)
    else:
        allowed = back[:, None] <= rows[None, :, None]
    p = _softmax(st, q, _values(kp, ks), allowed.repeat(1, r, 1)[:, None])
    out = torch.matmul(p, _values(vp, vs)).reshape(B, case["Hq"], Sq, D).to(st["q"].dtype)
    if case["op"] == "tree":
        return {"out": out}
    st["weights"].add_(p.sum(2))
    return {"out": out, "weights": st["weights"]}


def _plain_evict(st, lens, at):
    case = st["case"]
    B, Hkv, S, keep = case["B"], case["Hkv"], case["S"], case["keep"]
    n = lens[:, None, None]
    safe = (at < case["sink"]) | (at >= n - case["recent"])
    rank = torch.where(safe, math.inf, st["weights"])
    rank = torch.where(at < n, rank, -1.0)  # weights are at least 0
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    index = order.masked_fill(order >= n, S).sort(-1).values
    there = index < S
    at_rows = index.clamp(max=S - 1)[..., None]
    kept = [torch.where(there[..., None], t.gather(2, at_rows.expand(B, Hkv, keep, t.shape[-1])), dst)
            for t, dst in zip(st["cache"], st["kept"])]
    weights = torch.where(there, st["weights"].gather(2, at_rows[..., 0]), st["kept_weights"])
    return {"index": torch.where(there, index, -1).to(torch.int32), "kept": kept, "weights": weights}


def run(state):
    if not own:
        return _plain(state)
    path = os.path.join(_ROOT, "kv-cache-triton_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from kvint4 import ops

    case = state["case"]
    if case["op"] == "evict":
        index = ops.select_keys(state["weights"], case["keep"], recent=case["recent"], sink=case["sink"],
                                seq_lens=state["lens"])
        ops.move_rows((*state["cache"], state["weights"]), index, out=(*state["kept"], state["kept_weights"]))
        return {"index": index, "kept": state["kept"], "weights": state["kept_weights"]}
    shape = dict(n_kv_heads=case["Hkv"], group_size=case["G"], sm_scale=_sm_scale(case), seq_lens=state["lens"])
    if case["op"] == "weights":
        out = ops.attention_with_key_weights(state["q"], *state["cache"], state["weights"],
                                             is_causal=case["Sq"] > 1, **shape)
        return {"out": out, "weights": state["weights"]}
    if case["page"]:
        pages = ops.PageTable(state["table"], case["page"], state["cache"][0].shape[1] // case["page"])
        return {"out": ops.tree_attention_paged(state["q"], *state["cache"], pages, state["mask"], **shape)}
    return {"out": ops.tree_attention(state["q"], *state["cache"], state["mask"], **shape)}


# -- the same in 64 bits, sequence by sequence ---------------------------------


def _exact_values(codes, scales, n):
    """float64 values of the first n rows of codes [Hkv, ., W], by a table of a byte's two values."""
    pair = torch.tensor([[(b % 16) - 8, (b // 16) - 8] for b in range(256)], dtype=torch.float64, device="cuda")
    x = pair[codes[:, :n].long()].flatten(2)
    return x * scales[:, :n].double().repeat_interleave(x.shape[-1] // scales.shape[-1], -1)


def exact(case, seed):
    st = prepare(case, seed)
    B, Hkv = case["B"], case["Hkv"]
    if case["op"] == "evict":
        return {"index": None, "kept": [None] * 4, "weights": _exact_evicted(case, st)}
    Sq, r = case.get("T") or case["Sq"], case["Hq"] // Hkv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    weights = None if case["op"] == "tree" else st["weights"].double()
    for b, n in enumerate(st["lens_host"]):
        if case.get("page"):
            P = case["page"]
            ids = st["table"][b, :-(-n // P)].tolist()
            part = [torch.cat([t[:, i * P:(i + 1) * P] for i in ids], 1) for t in st["cache"]]
        else:
            part = [t[b] for t in st["cache"]]
        k, v = _exact_values(part[0], part[1], n), _exact_values(part[2], part[3], n)
        if case["op"] == "tree":
            hidden = ~st["mask"][b]
        else:
            hidden = torch.ones(Sq, Sq, dtype=torch.bool, device="cuda").triu(1)
        hidden = torch.cat([torch.zeros(Sq, n - Sq, dtype=torch.bool, device="cuda"), hidden], 1)
        for h in range(case["Hq"]):
            s = st["q"][b, h].double() @ k[h // r].mT.contiguous() / math.sqrt(case["D"])
            p = torch.softmax(s.masked_fill_(hidden, -math.inf), -1)
            out[b, h] = p @ v[h // r]
            if weights is not None:
                weights[b, h // r, :n] += p.sum(0)
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _exact_evicted(case, st):
    """The kept rows' weights: they are moved, not computed, so these are the inputs' own values."""
    kept = torch.zeros(case["B"], case["Hkv"], case["keep"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lens_host"]):
        w = st["weights"][b, :, :n].double()
        if n > case["keep"]:
            lo, hi = case["sink"], n - case["recent"]
            w = w.clone()
            mid = torch.argsort(w[:, lo:hi], dim=-1, descending=True, stable=True)[:, :case["keep"] - lo - case["recent"]]
            mid = mid.sort(-1).values + lo
            w = torch.cat([w[:, :lo], w.gather(1, mid), w[:, hi:]], 1)
        kept[b, :, :w.shape[1]] = w
    return kept
