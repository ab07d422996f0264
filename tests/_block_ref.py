"""Plain 64-bit restatement of attention of a block of queries over packed INT4 K/V, for the tests of tree attention and
key weights, and the error bounds that follow from the kernels' number formats."""

from __future__ import annotations

import math

import torch


def values(codes: torch.Tensor, scales: torch.Tensor, G: int, D: int) -> torch.Tensor:
    """float64 [..., D] of packed rows: element d is nibble d % G of its group's ceil(G / 2) bytes, times its scale."""
    d = torch.arange(D, device=codes.device)
    g, e = d // G, d % G
    byte = codes[..., g * ((G + 1) // 2) + e // 2].long()
    return (torch.where(e % 2 == 1, byte >> 4, byte & 15) - 8).double() * scales[..., g].double()


def allowed(kind: str, lens: list[int], T: int, S: int, mask: torch.Tensor | None, device) -> torch.Tensor:
    """bool [B, T, S]: which keys each query row attends. The block's own keys are the last T of a sequence's."""
    out = torch.zeros(len(lens), T, S, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(T):
            out[b, i, :max(n - T, 0)] = True
            for t in range(T):
                j = n - T + t
                if 0 <= j < n:
                    m = None if mask is None else mask if mask.dim() == 2 else mask[b]
                    out[b, i, j] = kind == "none" or (kind == "causal" and t <= i) or (kind == "tree" and bool(m[i, t]))
    return out.to(device)


class Reference:
    """Attention of q [B, Hq, T, D] over k, v [B, Hkv, S, D] (float64) with `keys` [B, T, S] saying what is attended.

    out      [B, Hq, T, D]
    weights  [B, Hkv, S]: softmax weights summed over the KV head's query heads and the rows
    spread   [B, Hq, T, D]: sum_j p_j |v_j|
    reach    max over rows and attended keys of |sm_scale| sum_d |q_d k_d|
    top      max |v| of attended keys
    """

    def __init__(self, q, k, v, keys, sm_scale):
        B, Hq, T, D = q.shape
        r = Hq // k.shape[1]
        k, v = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
        on = keys[:, None]
        used = keys.any(1)[:, None, :, None]
        k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)
        s = torch.matmul(q.double(), k.transpose(-1, -2).contiguous()) * sm_scale
        s = torch.where(on, s, -math.inf)
        m = s.amax(-1, keepdim=True)
        e = torch.where(on, torch.exp(s - torch.where(m.isinf(), 0.0, m)), 0.0)
        l = e.sum(-1, keepdim=True)
        p = e / torch.where(l == 0, 1.0, l)
        self.p = p
        self.out = torch.matmul(p, v)
        self.spread = torch.matmul(p, v.abs())
        self.weights = p.sum(2).reshape(B, -1, r, k.shape[2]).sum(2)
        a = torch.matmul(q.double().abs(), k.abs().transpose(-1, -2).contiguous()) * abs(sm_scale)
        self.reach = float(torch.where(on, a, 0.0).max()) if a.numel() else 0.0
        self.top = float(v.abs().max()) if v.numel() else 0.0
        self.S, self.D = k.shape[2], D

    def score_error(self) -> float:
        """A bound of a score's error, in nats: a dot product of D terms in fp32 (with the group sums and the scale's
        multiplication, D + 8 roundings of at most 2^-24 each, relative to the sum of the terms' magnitudes) and one
        more of the exponent's argument, whose size is at most that of the largest score difference, 2 reach."""
        return (self.D + 8) * 2.0 ** -24 * self.reach + 4 * self.reach * 2.0 ** -24 + 2.0 ** -22

    def tolerance(self, dtype: torch.dtype, weight_step: float) -> torch.Tensor:
        """Elementwise bound of |out - reference|. Weights off by a relative 2 d (score errors d in the numerator's and
        the denominator's terms) shift the output by at most 2 (e^2d - 1) / 2 ~ 4 d of the spread; weights and values
        rounded to `weight_step` (half a step, 0 where they stay fp32) each add that much of it; sums of S terms in
        fp32 add S 2^-24; weights under the smallest normal fp16 are off by 2^-25 of the largest weight; and the output
        is rounded once to its type."""
        d = self.score_error()
        soft = (4 * d + 2 * weight_step + (self.S + 16) * 2.0 ** -24) * self.spread
        floor = self.S * 2.0 ** -25 * self.top if weight_step else 0.0
        half = torch.finfo(dtype).eps / 2
        return soft * (1 + half) + floor + half * self.out.abs() + torch.finfo(dtype).tiny

    def weight_tolerance(self, T_rows: int, before: torch.Tensor) -> torch.Tensor:
        """Elementwise bound of |key weights - reference| in fp32: each row's weight is off by a relative 4 d, the sums
        over S keys (the denominator) and over the rows add their roundings, and the running sum is rounded once."""
        d = self.score_error()
        return self.weights * (4 * d + (self.S + T_rows + 16) * 2.0 ** -24) + (before + self.weights) * 2.0 ** -23 + 1e-30


def random_tree(T: int, g: torch.Generator, B: int | None = None) -> torch.Tensor:
    """Masks of random trees: node t's parent is one of the nodes before it, or the cache."""
    masks = []
    for _ in range(B or 1):
        m = torch.zeros(T, T, dtype=torch.bool)
        for t in range(T):
            up = int(torch.randint(-1, t, (1,), generator=g)) if t else -1
            if up >= 0:
                m[t] = m[up]
            m[t, t] = True
        masks.append(m)
    return torch.stack(masks) if B else masks[0]


def random_cache(B, H, S, D, G, scale_dtype, g, device, pad=0):
    """(codes, scales) of random rows; `pad`: extra bytes and scales a row, so that rows are strided."""
    w, ng = math.ceil(D / G) * ((G + 1) // 2), math.ceil(D / G)
    codes = torch.randint(0, 256, (B, H, S, w + pad), dtype=torch.uint8, generator=g).to(device)[..., :w]
    scales = (torch.rand(B, H, S, ng + pad, generator=g) * 0.2 + 0.05).to(scale_dtype).to(device)[..., :ng]
    return codes, scales
