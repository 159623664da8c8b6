"""Attention with changed scores over a paged pool, in 64 bits: the definition,
row by row, and how far a kernel may be from it.

TEST INFRASTRUCTURE ONLY. Rows of sequence s at positions p see key j < n where
first <= j and (j <= p and p - j < window, or j < prefix); scores are scale * q.k,
capped as c * tanh(t / c), less slope * |p - j|; a row that sees nothing is 0.

bound: |out - exact| of a kernel that rounds its probabilities P and its result
to the 2-byte type (unit roundoff u: 2^-8, 2^-11) and computes the rest in fp32:
- the result's rounding: u |out|;
- P's roundings, which both sums see: sum p (1 + d_j) v / sum p (1 + d_j) with
  |d_j| <= u moves by at most u (sum p |v| + |out|);
- fp16's P below its normal range (2^-14 of a largest P of 1 or more) is off by
  at most 2^-25 each: n 2^-25 (max |v| + |out|);
- a score off by e changes p by the factor exp(e): 2 e (sum p |v| + |out|) to first
  order for e << 1. e: the dot product's D fp32 additions, D 2^-24 scale |q| |k|;
  the cap's, the distance term's and the exponential's roundings, 8 2^-24 of the
  largest |t| among keys that count (p > 2^-30), or of the cap;
- accumulation of n products in fp32: n 2^-24 (sum p |v| + |out|), and the same
  again for the sums' merges.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gather(cache: torch.Tensor, table: torch.Tensor, n: int) -> torch.Tensor:
    """The first n rows of a sequence, [n, kv heads, D], as stored."""
    bs = cache.size(2)
    ids = table[: -(-n // bs)].long()
    c = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    rows = c[ids].permute(0, 2, 1, 3).reshape(-1, c.size(1), c.size(3))[:n]
    return rows.contiguous().view(torch.float8_e4m3fn) if cache.element_size() == 1 else rows


def attend(q, k, v, pos, n, scale, softcap=0.0, slopes=None, window=0, first=None, prefix=0):
    """q [T, H, D], k / v [n, KV, D] (any float type), pos [T] -> (out, bound less the
    part of u) as float64: out [T, H, D], and a function of (dtype) giving the bound."""
    T, H, D = q.shape
    KV = k.size(1)
    G = H // KV
    dev = q.device
    q, k, v = q.double(), k.double(), v.double()
    j = torch.arange(n, device=dev)
    p = pos.to(dev).long()[:, None]
    see = (j <= p) & (p - j < window) if window else j <= p
    see = see | (j < prefix)
    if first is not None:
        see = see & (j >= first.to(dev).long()[:, None])
    see = see & (p >= 0)
    out = torch.zeros(T, H, D, dtype=torch.float64, device=dev)
    spread = torch.zeros_like(out)     # sum p |v| + |out|
    err_t = torch.zeros(T, H, 1, dtype=torch.float64, device=dev)
    vmax = torch.zeros(T, H, 1, dtype=torch.float64, device=dev)
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        t = (q[:, h] @ kh.t().contiguous()) * scale
        if softcap:
            t = softcap * torch.tanh(t / softcap)
        if slopes is not None:
            t = t - float(slopes[h]) * (p - j).abs().double()
        t = torch.where(see, t, torch.full_like(t, -math.inf))
        m = t.amax(-1, keepdim=True) if n else torch.full((T, 1), -math.inf, device=dev)
        w = torch.where(see, torch.exp(t - torch.where(m == -math.inf, torch.zeros_like(m), m)),
                        torch.zeros_like(t))
        l = w.sum(-1, keepdim=True)
        w = torch.where(l > 0, w / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(w))
        vv = torch.where(see.any(0)[:, None], vh, torch.zeros_like(vh))
        kk = torch.where(see.any(0)[:, None], kh, torch.zeros_like(kh))
        out[:, h] = w @ vv
        spread[:, h] = w @ vv.abs() + out[:, h].abs()
        counts = w > 2.0 ** -30
        tm = torch.where(counts, t.abs(), torch.zeros_like(t)).amax(-1, keepdim=True) if n else l
        kn = kk.norm(dim=-1).max() if n else 0.0
        err_t[:, h] = 2.0 ** -24 * (D * scale * q[:, h].norm(dim=-1, keepdim=True) * kn
                                    + 8 * torch.clamp(tm, min=softcap) + 8)
        vmax[:, h] = vv.abs().max() if n else 0.0

    def bound(dtype):
        u = U[dtype]
        b = u * out.abs() + (u + 2 * err_t + 2 * n * 2.0 ** -24) * spread
        if dtype == torch.float16:
            b = b + n * 2.0 ** -25 * (vmax + out.abs()) + 2.0 ** -25
        return b * 1.01 + 1e-30

    return out, bound
