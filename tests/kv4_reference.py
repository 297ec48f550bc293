"""Plain 64-bit forms of the 4-bit cache's operators, on the CPU, with the bounds that the
kernels' roundings allow (used by test_kv4_gpu.py)."""
from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def values(codes, scales):
    """uint8 [..., D/2], uint8 [..., D/32] -> float64 [..., D]."""
    lo, hi = codes & 15, codes >> 4
    n = torch.stack((lo, hi), -1).flatten(-2).long()
    x = GRID[n & 7] * torch.where(n >= 8, -1.0, 1.0)
    s = torch.exp2(scales.clamp(67, 192).double() - 127)
    return (x.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def quantise(x):
    """float [..., D] -> (codes, scale bytes) by the format's rule, one element at a time in 64 bits."""
    x = x.double()
    blocks = x.unflatten(-1, (-1, 32))
    mag = torch.nan_to_num(blocks.abs(), nan=0.0, posinf=1e300)
    amax = mag.amax(-1)
    e = torch.where(amax > 0, torch.ceil(torch.log2(amax.clamp(min=1e-300) / 6)), torch.full_like(amax, -1000.0))
    byte = (e + 127).clamp(67, 192)
    y = (mag / torch.exp2(byte - 127).unsqueeze(-1)).clamp(max=8.0)  # past the grid: its last code
    d = (y.unsqueeze(-1) - GRID).abs()
    best = d.amin(-1, keepdim=True)
    # of two nearest codes the even one; beyond the grid the last
    near = d <= best
    even = torch.tensor([0, 9, 2, 9, 4, 9, 6, 9])
    first = torch.where(near, torch.arange(8), 99).amin(-1)
    tie = near.sum(-1) > 1
    pick = torch.where(tie, torch.where(near, even, 99).amin(-1), first)
    pick = torch.where(blocks.isnan(), torch.full_like(pick, 7), pick)
    n = (pick + 8 * (torch.signbit(blocks) & ~blocks.isnan())).flatten(-2).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), byte.to(torch.uint8)


def tokens(cache, name, table, b, page_size, n):
    """float64 [n, kv_heads, D]: sequence b's first n tokens."""
    j = torch.arange(n)
    page, slot = table[b][j // page_size].long(), j % page_size
    return values(cache[name][page, :, slot], cache[name + "_scale"][page, :, slot])


def scores(q, k, at, scale, causal, window, softcap, group):
    """(scores [rows, heads, n] with -inf where hidden, bound of their magnitude before the cap)."""
    kk = k.repeat_interleave(group, dim=1)
    s = torch.einsum("ihd,thd->iht", q.double(), kk) * scale
    size = torch.einsum("ihd,thd->iht", q.double().abs(), kk.abs()) * abs(scale)
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    t = torch.arange(k.shape[0])
    hidden = torch.zeros((len(at), k.shape[0]), dtype=torch.bool)
    if causal:
        hidden |= t > at[:, None]
    if window:
        hidden |= t <= at[:, None] - window
    return s.masked_fill(hidden[:, None], -math.inf), size.masked_fill(hidden[:, None], 0.0)


def attention(q, cache, table, lens, cu, page_size, scale, causal=True, window=0, softcap=0.0):
    """out, lse in 64 bits, and how far a kernel's may be off: (out bound, lse bound).

    Scores: products of bf16 values are exact, so a score is off by at most (D + 16) 2^-23 of the sum of
    its products' magnitudes (an fp32 sum in any order, truncating), by a few ulps of the scale and, with a
    cap, by 2^-20 of the cap.  Weights are rounded to bf16 before they meet V (2^-9), the output once more
    (2^-9): together 2^-8 of sum p |v|, with a tenth more for the scores' share."""
    rows, heads, D = q.shape
    hk = cache["k"].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(len(lens)):
        lo, hi, n = cu[b], cu[b + 1], lens[b]
        if lo == hi or n == 0:
            continue
        k, v = (tokens(cache, x, table, b, page_size, n) for x in ("k", "v"))
        at = n - (hi - lo) + torch.arange(hi - lo)
        s, size = scores(q[lo:hi], k, at, scale, causal, window, softcap, heads // hk)
        vv = v.repeat_interleave(heads // hk, dim=1)
        seen = torch.isfinite(s).any(-1)
        p = torch.where(seen[..., None], torch.softmax(torch.where(seen[..., None], s, torch.zeros_like(s)), -1), 0.0)
        out[lo:hi] = torch.einsum("iht,thd->ihd", p, vv)
        lse[lo:hi] = torch.where(seen, torch.logsumexp(s, -1), torch.full_like(lse[lo:hi], -math.inf))
        off = (D + 16) * 2.0 ** -23 * size.amax(-1) + (softcap * 2.0 ** -20 if softcap else 0.0)
        lse_tol[lo:hi] = off + 2.0 ** -20 + 2.0 ** -22 * lse[lo:hi].abs().nan_to_num(posinf=0.0)
        out_tol[lo:hi] = (1.1 * 2.0 ** -8 + 2 * off[..., None]) * torch.einsum("iht,thd->ihd", p, vv.abs()) + 1e-30
    return out, lse, out_tol, lse_tol


def gathered(q, lse, cache, table, lens, cu, page_size, scale, causal=True, window=0, softcap=0.0):
    """Per sequence: (weights [kv_heads, n] in 64 bits, bound)."""
    rows, heads, D = q.shape
    hk = cache["k"].shape[1]
    got = []
    for b in range(len(lens)):
        lo, hi, n = cu[b], cu[b + 1], lens[b]
        k = tokens(cache, "k", table, b, page_size, n)
        at = n - (hi - lo) + torch.arange(hi - lo)
        s, size = scores(q[lo:hi], k, at, scale, causal, window, softcap, heads // hk)
        l64 = lse[lo:hi].double()[..., None]
        p = torch.where(torch.isfinite(s), torch.exp(s - torch.where(torch.isfinite(l64), l64, 0.0)), 0.0)
        # exp of a difference: its absolute error is the weight's relative one
        off = (D + 16) * 2.0 ** -23 * size + (softcap * 2.0 ** -20 if softcap else 0.0) + 2.0 ** -20
        off = off + 2.0 ** -22 * torch.where(torch.isfinite(l64), l64.abs(), 0.0)
        w = p.sum(0).unflatten(0, (hk, -1)).sum(1)
        tol = (p * off).sum(0).unflatten(0, (hk, -1)).sum(1) + 2.0 ** -22 * w + 1e-30
        got.append((w, tol))
    return got


def kept(w, n, budget, sink, recent):
    """The token numbers that one kv head of a sequence of n tokens keeps."""
    if n <= budget:
        return list(range(n))
    middle = range(sink, n - recent)
    rank = sorted(middle, key=lambda j: (-math.inf if math.isnan(w[j]) else w[j], -j), reverse=True)
    # NaN ranks below -inf
    rank = [j for j in rank if not math.isnan(w[j])] + sorted(j for j in rank if math.isnan(w[j]))
    return sorted([*range(sink), *rank[:budget - sink - recent], *range(n - recent, n)])
