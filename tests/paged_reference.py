"""Attention with a window and sinks in 64 bits, and how far the kernels' outputs may be from it.

The bound, element by element (u = 2^-8, half a step of bf16, D channels, w the softmax weights):
  * the kernel rounds the probabilities to bf16 and divides by the sum of the rounded ones: the output moves by at most
    u * sum_j w_j |v_j - out| / (1 - u) <= u (A + |out|) / (1 - u), A = sum_j w_j |v_j|;
  * the output's own rounding: u |out'| where |out'| <= |out| + the former;
  * fp32: a logit is a sum of D products and two roundings of its scaling; each is off by 2^-24 relative, the sum by at most
    (D + 4) 2^-24 L with L = scale * max_j sum_d |q_d k_jd|; the exponential by 2^-21 relative; a weight then moves by e = 2 (D + 4) 2^-24 L + 2^-20
    relative (its own logit's and the maximum's), the output by e (A + |out|); sums of n products by n 2^-24 A beside it."""

import math

import torch

U = 2.0 ** -8


def reference(q, k, v, scale, window, sinks, seen=None):
    """q [Hq, n, D] the last n positions of k, v [Hkv, len, D] (bf16, CPU) -> (out [n, Hq, D], bound [n, Hq, D]) in 64 bits.  seen: bool
    [len], keys that exist.  A masked key takes no part, whatever its value."""
    hq, n, d = q.shape
    hkv, total, _ = k.shape
    g = hq // hkv
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    bound = torch.zeros(n, hq, d, dtype=torch.float64)
    q64, k64, v64 = q.double(), k.double(), v.double()
    j = torch.arange(total)
    for i in range(n):
        p = total - n + i
        keep = j <= p
        if window:
            keep &= (j > p - window) | (j < sinks)
        if seen is not None:
            keep &= seen
        idx = keep.nonzero().reshape(-1)
        if idx.numel() == 0:
            continue
        for h in range(hq):
            kk, vv = k64[h // g, idx], v64[h // g, idx]
            logits = (kk @ q64[h, i]) * scale
            w = torch.softmax(logits, 0)
            o = w @ vv
            a = w @ vv.abs()
            mag = scale * (kk.abs() @ q64[h, i].abs()).max().item()
            e = 2 * (d + 4) * 2.0 ** -24 * mag + 2.0 ** -20 + (idx.numel() + 8) * 2.0 ** -24
            first = (U / (1 - U) + e) * (a + o.abs())
            out[i, h] = o
            bound[i, h] = (first + U * (o.abs() + first)) * 1.001 + 1e-30
    return out, bound


def check(got, want, bound, what=""):
    """got bf16 [n, Hq, D]"""
    if got.numel() == 0:
        return
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {(err / bound).max().item():.2f} of it"
    # the largest errors come near a bound that counts every rounding at its worst; the mean must lie far below
    assert err.mean() <= 0.5 * bound.mean() + 1e-30, what


def make_pages(lens, hkv, d, page, gen, slack=5, token_major=False, fill=float("nan")):
    """Pools with the sequences' pages in random order, `fill` in every place that holds no token.
    -> (k_pages, v_pages [pages, Hkv, page, D] views, table int32 [B, W], [(k, v)] of every sequence [Hkv, len, D])"""
    need = [-(-n // page) for n in lens]
    total = sum(need) + slack
    order = torch.randperm(total, generator=gen)
    width = max(max(need), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    shape = (total, page, hkv, d) if token_major else (total, hkv, page, d)
    pools = [torch.full(shape, fill, dtype=torch.bfloat16) for _ in range(2)]
    if token_major:
        pools = [x.transpose(1, 2) for x in pools]
    at, kv = 0, []
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = ids.to(torch.int32)
        pair = []
        for pool in pools:
            x = torch.randn(hkv, n, d, generator=gen).to(torch.bfloat16)
            for i, page_id in enumerate(ids.tolist()):
                part = x[:, i * page:(i + 1) * page]
                pool[page_id, :, :part.shape[1]] = part
            pair.append(x)
        kv.append(tuple(pair))
    return pools[0], pools[1], table, kv


def starts(q_lens):
    out = [0]
    for n in q_lens:
        out.append(out[-1] + n)
    return out


def default_scale(d):
    return 1.0 / math.sqrt(d)
