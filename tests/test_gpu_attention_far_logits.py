"""Logits far from zero, up to the ends of fp32's range.  Every key's channels are one power of two and the query's another or three times one, so dot
products are exact (sums of D equal numbers of two bits, D a power of two) and, rounded by the scale alike, keys either share the largest logit or lie thousands of octaves below it: a row is the mean of the
values that share it.  Equal weights' sums are exact up to fp32 sums of n values; with the division and the output's rounding
|out - mean| <= 2^-8 |mean| 1.01 + n 2^-24 mean |v| (a value v alone comes out as itself up to 2^-8 |v| 1.01)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _mean(v, top):
    """v [Hkv, n, D] of one request, top: bool [n] -> [Hkv, D]"""
    return v[:, top].double().mean(1)


def _check(got, want, n, v, what):
    err = (got.double().cpu() - want).abs()
    allowed = want.abs() * 2.0 ** -8 * 1.01 + n * 2.0 ** -24 * v.double().abs().mean()
    assert (err <= allowed).all(), (what, err.max().item(), got.flatten()[:4].tolist())


# exponents of the keys that weigh (their logit: D times 2^(q + k)) and of the others, far below in value
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("q_exp,k_exp", [(3, 3), (9, 8), (12, 10), (14, 12), (20, 20), (40, 40), (48, 47), (58, 55)])
@pytest.mark.parametrize("three", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_are_the_mean_of_the_largest_logits(gpu_device, sign, q_exp, k_exp, three, d):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(q_exp)
    hq, hkv, n, page, scale = 4, 2, 700, 16, 1.0
    weigh = torch.rand(n, generator=gen) < 0.3
    weigh[0] = True
    # the largest logit is sign * D 2^(q + k); twice as negative, or as far on the other side of zero, for the rest
    k = torch.where(weigh, 2.0 ** k_exp, -(2.0 ** k_exp) if sign > 0 else 2.0 ** (k_exp + 1)).to(torch.bfloat16)[None, :, None].expand(hkv, n, d)
    q = torch.full((hq, n, d), three * sign * 2.0 ** q_exp, dtype=torch.bfloat16)
    v = torch.randn(hkv, n, d, generator=gen).to(torch.bfloat16)
    qd, kd, vd = q.to(gpu_device), k.contiguous().to(gpu_device), v.to(gpu_device)
    pos = torch.arange(n)
    for window in (None, 100):
        got = ops.window_attention(qd[None], kd[None], vd[None], scale, window=window)[0]
        one = ops.window_attention(qd[None, :, -1:], kd[None], vd[None], scale, window=window)[0]
        for p in (0, 1, 5, 63, 64, 127, 300, 511, 699):
            seen = (pos <= p) & (pos > p - (window or n))
            top = seen & weigh if (seen & weigh).any() else seen
            want = _mean(v, top).repeat_interleave(hq // hkv, 0)
            _check(got[p], want, n, v, f"position {p}, window {window}")
            if p == n - 1:
                _check(one[0], want, n, v, f"single token, window {window}")
    # a window of one key: its value, whatever the logit
    got = ops.window_attention(qd[None], kd[None], vd[None], scale, window=1)[0]
    assert torch.equal(got.cpu(), v.transpose(0, 1).repeat_interleave(hq // hkv, 1))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("q_exp,k_exp", [(14, 12), (20, 20), (58, 55)])
@pytest.mark.parametrize("three", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_parts_of_long_caches_are_weighed_by_their_own_maxima(gpu_device, sign, q_exp, k_exp, three, d):
    """Few rows over many keys: sequences are cut, and the parts' partials meet in a second launch.  The keys that weigh lie in the first half."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(q_exp)
    hq, hkv, n, page, scale = 4, 2, 6000, 64, 1.0
    pages = -(-n // page)
    weigh = torch.arange(n) < 2500
    k = torch.where(weigh, 2.0 ** k_exp, -(2.0 ** k_exp) if sign > 0 else 2.0 ** (k_exp + 1)).to(torch.bfloat16)[None, :, None].expand(hkv, n, d)
    v = torch.randn(hkv, n, d, generator=gen).to(torch.bfloat16)
    q = torch.full((hq, 5, d), three * sign * 2.0 ** q_exp, dtype=torch.bfloat16, device=gpu_device)
    pools = []
    for x in (k, v):
        pool = torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16)
        for i in range(pages):
            part = x[:, i * page:(i + 1) * page]
            pool[i, :, :part.shape[1]] = part
        pools.append(pool.to(gpu_device))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    table = torch.arange(pages, dtype=torch.int32, device=gpu_device)[None]
    want = _mean(v, weigh).repeat_interleave(hq // hkv, 0)
    chunk = ops.paged_attention(q, *pools, table, ints([n]), scale, cu_q=ints([0, 5]))
    single = ops.paged_attention(q[:, :1], *pools, table, ints([n]), scale)
    for row in (*chunk, *single):
        _check(row, want, n, v, "cut")


@pytest.mark.parametrize("first", [-(2.0 ** 100), -(2.0 ** 40), -(2.0 ** 27), 2.0 ** 27, 2.0 ** 40])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_come_from_afar(gpu_device, first, d):
    """The first 200 keys' logits lie far from zero, the others' are ordinary: with a negative start rows behind them are the definition's over the
    ordinary keys alone, with a positive one the first keys' mean.  One channel holds the far logit, with the query's 1 there."""
    from paged_reference import check, reference
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(4)
    hq, hkv, n = 4, 2, 460
    q, k, v = (torch.randn(h, n, d, generator=gen).to(torch.bfloat16) for h in (hq, hkv, hkv))
    q[..., 0], k[..., 0] = 3.0, 0.0
    k[:, :200] = 0.0
    k[:, :200, 0] = first
    scale = 0.125
    got = ops.window_attention(*(x[None].to(gpu_device) for x in (q, k, v)), scale)[0].cpu()
    one = ops.window_attention(q[None, :, -1:].to(gpu_device), k[None].to(gpu_device), v[None].to(gpu_device), scale)[0].cpu()
    for p in (0, 1, 70, 199):
        _check(got[p], _mean(v, torch.arange(n) <= p).repeat_interleave(hq // hkv, 0), n, v, f"position {p}")
    if first > 0:
        for p in (200, 333, n - 1):
            _check(got[p], _mean(v, torch.arange(n) < 200).repeat_interleave(hq // hkv, 0), n, v, f"position {p}")
        _check(one[0], _mean(v, torch.arange(n) < 200).repeat_interleave(hq // hkv, 0), n, v, "single token")
    else:
        want, bound = reference(q[:, 200:], k[:, 200:], v[:, 200:], scale, 0, 0)
        check(got[200:], want, bound)
        check(one, want[-1:], bound[-1:])


def test_a_row_without_keys_stays_zero(gpu_device):
    from shareprefill_amd import ops

    q = torch.full((4, 7, 64), -(2.0 ** 58), dtype=torch.bfloat16, device=gpu_device)
    pool = torch.full((3, 2, 16, 64), 2.0 ** 55, dtype=torch.bfloat16, device=gpu_device)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    out = ops.paged_attention(q, pool, pool, ints([[0, 1], [2, -1]]), ints([3, 0]), 1.0, cu_q=ints([0, 5, 7]))
    assert (out[:2] == 0).all() and (out[5:] == 0).all()
    assert (out[2:5] == 2.0 ** 55).all()
    assert math.isfinite(out.float().sum().item())
