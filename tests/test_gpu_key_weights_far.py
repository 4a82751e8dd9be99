"""Attention weight of cached keys where logits lie far from zero, up to the ends of fp32's range."""

import pytest
import torch

from paged_reference import make_pages

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _places(table, b, n, page):
    j = torch.arange(n)
    return table[b].long()[j // page], j % page


# Every key's channels are one power of two and the query's another: dot products are exact and keys either share a row's largest logit or lie far below it, so a
# row's weight is shared out evenly among those that have it.  Sums of n equal weights: n 2^-24 of it, twice (the row's, the key's), and a division's rounding.
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("q_exp,k_exp", [(3, 3), (9, 8), (12, 10), (14, 12), (20, 20), (40, 40), (58, 55)])
@pytest.mark.parametrize("three", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_logits_far_from_zero(gpu_device, sign, q_exp, k_exp, three, d):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(q_exp)
    hq, hkv, n, new, page = 4, 2, 1700, 5, 16
    weigh = torch.rand(n, generator=gen) < 0.3
    weigh[0] = True
    k_pages, v_pages, table, _ = make_pages([n], hkv, d, page, gen)
    pages, at = _places(table, 0, n, page)
    k_pages[pages, :, at] = torch.where(weigh, 2.0 ** k_exp, -(2.0 ** k_exp) if sign > 0 else 2.0 ** (k_exp + 1)).to(torch.bfloat16)[:, None, None].expand(n, hkv, d)
    q = torch.full((hq, new, d), three * sign * 2.0 ** q_exp, dtype=torch.bfloat16, device=gpu_device)
    args = (k_pages.to(gpu_device), table.to(gpu_device), _ints(gpu_device, [n]))
    live = torch.zeros(k_pages.shape[:3], device=gpu_device)
    ops.paged_key_weights(q, *args, 1.0, live, cu_q=_ints(gpu_device, [0, new]))
    want = torch.zeros(n, dtype=torch.float64)
    for i in range(new):
        top = weigh & (torch.arange(n) <= n - new + i)
        want[top] += hq // hkv / top.sum().item()
    rel = 2 * n * 2.0 ** -24 + 2.0 ** -20
    got = live.cpu()[pages, :, at].double()
    assert ((got - want[:, None]).abs() <= rel * want[:, None]).all(), (got.sum().item(), want.sum().item() * hkv)
    # single tokens: the same with their attention
    live.zero_()
    ops.shared_prefix_attention(q[:, -1:], args[0], v_pages.to(gpu_device), *args[1:], _ints(gpu_device, []), _ints(gpu_device, [0]), 1.0, weights=live)
    got = live.cpu()[pages, :, at].double()
    want = torch.where(weigh, hq // hkv / weigh.sum().item(), 0.0)[:, None].double()
    assert ((got - want).abs() <= rel * want).all()
