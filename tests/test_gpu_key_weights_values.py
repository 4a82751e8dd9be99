"""Attention weight of cached keys where rows are no numbers."""

import pytest
import torch

from paged_reference import default_scale, make_pages, starts
from shared_reference import weight_bound

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _places(table, b, n, page):
    j = torch.arange(n)
    return table[b].long()[j // page], j % page


@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 2, 64), (32, 1, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("accumulate", [False, True])
def test_keys_behind_a_row_that_is_no_number(gpu_device, heads, value, accumulate):
    """A row that is none makes none of the weights of the keys it sees; those behind it have what the other rows give them."""
    from shareprefill_amd import ops

    hq, hkv, d = heads
    g, page, scale = hq // hkv, 16, default_scale(d)
    lens, new = [300, 90, 400, 1], [20, 5, 64, 1]
    gen = torch.Generator().manual_seed(hq)
    k_pages, _, table, kv = make_pages(lens, hkv, d, page, gen)
    q = torch.randn(sum(new), hq, d, generator=gen).to(torch.bfloat16)
    before = torch.rand(k_pages.shape[:3], generator=gen)
    clean = q.clone()
    odd = {0: (3, 0), 1: (0, hq - 1), 2: (40, g - 1)}  # request: (row, query head)
    cu = starts(new)
    for b, (i, h) in odd.items():
        q[cu[b] + i, h, 5] = value
    live = before.to(gpu_device)
    ops.paged_key_weights(q.transpose(0, 1).to(gpu_device), k_pages.to(gpu_device), table.to(gpu_device), _ints(gpu_device, lens), scale, live,
                          cu_q=_ints(gpu_device, cu), accumulate=accumulate)
    got = live.cpu().double()
    for b, (total, n) in enumerate(zip(lens, new)):
        pages, at = _places(table, b, total, page)
        mine, old = got[pages, :, at].t(), before[pages, :, at].t().double()
        rel = weight_bound(clean[cu[b]:cu[b + 1]].transpose(0, 1), kv[b][0], scale)
        for kvh in range(hkv):
            want, spoilt = torch.zeros(total, dtype=torch.float64), 0
            for i in range(n):
                seen = total - n + i + 1
                for h in range(kvh * g, kvh * g + g):
                    if odd.get(b) == (i, h):
                        spoilt = seen
                    else:
                        want[:seen] += torch.softmax(kv[b][0][kvh, :seen].double() @ clean[cu[b] + i, h].double() * scale, 0)
            room = rel * want
            if accumulate:
                want[:total - n] += old[kvh, :total - n]
            room += 2.0 ** -23 * want
            assert mine[kvh, :spoilt].isnan().all(), f"request {b}, kv head {kvh}"
            assert ((mine[kvh] - want).abs() <= room)[spoilt:].all(), f"request {b}, kv head {kvh}"
