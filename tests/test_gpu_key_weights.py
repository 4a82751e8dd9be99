"""Attention weight of cached keys under a request's last queries against the definition in 64 bits."""

import pytest
import torch

from paged_reference import default_scale, make_pages, starts
from shared_reference import key_weights, weight_bound

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _run(dev, lens, new, heads, page, first=None, accumulate=False, seed=0, scale=None, single=False, hide=()):
    from shareprefill_amd import ops

    hq, hkv, d = heads
    gen = torch.Generator().manual_seed(seed)
    k_pages, _, table, kv = make_pages(lens, hkv, d, page, gen)
    for b, entry in hide:
        table[b, entry] = -1
    q = torch.randn(sum(new), hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    scale = scale or default_scale(d)
    before = torch.rand(k_pages.shape[:3], generator=gen)
    live = before.to(dev)
    got = ops.paged_key_weights(q.to(dev), k_pages.to(dev), table.to(dev), _ints(dev, lens), scale, live, cu_q=None if single else _ints(dev, starts(new)),
                                first=None if first is None else _ints(dev, first), accumulate=accumulate)
    assert got is live
    want, room, at = before.double(), torch.zeros(before.shape, dtype=torch.float64), 0
    for b, (total, n) in enumerate(zip(lens, new)):
        rows = q[:, at:at + n]
        at += n
        if n == 0 or total == 0:
            continue
        there = torch.tensor([table[b, j // page] >= 0 for j in range(total)])
        keys = kv[b][0]
        if not there.all():
            w = torch.zeros(hkv, total, dtype=torch.float64)
            for i in range(n):
                seen = there & (torch.arange(total) <= total - n + i)
                for h in range(hq):
                    w[h // (hq // hkv), seen] += torch.softmax(keys[h // (hq // hkv), seen].double() @ rows[h, i].double() * scale, 0)
        else:
            w = key_weights(rows, keys, scale)
        rel = weight_bound(rows, keys, scale)
        for j in range(first[b] if first else 0, total):
            if there[j]:
                place = (int(table[b, j // page]), slice(None), j % page)
                old = before[place].double() if accumulate and j < total - n else torch.zeros(hkv, dtype=torch.float64)
                want[place] = w[:, j] + old
                room[place] = rel * w[:, j] + 2.0 ** -23 * want[place]
    err = (live.cpu().double() - want).abs()
    assert (err <= room).all(), f"{lens} {new}: worst {(err / (room + 1e-300)).max().item():.2f} of the bound"
    return live


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 2, 64), (7, 1, 128), (4, 4, 64), (40, 2, 64)])
@pytest.mark.parametrize("lens,new", [([1], [1]), ([33], [33]), ([127, 128, 129], [3, 40, 1]), ([700, 5, 260], [64, 2, 17])])
def test_weights_match_the_definition(gpu_device, page, heads, lens, new):
    _run(gpu_device, lens, new, heads, page, seed=page + len(lens))
    _run(gpu_device, lens, new, heads, page, first=[n // 3 for n in lens], accumulate=True, seed=page)


def test_single_tokens_without_offsets(gpu_device):
    _run(gpu_device, [5, 300, 0, 64], [1, 1, 1, 1], (8, 2, 128), 16, accumulate=True, single=True)


def test_requests_without_rows_or_keys_and_firsts_past_the_end(gpu_device):
    _run(gpu_device, [50, 0, 70, 130], [0, 0, 3, 2], (8, 2, 64), 16)
    _run(gpu_device, [50, 256, 70], [1, 2, 3], (8, 2, 64), 32, first=[50, 256, 69])


def test_a_long_cache_and_many_requests(gpu_device):
    _run(gpu_device, [20000], [4], (4, 1, 64), 128)
    _run(gpu_device, [(37 * i) % 300 + 3 for i in range(150)], [i % 4 for i in range(150)], (4, 2, 64), 16)


def test_missing_pages_are_not_seen(gpu_device):
    _run(gpu_device, [100, 200], [4, 5], (8, 2, 128), 16, hide=[(0, 2), (1, 0), (1, 12)])


def test_far_logits(gpu_device):
    _run(gpu_device, [300, 90], [5, 7], (8, 2, 128), 16, scale=200.0)


def test_a_request_of_more_rows_than_keys(gpu_device):
    """Rows in front of the first key see nothing and give nothing."""
    from shareprefill_amd import ops

    dev, gen = gpu_device, torch.Generator().manual_seed(1)
    k_pages, _, table, kv = make_pages([4], 2, 64, 16, gen)
    q = torch.randn(9, 4, 64, generator=gen).to(torch.bfloat16).transpose(0, 1)
    live = torch.zeros(k_pages.shape[:3], device=dev)
    ops.paged_key_weights(q.to(dev), k_pages.to(dev), table.to(dev), _ints(dev, [4]), 0.1, live, cu_q=_ints(dev, [0, 9]))
    want = key_weights(q[:, 5:], kv[0][0], 0.1)
    got = live[int(table[0, 0]), :, :4].cpu().double()
    assert ((got - want).abs() <= weight_bound(q, kv[0][0], 0.1) * want).all()


def test_the_same_call_gives_the_same_bits_and_replays(gpu_device):
    from shareprefill_amd import ops

    dev, gen = gpu_device, torch.Generator().manual_seed(2)
    k_pages, _, table, _ = make_pages([900, 300, 40], 2, 128, 16, gen)
    q = torch.randn(12, 8, 128, generator=gen).to(torch.bfloat16).transpose(0, 1).to(dev)
    args = (q, k_pages.to(dev), table.to(dev), _ints(dev, [900, 300, 40]), 0.1)
    cu = _ints(dev, [0, 5, 9, 12])
    live = torch.zeros(k_pages.shape[:3], device=dev)
    ops.paged_key_weights(*args, live, cu_q=cu)
    want = live.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.paged_key_weights(*args, live, cu_q=cu)
    for _ in range(3):
        live.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(live[want != 0], want[want != 0]) and (live[want == 0] == 9.0).sum() == (want == 0).sum()
        assert torch.equal(ops.paged_key_weights(*args, torch.zeros_like(live), cu_q=cu), want)
