"""Eviction by weight against the definition, key by key; all of it is exact."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def definition(pools, table, lens, first, budget, recent, page):
    """-> (pools, lengths left); `pools` k, v and weights, changed in place"""
    left = []
    for b, total in enumerate(lens):
        f = min(first[b] if first else 0, total)
        mid = max(total - f - recent, 0)
        places = [(int(table[b, j // page]) if j // page < table.shape[1] else -1, j % page) for j in range(total)]
        if mid <= budget or any(not 0 <= p < pools[0].shape[0] for p, _ in places[f:]):
            left.append(total)
            continue
        left.append(total - mid + budget)
        for h in range(pools[0].shape[1]):
            w = [float(pools[2][p, h, s]) for p, s in places[f:f + mid]]
            w = [x if x > 0 else 0.0 for x in w]  # (a NaN is not above 0)
            stay = sorted(sorted(range(mid), key=lambda i: (-w[i], i))[:budget]) + list(range(mid, total - f))
            rows = [[pool[places[f + i][0], h, places[f + i][1]].clone() for i in stay] for pool in pools]
            for pool, moved in zip(pools, rows):
                for i, x in enumerate(moved):
                    pool[places[f + i][0], h, places[f + i][1]] = x
    return pools, left


def _run(dev, lens, budget, recent, hkv=2, d=64, page=16, first=None, seed=0, weight=None, spoil=(), narrow=0):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    for b, i, entry in spoil:
        table[b, i] = entry
    table = table[:, :table.shape[1] - narrow].contiguous()
    pools = [torch.randn(pages, hkv, page, d, generator=gen).to(torch.bfloat16) for _ in range(2)]
    pools.append((weight or (lambda shape: torch.exp(3 * torch.randn(shape, generator=gen))))((pages, hkv, page)))
    live = [x.to(dev) for x in pools]
    got = ops.paged_evict(*live, table.to(dev), _ints(dev, lens), budget, recent, first=None if first is None else _ints(dev, first))
    want, left = definition(pools, table, lens, first, budget, recent, page)
    assert got.tolist() == left
    for x, y in zip(live, want):
        assert torch.equal(x.cpu().view(torch.int16 if x.dtype is torch.bfloat16 else torch.int32), y.view(torch.int16 if y.dtype is torch.bfloat16 else torch.int32))


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("hkv,d", [(2, 128), (3, 64), (1, 40), (2, 136)])
def test_ragged_requests(gpu_device, page, hkv, d):
    _run(gpu_device, [300, 0, 1, 57, 1200], 40, 10, hkv, d, page, seed=page + d)
    _run(gpu_device, [300, 5, 130], 100, 0, hkv, d, page, first=[0, 5, 77], seed=page + d)


@pytest.mark.parametrize("budget,recent,first", [(0, 0, [0, 0]), (0, 7, [3, 3]), (1, 0, [16, 500]), (5, 1000, [0, 0]), (499, 0, [0, 0]), (500, 0, [0, 1]), (10 ** 9, 3, [0, 0])])
def test_budgets_at_their_ends(gpu_device, budget, recent, first):
    _run(gpu_device, [500, 90], budget, recent, first=first)


def test_lengths_around_the_tiles(gpu_device):
    for n in (1023, 1024, 1025, 2048, 4097):
        _run(gpu_device, [n], n // 2, 5, hkv=1, d=16, page=64, seed=n)
    _run(gpu_device, [9000], 8500, 20, hkv=1, d=16, page=64)  # (nearly all stay: tiles that overlap what they come from)


def _fast(dev, n, budget, recent, first, weight, width=0, page=64, seed=0):
    """One long request of one kv head, against torch's stable sort."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(seed)
    pages = -(-n // page)
    table = torch.randperm(pages, generator=gen).to(torch.int32)
    wide = torch.full((1, max(width, pages)), -1, dtype=torch.int32)
    wide[0, :pages] = table
    k, v = (torch.randn(pages, 1, page, 8, generator=gen).to(torch.bfloat16) for _ in range(2))
    w = weight((pages, 1, page))
    live = [x.to(dev) for x in (k, v, w)]
    got = ops.paged_evict(*live, wide.to(dev), _ints(dev, [n]), budget, recent, first=_ints(dev, [first]))
    place = lambda x: x[table.long(), 0].reshape(-1, *x.shape[3:])  # in the order of the keys
    mid = n - first - recent
    stay = torch.sort(place(w)[first:first + mid], descending=True, stable=True).indices[:budget].sort().values
    src = torch.cat((torch.arange(first), stay + first, torch.arange(first + mid, n)))
    assert got.tolist() == [src.numel()]
    for x, y in zip(live, (k, v, w)):
        want = place(y).clone()
        want[:src.numel()] = place(y)[src]
        assert torch.equal(place(x.cpu()), want)


@pytest.mark.parametrize("n", [16384, 16385, 16400, 40000, 60000, 140000])
@pytest.mark.parametrize("first", [0, 5, 64])
def test_long_requests(gpu_device, n, first):
    """Keys of a kv head that one workgroup's registers hold, and more, which are listed by one workgroup or by several."""
    gen = torch.Generator().manual_seed(n + first)
    spread = lambda shape: torch.exp(2 * torch.randn(shape, generator=gen))
    for weight in (spread, lambda shape: torch.full(shape, 0.25), lambda shape: 1.0 + torch.randint(0, 900, shape, generator=gen).float() * 2.0 ** -22):
        _fast(gpu_device, n, n // 16, 33, first, weight)
        _fast(gpu_device, n, n - first - 50, 33, first, weight)
    _fast(gpu_device, n, 700, 0, first, spread, width=4000)  # a table that has room for much more


def test_equal_weights_keep_the_first(gpu_device):
    _run(gpu_device, [3000, 700], 300, 20, weight=lambda shape: torch.zeros(shape))
    gen = torch.Generator().manual_seed(3)
    _run(gpu_device, [3000, 700], 300, 20, weight=lambda shape: torch.randint(0, 3, shape, generator=gen).float())
    _run(gpu_device, [3000], 300, 20, weight=lambda shape: 1.0 + torch.randint(0, 700, shape, generator=gen).float() * 2.0 ** -23)


def test_weights_that_are_no_weights(gpu_device):
    gen = torch.Generator().manual_seed(4)

    def odd(shape):
        w = torch.rand(shape, generator=gen)
        kind = torch.randint(0, 8, shape, generator=gen)
        for i, x in enumerate((float("nan"), float("inf"), -1.0, -0.0, 1e-45, 3e38)):
            w[kind == i] = x
        return w

    _run(gpu_device, [900, 333], 200, 4, weight=odd)
    _run(gpu_device, [900, 333], 700, 4, weight=odd)


def test_requests_with_a_missing_page_stay(gpu_device):
    _run(gpu_device, [300, 300, 300], 40, 10, spoil=[(0, 3, -1), (1, 18, 10 ** 6)])
    _run(gpu_device, [300, 300], 40, 10, first=[64, 64], spoil=[(0, 3, -1), (1, 4, -1)])  # (in front of the first that may go; at it)
    _run(gpu_device, [300, 100], 40, 10, narrow=2)


def test_strided_pools(gpu_device):
    from shareprefill_amd import ops

    dev, gen = gpu_device, torch.Generator().manual_seed(5)
    lens, page, hkv, d, pages = [200, 90], 16, 2, 64, 22
    table = torch.randperm(pages, generator=gen)[:20].to(torch.int32)
    table = torch.stack((table[:13], torch.cat((table[13:20], torch.full((6,), -1, dtype=torch.int32)))))
    pools = [torch.randn(pages, hkv, page, d, generator=gen).to(torch.bfloat16) for _ in range(2)] + [torch.rand(pages, hkv, page, generator=gen)]
    k = torch.zeros(pages, page, hkv, d, dtype=torch.bfloat16, device=dev).transpose(1, 2)
    v = torch.zeros(pages, hkv + 1, page, d + 8, dtype=torch.bfloat16, device=dev)[:, 1:, :, :d]
    w = torch.zeros(pages, hkv, page + 3, device=dev)[:, :, :page]
    for x, y in zip((k, v, w), pools):
        x.copy_(y)
    got = ops.paged_evict(k, v, w, table.to(dev), _ints(dev, lens), 50, 8)
    want, left = definition(pools, table, lens, None, 50, 8, page)
    assert got.tolist() == left and all(torch.equal(x.cpu(), y) for x, y in zip((k, v, w), want))


def test_a_replayed_eviction(gpu_device):
    from shareprefill_amd import ops

    dev, gen = gpu_device, torch.Generator().manual_seed(6)
    page, pages = 16, 40
    k, v = (torch.randn(pages, 2, page, 64, generator=gen).to(torch.bfloat16).to(dev) for _ in range(2))
    table = torch.randperm(pages, generator=gen).to(torch.int32).view(2, 20).to(dev)
    start = [k.clone(), v.clone(), torch.rand(pages, 2, page, generator=gen).to(dev)]
    w, lens = start[2].clone(), _ints(dev, [320, 300])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        left = ops.paged_evict(k, v, w, table, lens, 60, 10)
    for n in ([320, 300], [70, 71], [200, 0]):
        for x, y in zip((k, v, w), start):
            x.copy_(y)
        lens.copy_(_ints(dev, n))
        graph.replay()
        torch.cuda.synchronize()
        want, lefts = definition([x.cpu() for x in start], table.cpu(), n, None, 60, 10, page)
        assert left.tolist() == lefts and all(torch.equal(x.cpu(), y) for x, y in zip((k, v, w), want))


def test_a_table_that_is_full_to_its_last_place(gpu_device):
    """No last keys that stay, in requests as long as the table has room for."""
    for first in ([0, 0], [16, 5]):
        _run(gpu_device, [64, 64], 20, 0, first=first)
        _run(gpu_device, [1024, 1000], 700, 0, first=first, page=16)
