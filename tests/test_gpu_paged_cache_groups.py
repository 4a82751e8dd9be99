"""A server's run with shared starts of prompts, weights of the keys and evictions: every step against the definition over what each request holds."""

import random

import pytest
import torch

from paged_reference import check, default_scale, reference
from shared_reference import key_weights, weight_bound

pytestmark = pytest.mark.gpu


class Held:
    """What every request holds, layer by layer: keys, values [Hkv, n, D] and weights [Hkv, n] (64 bits), and how far the weights may be off."""

    def __init__(self, layers, rows, hkv, d):
        self.empty = lambda: [(torch.zeros(hkv, 0, d, dtype=torch.bfloat16),) * 2 + (torch.zeros(hkv, 0, dtype=torch.float64),) * 2 for _ in range(layers)]
        self.of = [self.empty() for _ in range(rows)]
        self.position = [0] * rows

    def add(self, row, layer, k, v):
        kk, vv, w, room = self.of[row][layer]
        pad = torch.zeros(w.shape[0], k.shape[1], dtype=torch.float64)
        self.of[row][layer] = (torch.cat((kk, k), 1), torch.cat((vv, v), 1), torch.cat((w, pad), 1), torch.cat((room, pad), 1))

    def weigh(self, row, layer, q, scale, first, adds):
        """q [Hq, n, D] of the last n keys; keys in front of `first` have no weight"""
        k, v, w, room = self.of[row][layer]
        new, rel, n = key_weights(q, k, scale), weight_bound(q, k, scale), q.shape[1]
        old, slack = w.clone(), room.clone()
        if not adds:
            old.zero_(), slack.zero_()
        old[:, k.shape[1] - n:], slack[:, k.shape[1] - n:] = 0, 0
        w, room = old + new, slack + rel * new + 2.0 ** -23 * (old + new)
        w[:, :first], room[:, :first] = 0, 0
        self.of[row][layer] = (k, v, w, room)


def _places(cache, row, n):
    j = torch.arange(n)
    table = cache.block_table[row].cpu().long()
    return table[j // cache.page_size], j % cache.page_size


def _check_weights(cache, held, row, layer, first):
    k, _, w, room = held.of[row][layer]
    pages, at = _places(cache, row, k.shape[1])
    got = cache.weights[layer].cpu()[pages, :, at].t().double()
    assert ((got - w).abs() <= room)[:, first:].all(), f"weights of request {row}"
    return got


@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (14, 2, 64, 32)])
def test_a_server_run(gpu_device, hq, hkv, d, page):
    from shareprefill_amd import PagedKVCache

    gen, rng = torch.Generator().manual_seed(page), random.Random(page)
    layers, rows, scale = 2, 7, default_scale(d)
    cache = PagedKVCache(layers, num_pages=-(-7 * 400 // page), num_kv_heads=hkv, head_dim=d, max_requests=rows, max_tokens=512, page_size=page,
                         device=gpu_device, group_sizes=[3, 2], key_weights=True)
    held = Held(layers, rows, hkv, d)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    shared = [0] * rows

    def step(new=None, active=None, observe=None):
        counts = new if new is not None else [int(a) for a in active]
        total = sum(new) if new is not None else rows
        if new is not None:
            tables = cache.begin_step(ints(new), total)
        else:
            tables = cache.begin_step(active=torch.tensor(active, device=gpu_device))
        assert tables.free_left.item() >= 0
        q_all = []
        for layer in range(layers):
            q, k, v = (torch.randn(total, h, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for h in (hq, hkv, hkv))
            cache.write(layer, k.to(gpu_device), v.to(gpu_device))
            out = cache.attend(layer, q.to(gpu_device), scale).cpu()
            at = 0
            for r, n in enumerate(counts):
                rows_of = slice(at, at + n) if new is not None else slice(r, r + n)
                if n:
                    held.add(r, layer, k[:, rows_of], v[:, rows_of])
                    check(out[rows_of], *reference(q[:, rows_of], *held.of[r][layer][:2], scale, 0, 0), f"request {r}")
                    if new is None:
                        held.weigh(r, layer, q[:, rows_of], scale, shared[r], True)
                at += n
            if observe is not None:
                cache.observe(layer, q.to(gpu_device), scale, last=observe[0], accumulate=observe[1])
                at = 0
                for r, n in enumerate(counts):
                    if n:
                        held.weigh(r, layer, q[:, max(at, at + n - observe[0]):at + n], scale, shared[r], observe[1])
                    at += n
        positions, at = tables.positions.tolist(), 0
        for r, n in enumerate(counts):
            mine = positions[at:at + n] if new is not None else positions[r:r + n]
            assert mine == list(range(held.position[r], held.position[r] + n)), f"request {r}"
            held.position[r] += n
            at += n

    def evict(budget, recent, sinks, mask):
        lens = cache.lens.tolist()
        want = []
        for r in range(rows):
            first, n = min(max(shared[r], sinks), lens[r]), lens[r]
            mid = max(n - first - recent, 0)
            keep = min(mid, budget)
            want.append(n - mid + keep if mask[r] and keep < mid else n)
            for layer in range(layers):
                if not (mask[r] and keep < mid):
                    continue
                k, v, w, room = held.of[r][layer]
                got = _check_weights(cache, held, r, layer, shared[r])
                stay = []
                for h in range(hkv):
                    order = sorted(range(mid), key=lambda i: (-got[h, first + i].item(), i))[:keep]
                    stay.append(list(range(first)) + [first + i for i in sorted(order)] + list(range(first + mid, n)))
                stay = torch.tensor(stay)
                pick = lambda x: torch.stack([x[h, stay[h]] for h in range(hkv)])
                held.of[r][layer] = tuple(pick(x) for x in (k, v, w, room))
        cache.evict(budget, recent, sinks, rows=None if all(mask) else torch.tensor(mask, device=gpu_device))
        assert cache.lens.tolist() == want
        for r in range(rows):
            for layer in range(layers):
                k, v = held.of[r][layer][:2]
                pages, at = _places(cache, r, k.shape[1])
                assert torch.equal(cache.pools[layer, 0].cpu()[pages, :, at].transpose(0, 1), k) and torch.equal(cache.pools[layer, 1].cpu()[pages, :, at].transpose(0, 1), v)
                _check_weights(cache, held, r, layer, shared[r])

    def share(group, tokens):
        cache.share(group, tokens)
        first, end = cache._group_starts[group:group + 2]
        n = tokens // page * page
        for r in range(first, end):
            shared[r] = n
            if r > first:
                held.of[r] = [tuple(x[:, :n].clone() for x in layer) for layer in held.of[first]]
                held.position[r] = n

    step(new=[150, 0, 0, 90, 0, 40, 0], observe=(8, False))
    share(0, 140), share(1, 33)
    step(new=[3, 30, 1, 0, 55, 1, 70], observe=(5, False))
    for i in range(6):
        step(active=[True, True, i % 2 == 0, i > 2, True, i != 1, True])
    step(new=[1, 4, 0, 9, 2, 1, 20], observe=(64, True))
    evict(20, 9, 4, [True] * rows)
    for i in range(4):
        step(active=[True, i != 1, True, True, True, i > 1, True])
    evict(10, 3, 0, [True, False, True, True, False, True, True])
    assert all(layer[0].shape[1] >= shared[r] for r in range(rows) for layer in held.of[r])
    step(new=[2, 3, 1, 1, 30, 1, 1], observe=(3, True))
    # requests end, others come into their rows behind the same start
    done = [1, 4, 6]
    mask = torch.tensor([r in done for r in range(rows)], device=gpu_device)
    cache.release(mask)
    for r in done:
        held.of[r], held.position[r] = held.empty(), 0
    cache.join(torch.tensor([r in (1, 4) for r in range(rows)], device=gpu_device))
    for r, first in ((1, 0), (4, 3)):
        held.of[r] = [tuple(x[:, :shared[r]].clone() for x in layer) for layer in held.of[first]]
        held.position[r] = shared[r]
    shared[6] = 0
    step(new=[1, 20, 1, 1, 7, 1, 33], observe=(4, False))
    step(active=[True] * rows)
    # a group's first row ends: its shared pages stay with the others, which go on by themselves
    cache.release(torch.tensor([r == 0 for r in range(rows)], device=gpu_device))
    held.of[0], held.position[0] = held.empty(), 0
    for r in (0, 1, 2):
        shared[r] = 0
    out_mask = [r != 0 for r in range(rows)]
    tables = cache.begin_step(active=torch.tensor(out_mask, device=gpu_device))
    assert cache.shared_lens.tolist() == [0, 32]
    for layer in range(layers):
        q, k, v = (torch.randn(rows, h, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for h in (hq, hkv, hkv))
        cache.write(layer, k.to(gpu_device), v.to(gpu_device))
        out = cache.attend(layer, q.to(gpu_device), scale).cpu()
        assert (out[0] == 0).all()
        for r in range(1, rows):
            held.add(r, layer, k[:, r:r + 1], v[:, r:r + 1])
            check(out[r:r + 1], *reference(q[:, r:r + 1], *held.of[r][layer][:2], scale, 0, 0), f"request {r}")
    cache.release(torch.ones(rows, dtype=torch.bool, device=gpu_device))
    assert cache.free_count.item() == cache.num_pages and sorted(cache._stack[:cache.num_pages].tolist()) == list(range(cache.num_pages))


def test_a_captured_step_of_groups(gpu_device):
    """A decode step of a cache with groups and weights, recorded once and replayed between evictions and releases."""
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(5)
    hq, hkv, d, page, rows, scale = 8, 2, 128, 16, 4, default_scale(128)
    make = lambda h, n: torch.randn(n, h, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1)
    cache = PagedKVCache(1, 64, hkv, d, rows, 300, page, device=gpu_device, group_sizes=[3], key_weights=True)
    cache.begin_step(torch.tensor([70, 0, 0, 20], dtype=torch.int32, device=gpu_device), 90)
    cache.write(0, make(hkv, 90), make(hkv, 90))
    cache.observe(0, make(hq, 90), scale)
    cache.share(0, 70)
    active = torch.ones(rows, dtype=torch.bool, device=gpu_device)
    q, k, v = (torch.zeros(rows, h, d, dtype=torch.bfloat16, device=gpu_device).transpose(0, 1) for h in (hq, hkv, hkv))
    out = torch.zeros(rows, hq, d, dtype=torch.bfloat16, device=gpu_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.begin_step(active=active)
        cache.write(0, k, v)
        cache.attend(0, q, scale, out=out)
    for i in range(12):
        for x, h in ((q, hq), (k, hkv), (v, hkv)):
            x.copy_(make(h, rows))
        active.copy_(torch.tensor([True, i != 3, i % 2 == 0, True]))
        state = [t.clone() for t in (cache.lens, cache.free_count, cache.block_table, cache.pools, cache.weights)]
        graph.replay()
        torch.cuda.synchronize()
        after = [t.clone() for t in (cache.lens, cache.free_count, cache.block_table, cache.pools, cache.weights)]
        replayed = out.clone()
        for t, s in zip((cache.lens, cache.free_count, cache.block_table, cache.pools, cache.weights), state):
            t.copy_(s)
        cache.begin_step(active=active)
        cache.write(0, k, v)
        assert torch.equal(cache.attend(0, q, scale)[active], replayed[active])
        for t, s in zip((cache.lens, cache.free_count, cache.block_table, cache.pools, cache.weights), after):
            assert torch.equal(t, s)
        if i == 5:
            cache.evict(10, 2, 1)
            assert cache.lens.tolist()[3] == 13 and cache.dropped.tolist()[3] == 13
        if i == 8:
            cache.release(torch.tensor([False, True, False, False], device=gpu_device))
            cache.join(torch.tensor([False, True, False, False], device=gpu_device))
            assert cache.lens.tolist()[1] == 64


def test_requests_of_a_group_that_share_nothing(gpu_device):
    """A group's first row ends before the others, which keep its pages through evictions, and rows of the group take requests that share nothing."""
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(6)
    hq, hkv, d, page, rows, scale = 8, 2, 64, 16, 4, default_scale(64)
    cache = PagedKVCache(1, 60, hkv, d, rows, 300, page, device=gpu_device, group_sizes=[4], key_weights=True)
    held = Held(1, rows, hkv, d)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    mask = lambda *r: torch.tensor([i in r for i in range(rows)], device=gpu_device)
    front = [0] * rows  # keys in pages of several

    def step(new=None, active=None):
        singles = new is None
        counts = [int(r in active) for r in range(rows)] if singles else new
        total = rows if singles else sum(new)
        tables = cache.begin_step(active=mask(*active)) if singles else cache.begin_step(ints(new), total)
        assert tables.free_left.item() >= 0
        q, k, v = (torch.randn(total, h, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for h in (hq, hkv, hkv))
        cache.write(0, k.to(gpu_device), v.to(gpu_device))
        out, at = cache.attend(0, q.to(gpu_device), scale).cpu(), 0
        if not singles:
            cache.observe(0, q.to(gpu_device), scale, last=4)
        for r, n in enumerate(counts):
            mine = slice(r, r + n) if singles else slice(at, at + n)
            if n:
                held.add(r, 0, k[:, mine], v[:, mine])
                check(out[mine], *reference(q[:, mine], *held.of[r][0][:2], scale, 0, 0), f"request {r}")
                seen = q[:, mine] if singles else q[:, mine][:, -4:]
                held.weigh(r, 0, seen, scale, front[r], singles)
            at += n

    def evict(budget, recent):
        got = [_check_weights(cache, held, r, 0, front[r]) for r in range(rows)]
        cache.evict(budget, recent)
        for r in range(rows):
            k, v, w, room = held.of[r][0]
            n, first = k.shape[1], front[r]
            mid = max(n - first - recent, 0)
            keep = min(mid, budget)
            stay = torch.tensor([list(range(first)) + sorted(first + i for i in sorted(range(mid), key=lambda i: (-got[r][h, first + i].item(), i))[:keep])
                                 + list(range(first + mid, n)) for h in range(hkv)])
            held.of[r] = [tuple(torch.stack([x[h, stay[h]] for h in range(hkv)]) for x in (k, v, w, room))]
            assert cache.lens[r].item() == stay.shape[1]

    step(new=[70, 0, 0, 0])
    cache.share(0, 70)
    front = [64] * rows
    for r in (1, 2, 3):
        held.of[r] = [tuple(x[:, :64].clone() for x in layer) for layer in held.of[0]]
    step(new=[2, 30, 25, 1])
    step(active=[0, 1, 2])
    cache.release(mask(0, 3))
    for r in (0, 3):
        held.of[r], front[r] = held.empty(), 0
    step(new=[150, 1, 3, 0])  # a request that shares nothing, in the first row
    step(new=[1, 1, 1, 90])   # and in another one
    for _ in range(3):
        step(active=[0, 1, 2, 3])
    evict(12, 5)
    step(active=[0, 1, 2, 3])
    cache.release(mask(2))
    held.of[2] = held.empty()
    cache.share(0, 16)  # of what the first row has now, to row 2 alone
    front[0] = front[2] = 16
    held.of[2] = [tuple(x[:, :16].clone() for x in layer) for layer in held.of[0]]
    assert cache.lens[2].item() == 16
    for _ in range(3):
        step(active=[0, 1, 2, 3])
    evict(3, 1)
    step(active=[1, 2, 3])
    step(new=[3, 4, 5, 6])
    cache.release(torch.ones(rows, dtype=torch.bool, device=gpu_device))
    assert cache.free_count.item() == 60


def test_new_keys_have_no_weight(gpu_device):
    """Places that earlier owners left weights in: 0 until something attends to the key."""
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(7)
    hq, hkv, d, page, rows, scale = 8, 2, 64, 16, 3, default_scale(64)
    cache = PagedKVCache(2, 20, hkv, d, rows, 100, page, device=gpu_device, key_weights=True)
    make = lambda n: [torch.randn(n, h, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1) for h in (hq, hkv, hkv)]

    def step(window, **kw):
        tables = cache.begin_step(**kw)
        for layer in range(2):
            q, k, v = make(tables.slots.numel())
            cache.write(layer, k, v)
            cache.attend(layer, q, scale, window=window)

    cache.weights.fill_(float("nan"))
    step(None, new_lens=torch.tensor([20, 0, 35], dtype=torch.int32, device=gpu_device), max_new_tokens=60)
    seen = lambda: [torch.stack([cache.weights[layer].cpu()[_places(cache, r, n)[0], :, _places(cache, r, n)[1]] for layer in range(2)])
                    for r, n in enumerate(cache.lens.tolist())]
    assert all((w == 0).all() for w in seen()) and cache.weights.isnan().sum().item() == 2 * hkv * (20 * page - 55)
    step(10, active=torch.tensor([True, False, True], device=gpu_device))
    assert [w.shape[1] for w in seen()] == [21, 0, 36] and all((w == 0).all() for w in seen())
    step(None, active=torch.tensor([True, True, True], device=gpu_device))
    for w in seen():  # the single tokens' weights sum to one a query head
        assert (w.double().sum(1) - hq // hkv).abs().max() < 1e-4


def test_a_captured_step_of_chunks(gpu_device):
    """A step of several tokens a request with its keys' weights, recorded once: every replay leaves what an eager twin has."""
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(8)
    hq, hkv, d, page, rows, most, scale = 8, 2, 64, 16, 4, 60, default_scale(64)
    caches = [PagedKVCache(1, 60, hkv, d, rows, 200, page, device=gpu_device, group_sizes=[3], key_weights=True) for _ in range(2)]
    q, k, v = (torch.zeros(most, h, d, dtype=torch.bfloat16, device=gpu_device).transpose(0, 1) for h in (hq, hkv, hkv))
    new, out = torch.zeros(rows, dtype=torch.int32, device=gpu_device), torch.zeros(most, hq, d, dtype=torch.bfloat16, device=gpu_device)

    def step(cache, to):
        cache.begin_step(new, most)
        cache.write(0, k, v)
        cache.attend(0, q, scale, out=to)
        cache.observe(0, q, scale, last=5, accumulate=True)

    step(caches[0], out)  # (nobody brings anything)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0], out)
    for i, counts in enumerate(([40, 0, 0, 7], [3, 20, 9, 1], [1, 2, 3, 4], [0, 5, 30, 25], [1, 1, 1, 1])):
        new.copy_(torch.tensor(counts, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape[1], x.shape[0], d, generator=gen).to(torch.bfloat16).transpose(0, 1))
        twin = torch.zeros_like(out)
        graph.replay()
        torch.cuda.synchronize()
        step(caches[1], twin)
        n = sum(counts)
        assert torch.equal(out[:n], twin[:n]), counts
        assert torch.equal(caches[0].weights, caches[1].weights) and torch.equal(caches[0].block_table, caches[1].block_table)
        assert torch.equal(caches[0].lens, caches[1].lens) and torch.equal(caches[0].pools, caches[1].pools)
        if i == 0:
            for c in caches:
                c.share(0, 33)
        if i == 2:
            for c in caches:
                c.evict(8, 4)
