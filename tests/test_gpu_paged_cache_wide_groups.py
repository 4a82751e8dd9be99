"""Weights of a cache's keys under more than 16 query heads to a kv head, whose single tokens are weighed behind their attention."""

import pytest
import torch

from paged_reference import check, default_scale, reference
from test_gpu_paged_cache_groups import Held, _check_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d", [(32, 1, 128), (34, 2, 64)])
@pytest.mark.parametrize("sizes", [None, [3]])
def test_single_tokens_of_many_heads_have_weights(gpu_device, hq, hkv, d, sizes):
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(hq)
    rows, page, scale = 4, 16, default_scale(d)
    cache = PagedKVCache(1, 60, hkv, d, rows, 200, page, device=gpu_device, group_sizes=sizes, key_weights=True)
    cache.weights.fill_(float("nan"))  # (left by nobody that matters)
    held, front = Held(1, rows, hkv, d), [0] * rows

    def step(counts, singles):
        total = rows if singles else sum(counts)
        mask = torch.tensor([n > 0 for n in counts], device=gpu_device)
        cache.begin_step(active=mask) if singles else cache.begin_step(torch.tensor(counts, dtype=torch.int32, device=gpu_device), total)
        q, k, v = (torch.randn(total, h, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for h in (hq, hkv, hkv))
        cache.write(0, k.to(gpu_device), v.to(gpu_device))
        out, at = cache.attend(0, q.to(gpu_device), scale).cpu(), 0
        if not singles:
            cache.observe(0, q.to(gpu_device), scale, last=3)
        for r, n in enumerate(counts):
            mine = slice(r, r + n) if singles else slice(at, at + n)
            if n:
                held.add(r, 0, k[:, mine], v[:, mine])
                check(out[mine], *reference(q[:, mine], *held.of[r][0][:2], scale, 0, 0), f"request {r}")
                held.weigh(r, 0, q[:, mine] if singles else q[:, mine][:, -3:], scale, front[r], singles)
            at += n
        for r in range(rows):
            _check_weights(cache, held, r, 0, front[r])

    step([40, 0, 0, 21], False)
    if sizes:
        cache.share(0, 40)
        front = [32, 32, 32, 0]
        for r in (1, 2):
            held.of[r] = [tuple(x[:, :32].clone() for x in layer) for layer in held.of[0]]
    step([1, 7, 9, 2], False)
    for active in ([1, 1, 1, 1], [0, 1, 0, 1], [1, 1, 1, 0]):
        step(active, True)


def test_a_captured_step_of_many_heads(gpu_device):
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(3)
    hq, hkv, d, rows, page, scale = 40, 2, 64, 3, 16, default_scale(64)
    caches = [PagedKVCache(1, 30, hkv, d, rows, 100, page, device=gpu_device, key_weights=True) for _ in range(2)]
    q, k, v = (torch.randn(rows, h, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1) for h in (hq, hkv, hkv))
    out = torch.zeros(rows, hq, d, dtype=torch.bfloat16, device=gpu_device)

    def step(cache, to):
        cache.begin_step()
        cache.write(0, k, v)
        return cache.attend(0, q, scale, out=to)

    for cache in caches:
        step(cache, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0], out)
    for _ in range(4):
        q.copy_(torch.randn(rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step(caches[1], None), out) and torch.equal(caches[0].weights, caches[1].weights)
        assert caches[0].lens.tolist() == caches[1].lens.tolist()
