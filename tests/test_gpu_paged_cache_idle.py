"""Decode steps of a server that is not full: requests that stand still, and rows of none, get no token and no page, and a prompt that comes to
such a row later finds it empty (paged_reference.py holds the bound)."""

import pytest
import torch

from paged_reference import default_scale
from test_gpu_paged_cache_rows import D, HKV, HQ, Server

pytestmark = pytest.mark.gpu


def _single(server, active, what):
    cache, n = server.cache, len(active)
    tables = cache.begin_step(active=torch.tensor(active, device=server.dev))
    q, k, v = server.rows(n)
    cache.write(0, k.to(server.dev), v.to(server.dev))
    out = cache.attend(0, q.to(server.dev), default_scale(D), window=server.window, sinks=server.sinks).cpu()
    before = [h[0].shape[1] for h in server.held]
    server.verify(out, [int(x) for x in active], list(range(n)), q, k, v, what)
    assert (out[~torch.tensor(active)] == 0).all()
    assert tables.positions.tolist() == [p if x else 0 for p, x in zip(before, active)]
    assert tables.slots.tolist() == [cache.block_table[r, p // 16].item() * 16 + p % 16 if x else -1 for r, (p, x) in enumerate(zip(before, active))]
    assert tables.seq_lens.tolist() == [p + x for p, x in zip(before, active)]


@pytest.mark.parametrize("window,sinks", [(None, 0), (25, 2)])
def test_requests_that_end_and_come(gpu_device, window, sinks):
    server = Server(gpu_device, 4, 3, window, sinks)
    server.step((20, 0, 31, 16), 67, "prompts")
    for i, active in enumerate([(True, False, True, True), (True, False, False, True), (True, False, True, True)]):
        _single(server, active, f"step {i}")
    server.cache.release(torch.tensor([False, False, True, False], device=gpu_device))
    server.held[2] = (torch.zeros(HKV, 0, D, dtype=torch.bfloat16),) * 2
    for i in range(18):
        _single(server, (True, False, False, i % 3 == 0), f"after the release {i}")
    # a prompt comes to the row that was given back and to the one that never was used; the others go on beside them
    server.step((1, 40, 25, 1), 67, "two prompts")
    _single(server, (True,) * 4, "all")
    _single(server, (False,) * 4, "none")
    _single(server, (False, True, True, False), "the new ones")


def test_a_captured_step_follows_its_mask(gpu_device):
    server = Server(gpu_device, 3, 4)
    server.step((30, 7, 0), 37)
    cache, dev = server.cache, gpu_device
    active = torch.zeros(3, dtype=torch.bool, device=dev)
    q_in, k_in, v_in = (torch.zeros(3, h, D, dtype=torch.bfloat16, device=dev).transpose(0, 1) for h in (HQ, HKV, HKV))
    out = torch.zeros(3, HQ, D, dtype=torch.bfloat16, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.begin_step(active=active)
        cache.write(0, k_in, v_in)
        cache.attend(0, q_in, default_scale(D), out=out)
    for i, mask in enumerate([(1, 1, 0), (0, 1, 0), (1, 1, 1), (0, 0, 0), (1, 0, 1), (0, 1, 1)]):
        active.copy_(torch.tensor(mask, dtype=torch.bool, device=dev))
        q, k, v = server.rows(3)
        q_in.copy_(q), k_in.copy_(k), v_in.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu()
        server.verify(got, mask, [0, 1, 2], q, k, v, f"replay {i}")
        assert (got[~torch.tensor(mask, dtype=torch.bool)] == 0).all()


def test_refusals(gpu_device):
    cache = Server(gpu_device, 3, 5).cache
    mask = torch.ones(3, dtype=torch.bool, device=gpu_device)
    for kw in (dict(active=mask[:2]), dict(active=mask.int()), dict(active=mask.cpu()),
               dict(active=mask, new_lens=mask.int(), max_new_tokens=3)):
        with pytest.raises(ValueError):
            cache.begin_step(**kw)
    cache.begin_step(active=mask)
