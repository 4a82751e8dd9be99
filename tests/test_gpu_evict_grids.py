"""Evictions of more chunks than a launch has workgroups for: those take chunk after chunk."""

import pytest

from test_gpu_evict import _run

pytestmark = pytest.mark.gpu


def test_a_workgroup_a_stream(gpu_device):
    """4096 requests: 12288 streams of K, V and weights, a workgroup each; of 96 rows a chunk."""
    lens = [0] * 4096
    lens[0], lens[5], lens[4000], lens[4095] = 2000, 700, 90, 1500
    _run(gpu_device, lens, 1100, 30, hkv=1, d=512, page=64, seed=1)


def test_as_many_chunks_as_a_long_table_has_room_for(gpu_device):
    """12288 streams of 345 chunks: more workgroups of 1024 threads than a launch may have, if each had one."""
    _run(gpu_device, [40000] + [0] * 4094 + [3], 33000, 100, hkv=1, d=512, page=1024, seed=2)


def test_few_workgroups_a_stream(gpu_device):
    """9000 streams, one workgroup each; 2520 of rows of three slices, three workgroups each for seven chunks."""
    _run(gpu_device, [2500] + [0] * 298 + [60], 1700, 9, hkv=10, d=64, page=16, seed=3)
    _run(gpu_device, [0, 0, 50, 0, 900, 0], 600, 9, hkv=60, d=1032, page=16, seed=4)


@pytest.mark.parametrize("batch,d", [(3, 64), (4096, 256)])
def test_replays_of_an_eviction(gpu_device, batch, d):
    """Recorded once, replayed with other lengths and weights: each replay is the eager call, also where workgroups take several chunks."""
    import torch

    from shareprefill_amd import ops

    gen = torch.Generator(device=gpu_device).manual_seed(batch)
    page, most, width = 64, 3, 24
    table = torch.full((batch, width), -1, dtype=torch.int32, device=gpu_device)
    table[:most] = torch.randperm(most * width, generator=gen, device=gpu_device).to(torch.int32).view(most, width)
    k, v = (torch.randn(most * width, 1, page, d, generator=gen, device=gpu_device).to(torch.bfloat16) for _ in range(2))
    w, lens = torch.zeros(most * width, 1, page, device=gpu_device), torch.zeros(batch, dtype=torch.int32, device=gpu_device)
    ops.paged_evict(k, v, w, table, lens, 700, 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        left = ops.paged_evict(k, v, w, table, lens, 700, 20)
    for n in ([1500, 60, 1000], [0, 721, 719], [1536, 1536, 1536], [720, 900, 1]):
        w.copy_(torch.rand(w.shape, generator=gen, device=gpu_device))
        lens[:most] = torch.tensor(n, dtype=torch.int32, device=gpu_device)
        twin = [x.clone() for x in (k, v, w)]
        graph.replay()
        torch.cuda.synchronize()
        want = ops.paged_evict(*twin, table, lens, 700, 20)
        assert torch.equal(left, want) and want.tolist()[:most] == [min(x, 720) for x in n]
        assert all(torch.equal(x, y) for x, y in zip((k, v, w), twin))
