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
