"""Tensors with odd strides on axes of length one: the same bits as without."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _odd(t):
    """The same tensor with strides of 3 wherever an axis has length one."""
    return t.as_strided(t.shape, [3 if n == 1 else s for n, s in zip(t.shape, t.stride())], t.storage_offset())


@pytest.mark.parametrize("hq,hkv,n,nk,batch", [(4, 1, 1, 90, 1), (1, 1, 40, 90, 1), (4, 2, 1, 1, 1), (1, 1, 1, 1, 3), (2, 1, 1, 70, 2), (32, 1, 1, 1, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_window_attention(gpu_device, hq, hkv, n, nk, batch, d):
    from shareprefill_amd import ops

    make = lambda h, x: torch.randn(batch, h, x, d, device=gpu_device).to(torch.bfloat16)
    q, k, v = make(hq, n), make(hkv, nk), make(hkv, nk)
    want = ops.window_attention(q, k, v, 0.1, window=30, sinks=2)
    assert torch.equal(ops.window_attention(_odd(q), _odd(k), _odd(v), 0.1, window=30, sinks=2), want)


@pytest.mark.parametrize("hq,hkv,tokens", [(4, 1, 1), (1, 1, 7), (4, 2, 1), (20, 1, 1)])
@pytest.mark.parametrize("singles", [False, True])
def test_pages(gpu_device, hq, hkv, tokens, singles):
    from shareprefill_amd import ops

    d, page = 64, 16
    tokens = 1 if singles else tokens
    q = torch.randn(hq, tokens, d, device=gpu_device).to(torch.bfloat16)
    k, v = (torch.randn(hkv, tokens, d, device=gpu_device).to(torch.bfloat16) for _ in range(2))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    table = ints([[0]])
    results = []
    for view in (lambda x: x, _odd):
        pools = [torch.ones(1, hkv, page, d, device=gpu_device, dtype=torch.bfloat16) for _ in range(2)]
        slots = torch.arange(5, 5 + tokens, device=gpu_device)
        ops.paged_cache_write(view(k), view(v), *(view(x) for x in pools), slots)
        out = ops.paged_attention(view(q), *(view(x) for x in pools), view(table), ints([14]), 0.1, cu_q=None if singles else ints([0, tokens]))
        results.append((*pools, out))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert torch.equal(results[1][0][0, :, 5:5 + tokens], k)
