"""Weights of single tokens where the keys in front lie in pages of several requests that no group reads together: they stay as they were."""

import pytest
import torch

from paged_reference import check, default_scale
from shared_reference import key_weights, make_shared, references, weight_bound

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (14, 2, 64, 64), (16, 1, 64, 32)])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("grouped", [False, True])
def test_keys_in_front_are_not_weighed(gpu_device, hq, hkv, d, page, aligned, grouped):
    """Three requests name the same first pages, as a group or by themselves; one has a first key inside a page of its own, one behind its end, one has none."""
    from shareprefill_amd import ops

    dev, scale = gpu_device, default_scale(d)
    gen = torch.Generator().manual_seed(hq + page)
    pools, table, lens, shared, cu, kv, prefix = make_shared([(128, [300, 45, 1])], [77, 50, 33], hkv, d, page, gen)
    first = [128, 128, 128, 23, 60, 0]
    q = torch.randn(6, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    room = torch.rand(pools[0].shape[0], hkv, page + (0 if aligned else 3), generator=gen)
    live = room.to(dev)
    view, before = live[:, :, :page], room[:, :, :page]
    args = [x.to(dev) for x in (q, *pools, table)] + [_ints(dev, lens)] + ([_ints(dev, shared), _ints(dev, cu)] if grouped else [_ints(dev, []), _ints(dev, [0])])
    out = ops.shared_prefix_attention(*args, scale, weights=view, first=_ints(dev, first))
    check(out, *references(q, kv, [1] * 6, scale))
    got, want, slack = view.cpu().double(), before.double(), torch.zeros(before.shape, dtype=torch.float64)
    for b, n in enumerate(lens):
        new, rel = key_weights(q[:, b:b + 1], kv[b][0], scale), weight_bound(q[:, b:b + 1], kv[b][0], scale)
        for j in range(first[b], n):
            place = (int(table[b, j // page]), slice(None), j % page)
            want[place] = new[:, j] + (want[place] if j < n - 1 else 0)
            slack[place] = rel * new[:, j] + 2.0 ** -23 * want[place]
    assert ((got - want).abs() <= slack).all()
    assert torch.equal(got[slack == 0], before.double()[slack == 0])
    if not aligned:
        assert torch.equal(live.cpu()[:, :, page:], room[:, :, page:])
    # without weights it says nothing
    assert torch.equal(ops.shared_prefix_attention(*args, scale, first=_ints(dev, first)), ops.shared_prefix_attention(*args, scale))


def test_firsts_of_another_kind_are_refused(gpu_device):
    from shareprefill_amd import ops

    dev, gen = gpu_device, torch.Generator().manual_seed(1)
    pools, table, lens, shared, cu, _, _ = make_shared([(16, [5, 6])], [], 2, 64, 16, gen)
    q = torch.zeros(2, 8, 64, dtype=torch.bfloat16, device=dev).transpose(0, 1)
    args = (q, *(x.to(dev) for x in (*pools, table)), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu), 0.1)
    for first in (_ints(dev, [0]), _ints(dev, [0, 0]).long(), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="first"):
            ops.shared_prefix_attention(*args, first=first)


@pytest.mark.parametrize("hq", [8, 36])
def test_weights_in_pages_of_several_requests_stay_behind_the_end_of_a_first_row(gpu_device, hq):
    """And the requests' own keys are weighed as before, the same from run to run."""
    from shareprefill_amd import PagedKVCache

    hkv, d, page, rows, scale = 2, 64, 16, 8, default_scale(64)
    runs = []
    for _ in range(2):
        gen = torch.Generator().manual_seed(4)
        make = lambda n: [torch.randn(n, h, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1) for h in (hq, hkv, hkv)]
        cache = PagedKVCache(1, 80, hkv, d, rows, 400, page, device=gpu_device, group_sizes=[rows], key_weights=True)

        def step(**kw):
            q, k, v = make(cache.begin_step(**kw).slots.numel())
            cache.write(0, k, v)
            cache.attend(0, q, scale)
            return q

        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
        cache.observe(0, step(new_lens=ints([200] + [0] * 7), max_new_tokens=200), scale)
        cache.share(0, 200)
        step(new_lens=ints([0] + [3 + i for i in range(7)]), max_new_tokens=60)
        common = cache.block_table[1, :12].long()
        before = cache.weights[0, common].clone()
        assert before.sum() > 0 and (cache.block_table[1:, :12].long() == common).all()
        cache.release(torch.arange(rows, device=gpu_device) == 0)
        for i in range(3):
            step(active=torch.tensor([False] + [True] * 7, device=gpu_device))
            assert torch.equal(cache.weights[0, common], before)
        own = cache.weights[0, cache.block_table[1:, 12].long()]
        assert (own[:, :, :3].sum() > 0).item()
        runs.append(cache.weights.clone())
    assert torch.equal(*runs)
