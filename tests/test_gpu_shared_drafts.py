"""A few tokens of every request (drafted ones, say), up to 16 rows each: against the definition in 64 bits."""

import pytest
import torch

from paged_reference import check, default_scale, starts
from shared_reference import make_shared, references

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _call(dev, q, pools, table, lens, shared, cu, cu_q, scale, **kw):
    from shareprefill_amd import ops

    return ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu), scale,
                                       cu_q=_ints(dev, cu_q), **kw)


@pytest.mark.parametrize("heads,most", [((8, 2, 128), 4), ((14, 2, 64), 2), ((7, 1, 128), 2), ((4, 4, 64), 16), ((32, 2, 128), 1)])
@pytest.mark.parametrize("groups,alone", [([(100, [40, 31, 33, 64])], [17, 300, 16]), ([], [1000, 70, 33, 32]), ([(64, [16, 17]), (31, [20] * 5)], [40]),
                                          ([(2000, [900] * 3)], [4000, 18])])
@pytest.mark.parametrize("page", [16, 128])
def test_a_few_tokens(gpu_device, heads, most, groups, alone, page):
    hq, hkv, d = heads
    gen = torch.Generator().manual_seed(page + most)
    pools, table, lens, shared, cu, kv, _ = make_shared(groups, alone, hkv, d, page, gen)
    for new in ([most] * len(lens), [1 + i * 7 % most for i in range(len(lens))], [i * 5 % (most + 1) for i in range(len(lens))]):
        q = torch.randn(max(sum(new), 1), hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
        out = _call(gpu_device, q, pools, table, lens, shared, cu, starts(new), default_scale(d))
        want, bound = references(q[:, :sum(new)], kv, new, default_scale(d))
        check(out[:sum(new)], want, bound, f"{new}")


def test_many_requests_and_all_lengths(gpu_device):
    """Requests of one to seventy keys, all of them new or one, more of them than there are parts."""
    hq, hkv, d = 4, 1, 64
    gen = torch.Generator().manual_seed(3)
    lens = [1 + i % 70 for i in range(900)]
    pools, table, _, shared, cu, kv, _ = make_shared([], lens, hkv, d, 16, gen)
    new = [min(1 + i % 4, n) for i, n in enumerate(lens)]
    q = torch.randn(sum(new), hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = _call(gpu_device, q, pools, table, lens, shared, cu, starts(new), default_scale(d))
    want, bound = references(q, kv, new, default_scale(d))
    check(out, want, bound)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_values_that_are_no_numbers(gpu_device, bad):
    """A new token's value that is not finite reaches its own row and those behind it, no others."""
    hq, hkv, d = 8, 2, 128
    gen = torch.Generator().manual_seed(4)
    pools, table, lens, shared, cu, kv, _ = make_shared([(48, [20, 25])], [30], hkv, d, 16, gen)
    new = [3, 4, 2]
    q = torch.randn(9, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    want, bound = references(q, kv, new, default_scale(d))
    j = lens[1] - 3  # the second of four
    pools[1][int(table[1, j // 16]), 0, j % 16, 5] = bad
    out = _call(gpu_device, q, pools, table, lens, shared, cu, starts(new), default_scale(d)).cpu()
    hit = torch.zeros(9, dtype=torch.bool)
    hit[4:7] = True
    check(out[~hit], want[~hit], bound[~hit])
    assert (~out[hit][:, :4, 5].isfinite()).all()
    check(out[hit][:, 4:], want[hit][:, 4:], bound[hit][:, 4:])


def test_offsets_that_go_back_and_rows_of_nobody(gpu_device):
    hq, hkv, d = 8, 2, 64
    gen = torch.Generator().manual_seed(5)
    pools, table, lens, shared, cu, kv, _ = make_shared([], [50, 20, 33, 70], hkv, d, 16, gen)
    q = torch.randn(20, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = torch.full((20, hq, d), 7.0, dtype=torch.bfloat16, device=gpu_device)
    _call(gpu_device, q, pools, table, lens, shared, cu, [3, 6, 4, 8, 10], default_scale(d), out=out)  # as 3, 6, 6, 8, 10
    assert (out[:3] == 7).all() and (out[10:] == 7).all()
    new = [3, 0, 2, 2]
    want, bound = references(q[:, 3:10], kv, new, default_scale(d))
    check(out[3:10], want, bound)


def test_replayed_between_few_tokens_and_many(gpu_device):
    """Recorded once, replayed with other numbers of tokens."""
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 128), 16
    gen = torch.Generator().manual_seed(6)
    pools, table, lens, shared, cu, kv, _ = make_shared([(64, [90, 80, 70])], [200], hkv, d, page, gen)
    q = torch.randn(100, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    on = [x.to(dev) for x in (q, *pools, table)]
    cu_q, out = _ints(dev, [0] * 5), torch.zeros(100, hq, d, dtype=torch.bfloat16, device=dev)
    call = lambda: ops.shared_prefix_attention(*on, _ints_of[0], _ints_of[1], _ints_of[2], default_scale(d), cu_q=cu_q, out=out)
    _ints_of = [_ints(dev, x) for x in (lens, shared, cu)]
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new in ([4, 4, 4, 4], [5, 4, 4, 4], [1, 0, 3, 2], [70, 1, 20, 9], [2, 2, 2, 2]):
        cu_q.copy_(_ints(dev, starts(new)))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want, bound = references(q[:, :sum(new)], kv, new, default_scale(d))
        check(got[:sum(new)], want, bound, f"{new}")
        call()
        assert torch.equal(out[:sum(new)], got[:sum(new)])
