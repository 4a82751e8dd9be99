"""Groups of many rows over tables with room for many keys, whose shared starts a launch of its own goes through: against the definition in 64 bits."""

import pytest
import torch

from paged_reference import check, default_scale, starts
from shared_reference import make_shared, references

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _room(table, tokens, heads, page):
    """The table, wide enough for tokens x heads x keys to pass 5e7; what lies behind a request's pages is never read."""
    width = max(table.shape[1], int(5.1e7 / (tokens * heads[0] * page)) + 1)
    assert width * page < 1 << 26
    return torch.cat((table, torch.full((table.shape[0], width - table.shape[1]), 1 << 30, dtype=torch.int32)), 1)


def _call(dev, q, pools, table, lens, shared, cu, new, heads, page, **kw):
    from shareprefill_amd import ops

    assert q.shape[1] * (heads[0] // heads[1]) > 256 * len(shared)
    return ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), _room(table, q.shape[1], heads, page).to(dev), _ints(dev, lens),
                                       _ints(dev, shared), _ints(dev, cu), kw.pop("scale", default_scale(heads[2])),
                                       cu_q=None if all(n == 1 for n in new) else _ints(dev, starts(new)), **kw)


CASES = [
    ([(100, [1 + i % 7 for i in range(70)])], [], None, (8, 2, 64), 64),
    ([(515, [1 + i % 40 for i in range(80)])], [33, 1], None, (14, 2, 64), 16),
    ([(1000, [30 + i for i in range(20)])], [50], [1 + 3 * (i % 9) for i in range(21)], (8, 2, 128), 128),
    ([(31, [64] * 9), (700, [20] * 40)], [5], [33] * 9 + [9] * 41, (7, 1, 128), 16),
    ([(0, [5] * 70), (257, [8] * 3), (64, [1])], [9], [8] * 73 + [1, 9], (28, 4, 128), 32),
    ([(3000, [400, 1, 300])], [600], [399, 1, 255, 600], (4, 4, 64), 256),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_groups_of_many_rows(gpu_device, case):
    groups, alone, new, heads, page = CASES[case]
    hq, hkv, d = heads
    gen = torch.Generator().manual_seed(20 + case)
    pools, table, lens, shared, cu, kv, _ = make_shared(groups, alone, hkv, d, page, gen)
    new = [1] * len(lens) if new is None else new
    q = torch.randn(sum(new), hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = _call(gpu_device, q, pools, table, lens, shared, cu, new, heads, page)
    want, bound = references(q, kv, new, default_scale(d))
    check(out, want, bound)


def test_far_logits_and_short_requests(gpu_device):
    """Logits of some 10^4; a request whose new tokens do not all stand behind the shared keys goes through them by itself."""
    hq, hkv, d = heads = (8, 2, 128)
    gen = torch.Generator().manual_seed(30)
    pools, table, lens, shared, cu, kv, _ = make_shared([(96, [20] * 30)], [70], hkv, d, 16, gen)
    new = [3] * 30 + [2]
    lens[4], kv[4] = 97, tuple(x[:, :97] for x in kv[4])
    lens[5], kv[5] = 40, tuple(x[:, :40] for x in kv[5])
    q = torch.randn(sum(new), hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = _call(gpu_device, q, pools, table, lens, shared, cu, new, heads, 16, scale=300.0)
    want, bound = references(q, kv, new, 300.0)
    check(out, want, bound)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_no_numbers(gpu_device, bad):
    hq, hkv, d = heads = (8, 2, 64)
    gen = torch.Generator().manual_seed(31)
    pools, table, lens, shared, cu, kv, _ = make_shared([(300, [6] * 66)], [30], hkv, d, 16, gen)
    new = [2] * 67
    q = torch.randn(134, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    want, bound = references(q, kv, new, default_scale(d))
    pools[1][int(table[0, 1]), 0, 3, 7] = bad
    out = _call(gpu_device, q, pools, table, lens, shared, cu, new, heads, 16).cpu()
    assert (~out[:132, :4, 7].isfinite()).all()
    check(out[132:], want[132:], bound[132:])
    check(out[:132, 4:], want[:132, 4:], bound[:132, 4:])


def test_pages_that_are_none_and_rows_of_nobody(gpu_device):
    from paged_reference import reference

    hq, hkv, d = heads = (8, 2, 128)
    gen = torch.Generator().manual_seed(32)
    pools, table, lens, shared, cu, kv, _ = make_shared([(64, [40] * 34)], [60], hkv, d, 16, gen)
    new = [2] * 35
    shown = [torch.ones(n, dtype=torch.bool) for n in lens]
    table[:34, 1] = -1
    for b in range(34):
        shown[b][16:32] = False
    table[7, 5] = 10 ** 6
    shown[7][80:96] = False
    q = torch.randn(75, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    to = torch.full((75, hq, d), 7.0, dtype=torch.bfloat16, device=gpu_device)
    from shareprefill_amd import ops
    out = ops.shared_prefix_attention(q.to(gpu_device), pools[0].to(gpu_device), pools[1].to(gpu_device), _room(table, 75, heads, 16).to(gpu_device),
                                      _ints(gpu_device, lens), _ints(gpu_device, shared), _ints(gpu_device, cu), default_scale(d),
                                      cu_q=_ints(gpu_device, [2 + x for x in starts(new)]), out=to)
    assert (out[:2] == 7).all() and (out[72:] == 7).all()
    for b in range(35):
        want, bound = reference(q[:, 2 + 2 * b:4 + 2 * b], *kv[b], default_scale(d), 0, 0, seen=shown[b])
        check(out[2 + 2 * b:4 + 2 * b], want, bound, f"request {b}")


def test_a_captured_step(gpu_device):
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 128), 16
    gen = torch.Generator().manual_seed(33)
    runs = [make_shared([(s, [20 + i % 5 for i in range(70)])], [a], hkv, d, page, gen, slack=x) for s, a, x in ((64, 9, 4), (100, 120, 30), (0, 300, 9))]
    table = _room(torch.full((71, max(r[1].shape[1] for r in runs)), -1, dtype=torch.int32), 71, (hq, hkv, d), page).to(dev)
    pages = max(r[0][0].shape[0] for r in runs)
    pools = [torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    lens, shared, cu = _ints(dev, [0] * 71), _ints(dev, [0]), _ints(dev, [0, 70])
    q = torch.zeros(71, hq, d, dtype=torch.bfloat16, device=dev).transpose(0, 1)
    out = torch.zeros(71, hq, d, dtype=torch.bfloat16, device=dev)
    call = lambda to: ops.shared_prefix_attention(q, *pools, table, lens, shared, cu, default_scale(d), out=to)
    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for r in runs * 2:
        for pool, x in zip(pools, r[0]):
            pool[:x.shape[0]].copy_(x)
        table[:, :r[1].shape[1]] = r[1].to(dev)
        lens.copy_(_ints(dev, r[2])), shared.copy_(_ints(dev, r[3]))
        qx = torch.randn(71, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
        q.copy_(qx)
        graph.replay()
        torch.cuda.synchronize()
        want, bound = references(qx, r[5], [1] * 71, default_scale(d))
        check(out, want, bound)
        eager = torch.zeros_like(out)
        call(eager)
        assert torch.equal(eager, out)


def test_offsets_that_go_back(gpu_device):
    """An offset counts as the largest in front of it: tokens that two requests seem to have are the first one's, and so is their group."""
    hq, hkv, d = heads = (8, 2, 128)
    gen = torch.Generator().manual_seed(34)
    pools, table, lens, shared, cu, kv, _ = make_shared([(64, [40, 30]), (96, [50] * 8)], [60], hkv, d, 16, gen)
    offsets = [0, 30, 22, 60, 50, 80, 90, 100, 110, 150, 160, 162]
    new, top = [], 0
    for a, b in zip(offsets, offsets[1:]):
        top = max(top, a)
        new.append(max(b - top, 0))
    q = torch.randn(162, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    from shareprefill_amd import ops
    out = ops.shared_prefix_attention(q.to(gpu_device), pools[0].to(gpu_device), pools[1].to(gpu_device), _room(table, 162, heads, 16).to(gpu_device),
                                      _ints(gpu_device, lens), _ints(gpu_device, shared), _ints(gpu_device, cu), default_scale(d), cu_q=_ints(gpu_device, offsets))
    assert len(new) == 11 and sum(new) == 162
    want, bound = references(q, kv, new, default_scale(d))
    check(out, want, bound)
