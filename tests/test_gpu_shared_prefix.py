"""Attention over requests that share a start against the definition in 64 bits, request by request."""

import pytest
import torch

from paged_reference import check, default_scale, starts
from shared_reference import key_weights, make_shared, references, weight_bound

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 128), (14, 2, 64), (7, 1, 128), (4, 4, 64)]


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _run(dev, groups, alone, new, heads, page, seed=0, weigh=False, scale=None, fill=float("nan")):
    from shareprefill_amd import ops

    hq, hkv, d = heads
    gen = torch.Generator().manual_seed(seed)
    pools, table, lens, shared, cu, kv, prefix = make_shared(groups, alone, hkv, d, page, gen, fill=fill)
    new = [1] * len(lens) if new is None else new
    total = sum(new)
    q = torch.randn(total, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    scale = scale or default_scale(d)
    weights = torch.rand(pools[0].shape[:3], generator=gen) if weigh else None
    live = weights.to(dev) if weigh else None
    out = ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu),
                                      scale, cu_q=None if all(n == 1 for n in new) else _ints(dev, starts(new)), weights=live)
    want, bound = references(q, kv, new, scale)
    check(out, want, bound, f"{groups} {alone} {new}")
    if weigh:
        for b, (k, _) in enumerate(kv):
            if lens[b] == 0:
                continue
            w = key_weights(q[:, b:b + 1], k, scale)
            rel = weight_bound(q[:, b:b + 1], k, scale)
            for j in range(prefix[b], lens[b]):
                at = (int(table[b, j // page]), slice(None), j % page)
                old = weights[at].double() if j < lens[b] - 1 else torch.zeros(hkv, dtype=torch.float64)
                expect = w[:, j] + old
                assert ((live[at].cpu().double() - expect).abs() <= rel * w[:, j] + 2.0 ** -23 * expect).all(), (b, j)
                weights[at] = live[at].cpu()
        assert torch.equal(live.cpu(), weights), "a place of no key changed"
    return out


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("members", [1, 3, 17])
@pytest.mark.parametrize("shared", [1, 31, 32, 100, 515])
def test_single_tokens(gpu_device, page, heads, members, shared):
    owns = [1 + (7 * i + shared) % 90 for i in range(members)]
    _run(gpu_device, [(shared, owns)], [], None, heads, page, seed=members + shared)


@pytest.mark.parametrize("heads", HEADS)
def test_groups_beside_requests_that_share_nothing(gpu_device, heads):
    _run(gpu_device, [(64, [1, 2, 3]), (0, [5, 9]), (200, [40] * 5), (33, [70])], [1, 300, 64], None, heads, 32, weigh=heads[0] // heads[1] <= 16)
    _run(gpu_device, [], [1, 17, 500], None, heads, 16, weigh=True)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("new", [[2, 1, 4, 3], [9, 1, 1, 30], [0, 3, 0, 2], [70, 1, 33, 2]])
def test_several_tokens_of_a_request(gpu_device, heads, new):
    _run(gpu_device, [(90, [max(new[0], 1), new[1] + 60, max(new[2], 1)])], [new[3] + 5], new, heads, 16, seed=sum(new))


@pytest.mark.parametrize("members", [40, 130])
def test_many_rows_and_cuts(gpu_device, members):
    """Groups of many row tiles, and lines that are cut inside shared keys and inside a request's own."""
    _run(gpu_device, [(1000, [1 + i % 7 for i in range(members)])], [3000], None, (8, 2, 64), 64, weigh=True)


def test_one_request_over_every_workgroup(gpu_device):
    _run(gpu_device, [(6000, [2000])], [], None, (4, 1, 64), 128, weigh=True)
    _run(gpu_device, [], [9000], None, (4, 1, 128), 16, weigh=True)


def test_idle_requests_and_short_ones_take_no_part(gpu_device):
    """Rows whose request has no keys are zero, and one whose new token lies in front of the shared length is computed by itself."""
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 128), 16
    gen = torch.Generator().manual_seed(5)
    pools, table, lens, shared, cu, kv, _ = make_shared([(64, [30, 20, 10, 5])], [], hkv, d, page, gen)
    lens[2], kv[2] = 40, tuple(x[:, :40] for x in kv[2])  # (its table still names the shared pages)
    lens[3], kv[3] = 0, tuple(x[:, :0] for x in kv[3])
    q = torch.randn(4, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu),
                                      default_scale(d))
    want, bound = references(q, kv[:3], [1, 1, 1], default_scale(d))
    check(out[:3], want, bound)
    assert (out[3] == 0).all()


@pytest.mark.parametrize("heads", [(8, 2, 128), (14, 2, 64)])
def test_rows_outside_every_request_stay(gpu_device, heads):
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, heads, 32
    gen = torch.Generator().manual_seed(6)
    pools, table, lens, shared, cu, kv, _ = make_shared([(70, [12, 30])], [9], hkv, d, page, gen)
    q = torch.randn(20, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = torch.full((20, hq, d), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu),
                                      default_scale(d), cu_q=_ints(dev, [2, 7, 7 + 9, 18]), out=out)
    assert got is out and (out[:2] == 7).all() and (out[18:] == 7).all()
    want, bound = references(q[:, 2:18], kv, [5, 9, 2], default_scale(d))
    check(out[2:18], want, bound)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_no_numbers(gpu_device, bad):
    """A new token's value that is not finite makes the rows at and behind it not finite and leaves those in front of it alone; one of the shared keys
    reaches all."""
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (4, 1, 128), 16
    gen = torch.Generator().manual_seed(8)
    pools, table, lens, shared, cu, kv, _ = make_shared([(48, [20, 25])], [30], hkv, d, page, gen)
    new = [6, 7, 8]
    q = torch.randn(21, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    call = lambda: ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared),
                                               _ints(dev, cu), default_scale(d), cu_q=_ints(dev, starts(new))).cpu()
    want, bound = references(q, kv, new, default_scale(d))
    for b, at in ((0, 3), (2, 0)):  # the value of a request's new token number `at`
        j = lens[b] - new[b] + at
        place = (int(table[b, j // page]), 0, j % page, 5)
        kept, pools[1][place] = pools[1][place].clone(), bad
        out, row = call(), starts(new)[b] + at
        hit = torch.zeros(21, dtype=torch.bool)
        hit[row:starts(new)[b + 1]] = True
        check(out[~hit], want[~hit], bound[~hit], f"request {b}")
        assert (~out[hit].isfinite()).reshape(int(hit.sum()), hq, -1).any(2).all()
        pools[1][place] = kept
    pools[1][int(table[0, 1]), 0, 3, 7] = bad
    out = call()
    assert (~out[:13, :, 7].isfinite()).all()
    check(out[13:], want[13:], bound[13:])


def test_far_logits(gpu_device):
    """Logits of some 10^4: the weight lies on the largest one."""
    _run(gpu_device, [(100, [30, 1, 64])], [50], None, (8, 2, 128), 16, scale=300.0, weigh=False)
    _run(gpu_device, [(100, [30, 5, 64])], [50], [3, 2, 1, 4], (8, 2, 64), 16, scale=300.0)


def test_pages_that_are_none_are_not_seen(gpu_device):
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 128), 16
    gen = torch.Generator().manual_seed(9)
    pools, table, lens, shared, cu, kv, _ = make_shared([(64, [40, 50])], [60], hkv, d, page, gen)
    shown = [torch.ones(n, dtype=torch.bool) for n in lens]
    for b, at, entry in ((0, 1, -1), (0, 5, 10 ** 6), (2, 0, -7)):
        table[b, at] = entry
        shown[b][at * page:(at + 1) * page] = False
        if at * page < 64 and b == 0:
            table[1, at] = entry
            shown[1][at * page:(at + 1) * page] = False
    q = torch.randn(3, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu),
                                      default_scale(d))
    from paged_reference import reference
    for b in range(3):
        want, bound = reference(q[:, b:b + 1], *kv[b], default_scale(d), 0, 0, seen=shown[b])
        check(out[b:b + 1], want, bound, f"request {b}")


def test_strided_pools_and_queries(gpu_device):
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 64), 32
    gen = torch.Generator().manual_seed(10)
    pools, table, lens, shared, cu, kv, _ = make_shared([(80, [20, 33])], [7], hkv, d, page, gen)
    token_major = [p.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for p in pools]
    wide = torch.full((3, table.shape[1] + 5), 99, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table.to(dev)
    weights = torch.zeros(pools[0].shape[0], hkv + 3, page + 4, device=dev)
    view = weights[:, 1:1 + hkv, :page]
    q = torch.randn(hq, 3, d + 8, generator=gen).to(torch.bfloat16)[:, :, :d]
    qg = torch.zeros(hq, 3, d + 8, dtype=torch.bfloat16, device=dev)[:, :, :d]
    qg.copy_(q)
    out = ops.shared_prefix_attention(qg, *token_major, wide[:, :table.shape[1]], _ints(dev, lens), _ints(dev, shared), _ints(dev, cu),
                                      default_scale(d), weights=view)
    want, bound = references(q, kv, [1, 1, 1], default_scale(d))
    check(out, want, bound)
    total = sum(hq * (1 - key_weights(q[:, b:b + 1], kv[b][0], default_scale(d))[:, :80 if b < 2 else 0].sum().item() / hq) for b in range(3))
    assert abs(view.double().sum().item() - total) < 1e-4
    view.zero_()
    assert (weights == 0).all()


def test_a_captured_step(gpu_device):
    """Recorded once, replayed with other lengths, prefixes and pages."""
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 128), 16
    gen = torch.Generator().manual_seed(11)
    runs = [make_shared(g, a, hkv, d, page, gen, slack=s) for g, a, s in (([(64, [30, 20, 10])], [9], 40), ([(100, [3, 2, 1])], [120], 37), ([(0, [5, 6, 7])], [300], 30))]
    width, pages = max(r[1].shape[1] for r in runs), max(r[0][0].shape[0] for r in runs)
    table = torch.full((4, width), -1, dtype=torch.int32, device=dev)
    pools = [torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    lens, shared, cu = _ints(dev, [0] * 4), _ints(dev, [0]), _ints(dev, [0, 3])
    q = torch.zeros(4, hq, d, dtype=torch.bfloat16, device=dev).transpose(0, 1)
    weights = torch.zeros(pages, hkv, page, device=dev)
    out = torch.zeros(4, hq, d, dtype=torch.bfloat16, device=dev)
    call = lambda to: ops.shared_prefix_attention(q, *pools, table, lens, shared, cu, default_scale(d), weights=weights, out=to)
    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for r in runs * 2:
        for pool, x in zip(pools, r[0]):
            pool[:x.shape[0]].copy_(x)
        table.fill_(-1)
        table[:, :r[1].shape[1]] = r[1].to(dev)
        lens.copy_(_ints(dev, r[2])), shared.copy_(_ints(dev, r[3]))
        qx = torch.randn(4, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
        q.copy_(qx)
        weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, bound = references(qx, r[5], [1] * 4, default_scale(d))
        check(out, want, bound)
        kept, replayed = weights.clone(), out.clone()
        weights.zero_()
        assert torch.equal(call(None), replayed) and torch.equal(weights, kept), "a replay differs from the eager call"


@pytest.mark.parametrize("single", [True, False])
def test_requests_that_have_not_joined(gpu_device, single):
    """They go through all of their keys by themselves, though the group's are as long."""
    from shareprefill_amd import ops

    dev, (hq, hkv, d), page = gpu_device, (8, 2, 128), 16
    gen = torch.Generator().manual_seed(12)
    pools, table, lens, shared, cu, kv, prefix = make_shared([(64, [30, 20])], [90, 70], hkv, d, page, gen)
    new = [1] * 4 if single else [2, 5, 3, 1]
    q = torch.randn(sum(new), hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    weights = torch.zeros(pools[0].shape[:3], device=dev) if single else None
    # (all four rows are the group's; the last two share nothing with it)
    out = ops.shared_prefix_attention(q.to(dev), pools[0].to(dev), pools[1].to(dev), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, [0, 4]),
                                      default_scale(d), cu_q=None if single else _ints(dev, starts(new)), weights=weights, joined=_ints(dev, [64, 90, 63, -5]))
    want, bound = references(q, kv, new, default_scale(d))
    check(out, want, bound)
    if single:
        total = sum(hq - key_weights(q[:, b:b + 1], kv[b][0], default_scale(d))[:, :prefix[b]].sum().item() for b in range(4))
        assert abs(weights.double().sum().item() - total) < 1e-3  # (8 rows of weights that sum to one, 2^-20 each at most)
