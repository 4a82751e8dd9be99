"""Calls of the operators for shared starts, key weights and evictions: what is refused in Python, other streams, pages far behind the pool's start."""

import pytest
import torch

from paged_reference import check, default_scale
from shared_reference import key_weights, make_shared, references, weight_bound

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.fixture
def case(gpu_device):
    hq, hkv, d, page = 8, 2, 64, 16
    gen = torch.Generator().manual_seed(1)
    pools, table, lens, shared, cu, kv, prefix = make_shared([(48, [30, 20])], [40], hkv, d, page, gen, fill=0.0)
    q = torch.randn(3, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    return dict(q=q.to(gpu_device), k=pools[0].to(gpu_device), v=pools[1].to(gpu_device), table=table.to(gpu_device), lens=_ints(gpu_device, lens),
                shared=_ints(gpu_device, shared), cu=_ints(gpu_device, cu), weights=torch.zeros(pools[0].shape[:3], device=gpu_device), kv=kv, q_cpu=q,
                prefix=prefix)


def _attend(c, **kw):
    from shareprefill_amd import ops

    at = {**c, **kw}
    return ops.shared_prefix_attention(at["q"], at["k"], at["v"], at["table"], at["lens"], at["shared"], at["cu"], at.get("scale", 0.125),
                                       **{x: at[x] for x in ("cu_q", "out", "joined") if x in at}, weights=at["weights"])


def test_attention_refuses(case, gpu_device):
    c = case
    wrong = [dict(q=c["q"].float()), dict(q=c["q"][:, :2]), dict(q=c["q"].cpu()), dict(k=c["k"].half()), dict(v=c["v"][:-1]), dict(table=c["table"].long()),
             dict(table=c["table"][:2]), dict(lens=c["lens"].long()), dict(shared=c["shared"].float()), dict(cu=c["cu"][:1]), dict(cu=c["cu"].cpu()),
             dict(weights=c["weights"].half()), dict(weights=c["weights"][:-1]), dict(weights=c["weights"].transpose(0, 2).contiguous().transpose(0, 2)),
             dict(weights=c["weights"].cpu()), dict(out=torch.zeros(3, 8, 64, device=gpu_device)), dict(joined=c["lens"][:2]), dict(joined=c["lens"].long()),
             dict(cu_q=_ints(gpu_device, [0, 1, 2, 3])), dict(weights=None, cu_q=_ints(gpu_device, [0, 1, 3]))]
    for kw in wrong:
        with pytest.raises((ValueError, TypeError, AssertionError)):
            _attend(c, **kw)
    for kw in (dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(ValueError, match="softmax_scale"):
            _attend(c, **kw)
    wide = torch.zeros(34, 3, 64, dtype=torch.bfloat16, device=gpu_device)
    with pytest.raises(NotImplementedError, match="16"):
        _attend(c, q=wide)  # 17 query heads a kv head, with weights
    assert _attend(c, q=wide, weights=None).shape == (3, 34, 64)
    assert (c["weights"] == 0).all()


def test_weights_and_eviction_refuse(case, gpu_device):
    from shareprefill_amd import ops

    c = case
    weigh = lambda **kw: ops.paged_key_weights(*[{**c, **kw}[x] for x in ("q", "k", "table", "lens")], {**c, **kw}.get("scale", 0.125), {**c, **kw}["weights"],
                                               **{x: kw[x] for x in ("cu_q", "first") if x in kw})
    evict = lambda budget=5, recent=2, **kw: ops.paged_evict(*[{**c, **kw}[x] for x in ("k", "v", "weights", "table", "lens")], budget, recent,
                                                             **{x: kw[x] for x in ("first",) if x in kw})
    for kw in (dict(q=c["q"].float()), dict(q=c["q"][:, :2]), dict(lens=c["lens"].long()), dict(weights=c["weights"].half()), dict(first=c["lens"][:2]),
               dict(first=c["lens"].long()), dict(cu_q=_ints(gpu_device, [0, 3])), dict(table=c["table"].cpu())):
        with pytest.raises((ValueError, TypeError, AssertionError)):
            weigh(**kw)
    with pytest.raises(ValueError, match="softmax_scale"):
        weigh(scale=-1.0)
    for kw in (dict(budget=-1), dict(recent=-1), dict(k=c["k"].cpu()), dict(k=c["k"][0]), dict(weights=c["weights"][:, :1]), dict(lens=c["lens"][:2]),
               dict(first=c["lens"].long()), dict(table=c["table"].long())):
        with pytest.raises((ValueError, TypeError, AssertionError)):
            evict(**kw)
    before = [c[x].clone() for x in ("k", "v", "weights", "lens")]
    assert (c["weights"] == 0).all() and torch.equal(c["lens"], before[3])


def test_no_rows_at_all(case, gpu_device):
    from shareprefill_amd import ops

    c, none = case, _ints(gpu_device, [0] * 4)
    q = c["q"][:, :0]
    assert _attend(c, q=q, cu_q=none, weights=None).shape == (0, 8, 64)
    c["weights"].fill_(3.0)
    ops.paged_key_weights(q, c["k"], c["table"], c["lens"], 0.125, c["weights"], cu_q=none)
    assert (c["weights"] == 3).all()


def test_on_another_stream_and_on_two_at_once(case, gpu_device):
    from shareprefill_amd import ops

    c, own = case, _ints(gpu_device, case["prefix"])

    def run():
        w = torch.zeros_like(c["weights"])
        out = _attend(c, weights=w)
        ops.paged_key_weights(c["q"], c["k"], c["table"], c["lens"], 0.125, w, accumulate=True, first=own)
        pools = [c["k"].clone(), c["v"].clone()]
        left = ops.paged_evict(*pools, w, c["table"], c["lens"], 7, 3, first=own)
        return out, w, *pools, left

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, want))


def test_pages_far_behind_the_pool_s_start(gpu_device):
    """Places past 2^32 bytes, pages' offsets past 2^31 elements."""
    from shareprefill_amd import ops

    hq, hkv, d, page, pages = 8, 8, 128, 256, 9000
    gen = torch.Generator().manual_seed(2)
    small, table, lens, shared, cu, kv, prefix = make_shared([(600, [300, 200, 1])], [700], hkv, d, page, gen, fill=0.0)
    shift = pages - small[0].shape[0]
    assert shift * hkv * page * d > 2 ** 31
    pools = [torch.empty(pages, hkv, page, d, dtype=torch.bfloat16, device=gpu_device) for _ in range(2)]
    for big, x in zip(pools, small):
        big[shift:] = x.to(gpu_device)
    weights = torch.zeros(pages, hkv, page, device=gpu_device)
    far = torch.where(table < 0, table, table + shift).to(gpu_device)
    q = torch.randn(4, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    scale = default_scale(d)
    out = ops.shared_prefix_attention(q.to(gpu_device), *pools, far, _ints(gpu_device, lens), _ints(gpu_device, shared), _ints(gpu_device, cu), scale, weights=weights)
    check(out, *references(q, kv, [1] * 4, scale))
    own = weights[shift:].cpu()
    again = torch.zeros_like(weights)
    ops.paged_key_weights(q.to(gpu_device), pools[0], far, _ints(gpu_device, lens), scale, again, first=_ints(gpu_device, prefix))
    for w, at in ((own, "attention"), (again[shift:].cpu(), "weights")):
        for b, (k, _) in enumerate(kv):
            j = torch.arange(prefix[b], lens[b])
            got = w[table[b].long()[j // page], :, j % page].t().double()
            want = key_weights(q[:, b:b + 1], k, scale)[:, prefix[b]:]
            assert ((got - want).abs() <= weight_bound(q[:, b:b + 1], k, scale) * want + 2.0 ** -23 * want).all(), at
    near = [x.clone() for x in (*[p[shift:].cpu() for p in pools], own)]
    at_start = [x.to(gpu_device) for x in near]
    left = ops.paged_evict(*pools, weights, far, _ints(gpu_device, lens), 40, 9, first=_ints(gpu_device, [512, 512, 512, 0]))
    left_near = ops.paged_evict(*at_start, table.to(gpu_device), _ints(gpu_device, lens), 40, 9, first=_ints(gpu_device, [512, 512, 512, 0]))
    assert torch.equal(left, left_near) and left.tolist() == [561, 561, 561, 49]
    for big, x in zip((*pools, weights), at_start):
        assert torch.equal(big[shift:], x)
