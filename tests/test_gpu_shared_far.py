"""Logits far from zero behind shared starts, as in test_gpu_attention_far_logits.py: every key's channels are one power of two, the query's another, so that keys either share
a row's largest logit or lie thousands of octaves below it, and a row is the mean of the values that share it.  |out - mean| <= 2^-8 |mean| 1.01 + n 2^-24 mean |v| for
weights that are equal and rounded alike, and 2^-16 of the values for the sides of a row, whose probabilities have one part or two."""

import pytest
import torch

from shared_reference import make_shared

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("q_exp,k_exp", [(3, 3), (12, 10), (14, 12), (20, 20), (40, 40), (58, 55)])
@pytest.mark.parametrize("three", [1, 3])
@pytest.mark.parametrize("d,new,members,prefix,width", [(128, 1, 5, 300, 0), (64, 3, 4, 200, 0), (128, 40, 4, 1030, 320), (64, 1, 90, 600, 560)])
@pytest.mark.parametrize("where", ["everywhere", "shared", "own"])
def test_rows_are_the_mean_of_the_largest_logits(gpu_device, sign, q_exp, k_exp, three, d, new, members, prefix, width, where):
    """The last two, whose tables have room for many keys, go to the launch for groups of many rows.  The keys that weigh are among all, among the shared or among the
    own ones alone."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(q_exp)
    hq, hkv, page, own = 16, 2, 64, 45
    pools, table, lens, shared, cu, kv, _ = make_shared([(prefix, [own] * members)], [], hkv, d, page, gen, fill=0.0)
    total = prefix + own
    weigh = torch.rand(total, generator=gen) < 0.3
    weigh[:prefix] &= where != "own"
    weigh[prefix:] &= where != "shared"
    weigh[0], weigh[prefix] = where != "own", where != "shared"
    low = -(2.0 ** k_exp) if sign > 0 else 2.0 ** (k_exp + 1)
    keys = torch.where(weigh, 2.0 ** k_exp, low).to(torch.bfloat16)
    j = torch.arange(total)
    for b in range(members):
        pools[0][table[b].long()[j // page], :, j % page] = keys[:, None, None].expand(total, hkv, d)
    if width:
        table = torch.cat((table, torch.full((members, width - table.shape[1]), -1, dtype=torch.int32)), 1).contiguous()
    q = torch.full((hq, members * new, d), three * sign * 2.0 ** q_exp, dtype=torch.bfloat16)
    out = ops.shared_prefix_attention(q.to(gpu_device), *(x.to(gpu_device) for x in pools), table.to(gpu_device), _ints(gpu_device, lens), _ints(gpu_device, shared),
                                      _ints(gpu_device, cu), 1.0, cu_q=None if new == 1 else _ints(gpu_device, [new * b for b in range(members + 1)])).cpu().double()
    for b in range(members):
        v = kv[b][1]
        for i in (range(new) if new < 10 else (0, new // 2, new - 1)):
            top = weigh & (j <= total - new + i)
            want = v[:, top].double().mean(1).repeat_interleave(hq // hkv, 0)
            room = want.abs() * 2.0 ** -8 * 1.01 + (total * 2.0 ** -24 + 2.0 ** -16) * v.double().abs().mean() * 2
            assert ((out[b * new + i] - want).abs() <= room).all(), (b, i)
