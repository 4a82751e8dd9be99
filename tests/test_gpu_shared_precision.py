"""What attention over shared starts loses against the attention in 64 bits: probabilities enter the product with V as two bf16 values, so that a weight is off by 2^-16 of
itself (truncation leaves 2^-7 of it, whose rounding to bf16 takes 2^-9 of that) and 2^-23 (what the second value has at least), not by bf16's 2^-9."""

import pytest
import torch

from shared_reference import make_shared

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (14, 2, 64), (24, 1, 64)])
@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("at", [(35, 50), (75, 90), (20, 99)])  # (shared, side by side: one running maximum; own; one of either)
def test_two_keys_that_cancel(gpu_device, hq, hkv, d, new, at):
    _check_cancelling(gpu_device, hq, hkv, d, new, at, 4, 0)


@pytest.mark.parametrize("hq,hkv,d,new,members", [(8, 2, 128, 1, 70), (14, 2, 64, 3, 14), (24, 1, 64, 1, 12)])
@pytest.mark.parametrize("at", [(35, 50), (20, 99)])
def test_two_keys_that_cancel_in_a_launch_of_their_own(gpu_device, hq, hkv, d, new, members, at):
    """More than 256 rows, and a table with room for 3e7 keys times tokens and heads."""
    _check_cancelling(gpu_device, hq, hkv, d, new, at, members, 160000)


def _check_cancelling(gpu_device, hq, hkv, d, new, at, members, room_of_table):
    """Two keys of nearly the same weight have all of it, and values of either sign: what is left of them is small, and a weight's rounding shows."""
    from shareprefill_amd import ops

    dev, page = gpu_device, 16
    gen = torch.Generator().manual_seed(hq + new)
    pools, table, lens, shared, cu, kv, _ = make_shared([(70, [40 + i for i in range(members)])], [], hkv, d, page, gen)
    q = 0.125 * torch.randn(members * new, hq, d, generator=gen)
    q[:, :, 0], q[:, :, 1] = 4.0, torch.rand(members * new, hq, generator=gen)
    q = q.to(torch.bfloat16).transpose(0, 1)
    one = torch.zeros(2, d)
    one[1, 1] = 0.25
    value = torch.zeros(2, d)
    value[0], value[1] = 1.0, -1.0
    pools[0][..., 0] = -8.0  # (32 below the two)
    for k, _ in kv:
        k[..., 0] = -8.0
    for b in range(members):
        for i, j in enumerate(at):
            kv[b][0][:, j], kv[b][1][:, j] = one[i].to(torch.bfloat16), value[i].to(torch.bfloat16)
            pools[0][table[b, j // page], :, j % page], pools[1][table[b, j // page], :, j % page] = one[i].to(torch.bfloat16), value[i].to(torch.bfloat16)
    if room_of_table:
        table = torch.cat((table, torch.full((members, room_of_table // page - table.shape[1]), -1, dtype=torch.int32)), 1).contiguous()
    out = ops.shared_prefix_attention(q.to(dev), *(x.to(dev) for x in pools), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu), 1.0,
                                      cu_q=None if new == 1 else _ints(dev, [new * b for b in range(members + 1)]))
    for b, n in enumerate(lens):
        for i in range(new):
            seen = n - new + i + 1
            for h in range(hq):
                k, v = (x[h // (hq // hkv), :seen].double() for x in kv[b])
                x = q[h, b * new + i].double()
                w = torch.softmax(k @ x, 0)
                want, size = w @ v, w @ v.abs()
                # the two's logits by (D + 4) 2^-24 of their terms, exponentials 2^-21, sums 2^-24 a term; the weights; the output's rounding.  (The others weigh
                # e^-32 at most, twice that if their logits are off by 2^-14 of 35.)
                e = 2 * (d + 4) * 2.0 ** -24 * (k[list(at)].abs() @ x.abs()).max() + 2.0 ** -20 + (seen + 8) * 2.0 ** -24
                off = (e + 2.0 ** -16 + 2.0 ** -22) * (size + want.abs()) + seen * 4.0 * 2.0 ** -46
                room = off + 2.0 ** -8 * (want.abs() + off)
                assert ((out[b * new + i, h].cpu().double() - want).abs() <= room).all(), (b, i, h)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("at", [10, 90])
def test_an_infinite_value_makes_an_infinity(gpu_device, sign, at):
    from shareprefill_amd import ops

    dev, page, hq, hkv, d = gpu_device, 16, 8, 2, 128
    gen = torch.Generator().manual_seed(2)
    pools, table, lens, shared, cu, kv, _ = make_shared([(70, [40, 35])], [33], hkv, d, page, gen)
    for b in (0, 1):
        pools[1][table[b, at // page], :, at % page, 5] = sign * float("inf")
    q = torch.randn(3, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    out = ops.shared_prefix_attention(q.to(dev), *(x.to(dev) for x in pools), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu), d ** -0.5).cpu()
    assert (out[:2, :, 5] == sign * float("inf")).all() and out[:2, :, :5].isfinite().all() and out[:2, :, 6:].isfinite().all() and out[2].isfinite().all()


def test_large_values_behind_a_row_take_no_part(gpu_device):
    """The second of two tokens has a value of bf16's largest, which the first does not see."""
    from shareprefill_amd import ops

    dev, page, hq, hkv, d = gpu_device, 16, 8, 2, 64
    gen = torch.Generator().manual_seed(3)
    pools, table, lens, shared, cu, kv, _ = make_shared([(32, [9, 30])], [20], hkv, d, page, gen)
    clean = [x.clone() for x in pools]
    for b, n in enumerate(lens):
        pools[1][table[b, (n - 1) // page], :, (n - 1) % page] = torch.finfo(torch.bfloat16).max
    q = torch.randn(6, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    call = lambda p: ops.shared_prefix_attention(q.to(dev), *(x.to(dev) for x in p), table.to(dev), _ints(dev, lens), _ints(dev, shared), _ints(dev, cu),
                                                 d ** -0.5, cu_q=_ints(dev, [0, 2, 4, 6])).cpu()
    assert torch.equal(call(pools)[::2], call(clean)[::2])
