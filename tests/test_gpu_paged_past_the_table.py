"""Requests that are longer than their rows of the block table: what has no page is not seen, and a window is counted from the row's own
position, on the kernel for many new tokens and on the one for single ones alike (paged_reference.py holds the bound)."""

import pytest
import torch

from paged_reference import check, default_scale, make_pages, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(111, 0), (112, 0), (113, 4), (130, 0), (150, 20), (1 << 20, 0), (0, 0), (112, 111), (112, 112), (40, 500)])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 16), (128, 112)])
def test_a_window_at_and_above_the_tables_room(gpu_device, window, sinks, d, page):
    from shareprefill_amd import ops

    if page == 112:
        page, room = 128, 128
    else:
        room = 112
    gen = torch.Generator().manual_seed(window + sinks + d)
    hq, hkv, rows, lens = 4, 2, 20, [150, 300, room, 90]
    kp, vp, table, kv = make_pages(lens, hkv, d, page, gen)
    width = room // page
    q = torch.randn(len(lens) * rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    args = kp.to(gpu_device), vp.to(gpu_device), table[:, :width].contiguous().to(gpu_device), ints(lens), default_scale(d)
    kw = dict(window=window or None, sinks=sinks)
    got = ops.paged_attention(q.to(gpu_device), *args, cu_q=ints([rows * b for b in range(len(lens) + 1)]), **kw).cpu()
    last = [rows * b + rows - 1 for b in range(len(lens))]
    one = ops.paged_attention(q[:, last].to(gpu_device), *args, **kw).cpu()
    for b, n in enumerate(lens):
        want, bound = reference(q[:, rows * b:rows * (b + 1)], *kv[b], default_scale(d), window, sinks, torch.arange(n) < room)
        check(got[rows * b:rows * (b + 1)], want, bound, f"sequence {b} of {n} keys")
        check(one[b:b + 1], want[-1:], bound[-1:], f"last token of sequence {b} of {n} keys")
