"""Offsets of the requests' rows that are not in order: one that goes back counts as the largest in front of it, and every request's rows are
what the definition says of the offsets held like that (paged_reference.py holds the bound)."""

import random

import pytest
import torch

from paged_reference import check, default_scale, make_pages, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 1, 64), (20, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 3)])
@pytest.mark.parametrize("batch,tokens", [(3, 40), (5, 130), (70, 200), (300, 150)])
def test_offsets_that_go_back_are_held(gpu_device, hq, hkv, d, window, sinks, batch, tokens):
    from shareprefill_amd import ops

    rng = random.Random(batch + d + window)
    gen = torch.Generator().manual_seed(batch)
    offsets = [rng.randrange(-20, tokens + 20) for _ in range(batch + 1)]
    if batch < 10:
        offsets[:4] = [0, tokens // 2, tokens // 4, tokens - 3]
        offsets[4:] = sorted(offsets[4:], reverse=True)
    else:
        # mostly in order, so that many requests have rows
        offsets = sorted(offsets)
        for _ in range(batch // 4):
            offsets[rng.randrange(batch + 1)] = rng.randrange(tokens)
    held, top = [], 0
    for x in offsets:
        top = max(top, min(max(x, 0), tokens))
        held.append(top)
    lens = [rng.choice((0, 1, rng.randrange(90), 60 + rng.randrange(90))) for _ in range(batch)]
    kp, vp, table, kv = make_pages(lens, hkv, d, 16, gen)
    q = torch.randn(tokens, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    out = torch.full((tokens, hq, d), 7.0, dtype=torch.bfloat16, device=gpu_device)
    ops.paged_attention(q.to(gpu_device), kp.to(gpu_device), vp.to(gpu_device), table.to(gpu_device), ints(lens), default_scale(d),
                        cu_q=ints(offsets), window=window or None, sinks=sinks, out=out)
    got = out.cpu()
    for b, n in enumerate(lens):
        r0, r1 = held[b], held[b + 1]
        shown = min(r1 - r0, n)
        assert (got[r0:r1 - shown] == 0).all()
        if shown:
            check(got[r1 - shown:r1], *reference(q[:, r1 - shown:r1], *kv[b], default_scale(d), window, sinks), f"request {b}")
    assert (got[:held[0]] == 7.0).all() and (got[held[-1]:] == 7.0).all()
