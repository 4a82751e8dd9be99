"""A value that is not finite in what later tokens see: their rows are no numbers, the others are the definition's, and the call takes about as
long as without it."""

import pytest
import torch

from paged_reference import check, default_scale, make_pages, reference

pytestmark = pytest.mark.gpu


def _times(run, n=5):
    run()
    out = []
    for _ in range(n):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        run()
        b.record()
        b.synchronize()
        out.append(a.elapsed_time(b))
    return min(out)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("channels", [1, 128])
@pytest.mark.parametrize("window", [None, 3000])
def test_a_chunk_over_a_cache_with_one_bad_value_is_not_held_up(gpu_device, bad, channels, window):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(1)
    hq, hkv, d, page, n, rows = 8, 2, 128, 64, 4096, 256
    kp, vp, table, kv = make_pages([n], hkv, d, page, gen, fill=0.0)
    at = 1500  # seen by every new token, far from their own positions and from a window's start
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    q = torch.randn(rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    args = [q.to(gpu_device), kp.to(gpu_device), vp.to(gpu_device), table.to(gpu_device), ints([n]), default_scale(d)]
    run = lambda: ops.paged_attention(*args, cu_q=ints([0, rows]), window=window)
    clean, clean_ms = run().cpu(), _times(run)
    args[2][table[0, at // page], 0, at % page, :channels] = bad
    got, bad_ms = run().cpu(), _times(run)
    assert torch.equal(got[:, 4:], clean[:, 4:]), "heads of the other kv head"
    assert not torch.isfinite(got[:, :4, :channels].float()).any()
    assert torch.equal(got[:, :4, channels:], clean[:, :4, channels:]), "channels without it"
    assert bad_ms < 5 * clean_ms + 0.1, (clean_ms, bad_ms)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (2, 2)])
def test_rows_in_front_of_and_behind_bad_values(gpu_device, bad, d, page, hq, hkv, window, sinks):
    """Bad values among the new tokens and behind the window, beside one that everybody sees in another channel: rows that see none of them in a
    channel have the definition's value there."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(2)
    n, rows = 500, 200
    kp, vp, table, kv = make_pages([n], hkv, d, page, gen, fill=0.0)
    spoilt = {(2, 7): "a sink", (350, 11): "a new token", (351, 11): "the next", (420, 3): "a later one", (499, 20): "the last"}
    if not window:
        spoilt[(100, 15)] = "cached"
    for j, c in spoilt:
        kv[0][1][0, j, c] = bad
        vp[table[0, j // page], 0, j % page, c] = bad
    q = torch.randn(rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    got = ops.paged_attention(q.to(gpu_device), kp.to(gpu_device), vp.to(gpu_device), table.to(gpu_device), ints([n]), default_scale(d),
                              cu_q=ints([0, rows]), window=window or None, sinks=sinks).cpu()
    finite = [(torch.where(torch.isfinite(x.float()), x.float(), torch.zeros(())).to(torch.bfloat16)) for x in kv[0]]
    want, bound = reference(q, *finite, default_scale(d), window, sinks)
    p = torch.arange(n - rows, n)
    sees = torch.zeros(rows, hq, d, dtype=torch.bool)
    for j, c in spoilt:
        s = (p >= j) & ((p - j < window) | (j < sinks) if window else True)
        sees[:, :hq // hkv, c] |= s[:, None]
    assert sees.any() and not sees.all()
    check(got[~sees], want[~sees], bound[~sees], "elements that see no bad value")
    assert not torch.isfinite(got[sees].float()).any(), "elements that see one"
