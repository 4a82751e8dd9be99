"""Sliding-window attention with sinks over contiguous keys and values against its definition in 64 bits (paged_reference.py)."""

import pytest
import torch

from paged_reference import check, default_scale, reference

pytestmark = pytest.mark.gpu


def _run(dev, batch, n, nk, hq, hkv, d, window, sinks, seed=0, token_major=True):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(seed)

    def make(heads, length):
        if token_major:
            return torch.randn(batch, length, heads, d, generator=gen).to(torch.bfloat16).transpose(1, 2)
        return torch.randn(batch, heads, length, d, generator=gen).to(torch.bfloat16)

    q, k, v = make(hq, n), make(hkv, nk), make(hkv, nk)
    got = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), default_scale(d), window=window or None, sinks=sinks).cpu()
    assert got.shape == (batch, n, hq, d)
    for b in range(batch):
        check(got[b], *reference(q[b], k[b], v[b], default_scale(d), window, sinks), f"sequence {b}")


@pytest.mark.parametrize("n,nk", [(1, 1), (7, 7), (64, 64), (65, 65), (200, 200), (50, 170), (1, 130), (33, 300)])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 128), (7, 1, 64), (2, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 4), (64, 0), (100, 70)])
def test_prompts_and_chunks_match_the_definition(gpu_device, n, nk, hq, hkv, d, window, sinks):
    _run(gpu_device, 2, n, nk, hq, hkv, d, window, sinks, seed=n + nk)


@pytest.mark.parametrize("nk", [1, 31, 32, 33, 64, 500, 4000])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (14, 2, 64), (32, 2, 128), (34, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 2), (40, 4), (1000, 33)])
def test_single_tokens_match_the_definition(gpu_device, nk, hq, hkv, d, window, sinks):
    _run(gpu_device, 3, 1, nk, hq, hkv, d, window, sinks, seed=nk, token_major=False)


def test_a_long_prompt_in_rows_spread_over_many_workgroups(gpu_device):
    """Enough row tiles that no cut is needed, and a few rows of them checked."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(1)
    n, hq, hkv, d = 9001, 32, 8, 128
    q, k, v = (torch.randn(n, h, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for h in (hq, hkv, hkv))
    for window, sinks in ((700, 4), (0, 0)):
        got = ops.window_attention(*(t[None].to(gpu_device) for t in (q, k, v)), default_scale(d), window=window or None, sinks=sinks)[0].cpu()
        for p in (0, 1, 63, 64, 699, 700, 703, 704, 4095, 8999, 9000):
            want, bound = reference(q[:, p:p + 1], k[:, :p + 1], v[:, :p + 1], default_scale(d), window, sinks)
            check(got[p:p + 1], want, bound, f"position {p}")


def test_every_row_is_the_mean_of_what_it_sees(gpu_device):
    """With q = 0 all weights are equal: every row of a long prompt in closed form.  The weights are powers of two and sums of them, exact, so
    what is left is the output's rounding and fp32 sums of up to n values, and the division's rounding."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(1)
    for n, hq, hkv, d, window, sinks in ((6000, 28, 4, 128, 1000, 70), (5003, 4, 1, 64, 0, 0), (3333, 8, 8, 64, 65, 1)):
        q = torch.zeros(1, hq, n, d, dtype=torch.bfloat16, device=gpu_device)
        k = torch.randn(1, hkv, n, d, generator=gen).to(torch.bfloat16).to(gpu_device)
        v = torch.randn(1, hkv, n, d, generator=gen).to(torch.bfloat16).to(gpu_device)
        got = ops.window_attention(q, k, v, 0.1, window=window or None, sinks=sinks)[0].double()
        sums = torch.cat((torch.zeros(hkv, 1, d, device=gpu_device, dtype=torch.float64), v[0].double().cumsum(1)), 1)
        p = torch.arange(n, device=gpu_device)
        lo = (p - (window or n + 1) + 1).clamp(min=0)
        front = torch.minimum(lo, torch.full_like(lo, sinks))
        total = sums[:, p + 1] - sums[:, lo] + sums[:, front]
        want = (total / (p + 1 - lo + front)[None, :, None]).transpose(0, 1).repeat_interleave(hq // hkv, 1)
        mean_abs = v.double().abs().mean().item()
        err = (got - want).abs()
        assert (err <= want.abs() * 2.0 ** -8 * 1.01 + n * 2.0 ** -24 * mean_abs).all(), (n, window, err.max().item())


@pytest.mark.parametrize("batch,n,nk,hq,hkv,d", [(5, 700, 700, 8, 1, 128), (33, 70, 70, 16, 2, 64), (3, 130, 400, 160, 1, 64), (2, 9, 40, 300, 1, 128),
                                                (70, 33, 33, 8, 8, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (65, 3)])
def test_batches(gpu_device, batch, n, nk, hq, hkv, d, window, sinks):
    """Row tiles kept whole and cut ones, several of a sequence and one, tokens that reach over row tiles; enough sequences that they are dealt
    to the workgroups in more than one go."""
    _run(gpu_device, batch, n, nk, hq, hkv, d, window, sinks, seed=batch)


def test_many_short_sequences(gpu_device):
    """4096 single tokens; 2048 sequences where there are more than one or large groups, no more."""
    from shareprefill_amd import ops

    _run(gpu_device, 2048, 2, 3, 2, 1, 64, 2, 0, seed=1)
    _run(gpu_device, 4096, 1, 2, 2, 1, 64, 0, 0, seed=1)
    make = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=gpu_device)
    for batch, n, hq in ((4097, 1, 2), (2049, 2, 2), (2049, 1, 17)):
        with pytest.raises(RuntimeError, match="batch"):
            ops.window_attention(make(batch, hq, n, 64), make(batch, 1, 2, 64), make(batch, 1, 2, 64), 0.1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_out_of_sight_do_not_matter(gpu_device, bad):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(3)
    n, hq, hkv, d, window = 140, 4, 2, 128, 30
    q, k, v = (torch.randn(h, n, d, generator=gen).to(torch.bfloat16) for h in (hq, hkv, hkv))
    k[:, 50] = bad
    v[:, 50] = bad
    got = ops.window_attention(*(t[None].to(gpu_device) for t in (q, k, v)), default_scale(d), window=window)[0].cpu()
    want, bound = reference(q, k, v, default_scale(d), window, 0)
    clean = (torch.arange(n) < 50) | (torch.arange(n) >= 80)
    check(got[clean], want[clean], bound[clean])
    assert not torch.isfinite(got[~clean].float()).any()
    # the next token: position 139 does not see it
    one = ops.window_attention(q[None, :, -1:].to(gpu_device), k[None].to(gpu_device), v[None].to(gpu_device), default_scale(d), window=window)[0].cpu()
    check(one, want[-1:], bound[-1:])


@pytest.mark.parametrize("n,nk", [(900, 900), (40, 3000), (1, 3000)])
def test_a_captured_call_replays(gpu_device, n, nk):
    """Whole row tiles, cut ones and single tokens: a replay gives the eager run's bits for whatever stands in its tensors."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(n)
    make = lambda heads, length: torch.randn(2, length, heads, 128, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(1, 2)
    sets = [(make(8, n), make(2, nk), make(2, nk)) for _ in range(2)]
    eager = [ops.window_attention(*s, 0.1, window=500, sinks=4) for s in sets]
    live = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.window_attention(*live, 0.1, window=500, sinks=4)
    for i in (0, 1, 1, 0):
        for a, b in zip(live, sets[i]):
            a.copy_(b)
        out.zero_()
        graph.replay()
        assert torch.equal(ops.window_attention(*sets[1 - i], 0.1, window=500, sinks=4), eager[1 - i])
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i])


def test_keys_shared_by_a_batch(gpu_device):
    """A batch stride of zero: samples that go on from one prompt."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(5)
    q = torch.randn(3, 4, 70, 64, generator=gen).to(torch.bfloat16)
    k, v = (torch.randn(1, 2, 200, 64, generator=gen).to(torch.bfloat16).expand(3, -1, -1, -1) for _ in range(2))
    for queries in (q, q[:, :, -1:]):
        got = ops.window_attention(queries.to(gpu_device), k[:1].to(gpu_device).expand(3, -1, -1, -1), v[:1].to(gpu_device).expand(3, -1, -1, -1),
                                   0.1, window=90, sinks=2).cpu()
        for b in range(3):
            check(got[b], *reference(queries[b], k[b], v[b], 0.1, 90, 2))


@pytest.mark.parametrize("window", [0, 70])
def test_rows_that_are_no_numbers_stay_with_themselves(gpu_device, window):
    """A query with a NaN, one whose logits overflow: their rows are NaN, the others the definition's."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(6)
    n, hq, hkv, d = 300, 4, 2, 128
    q, k, v = (torch.randn(h, n, d, generator=gen).to(torch.bfloat16) for h in (hq, hkv, hkv))
    q[1, 77, 5] = float("nan")
    q[2, 200] = float("inf")
    got = ops.window_attention(*(t[None].to(gpu_device) for t in (q, k, v)), default_scale(d), window=window or None)[0].cpu()
    want, bound = reference(q, k, v, default_scale(d), window, 0)
    clean = torch.ones(n, hq, dtype=torch.bool)
    clean[77, 1] = clean[200, 2] = False
    check(got[clean], want[clean], bound[clean])
    assert torch.isnan(got[~clean].float()).all()


def test_a_window_as_long_as_the_prompt_is_none(gpu_device):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, h, 333, 64, generator=gen).to(torch.bfloat16).to(gpu_device) for h in (6, 3, 3))
    a = ops.window_attention(q, k, v, 0.1)
    for window, sinks in ((333, 0), (10 ** 12, 5), (1, 333), (5, 10 ** 12)):
        assert torch.equal(a, ops.window_attention(q, k, v, 0.1, window=window, sinks=sinks))


def test_empty_and_refused_calls(gpu_device):
    from shareprefill_amd import ops

    make = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=gpu_device)
    assert ops.window_attention(make(2, 4, 0, 64), make(2, 2, 5, 64), make(2, 2, 5, 64), 0.1, window=3).shape == (2, 0, 4, 64)
    assert ops.window_attention(make(2, 4, 0, 64), make(2, 2, 0, 64), make(2, 2, 0, 64), 0.1, window=3).shape == (2, 0, 4, 64)
    q, k = make(1, 4, 8, 64), make(1, 2, 8, 64)
    for error, args, kw in [
        (ValueError, (make(1, 4, 9, 64), k, k), {}), (ValueError, (q, k, k[:, :1]), {}), (ValueError, (make(2, 4, 8, 64), k, k), {}),
        (ValueError, (q[0], k, k), {}), (AssertionError, (q.half(), k, k), {}), (ValueError, (q.cpu(), k, k), {}), (ValueError, (q, k, k.cpu()), {}),
        (ValueError, (make(1, 3, 8, 64), k, k), {}), (ValueError, (q, k, k), dict(window=0)), (ValueError, (q, k, k), dict(sinks=-2)),
        (ValueError, (q.transpose(2, 3).contiguous().transpose(2, 3), k, k), {}),
        (NotImplementedError, (make(1, 4, 8, 96), make(1, 2, 8, 96), make(1, 2, 8, 96)), {})]:
        with pytest.raises(error):
            ops.window_attention(*args, 0.1, **kw)
