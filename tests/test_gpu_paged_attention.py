"""Attention over a cache in pages against its definition in 64 bits (paged_reference.py holds the derivation of the bound)."""

import pytest
import torch

from paged_reference import check, default_scale, make_pages, reference, starts

pytestmark = pytest.mark.gpu


def _run(dev, lens, q_lens, hq, hkv, d, page, window=0, sinks=0, seed=0, token_major=False, singles=False, extra_rows=0, scale=None):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(seed)
    kp, vp, table, kv = make_pages(lens, hkv, d, page, gen, token_major=token_major)
    at = starts(q_lens)
    rows = at[-1] + extra_rows
    q = torch.randn(rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    scale = default_scale(d) if scale is None else scale
    out = torch.full((rows, hq, d), 7.0, dtype=torch.bfloat16, device=dev)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)

    def pool(x):
        return x.transpose(1, 2).to(dev).transpose(1, 2) if token_major else x.to(dev)

    got = ops.paged_attention(q.to(dev), pool(kp), pool(vp), table.to(dev), ints(lens), scale, cu_q=None if singles else ints(at),
                              window=window or None, sinks=sinks, out=out)
    assert got is out
    got = got.cpu()
    for b, (n, ql) in enumerate(zip(lens, q_lens)):
        k, v = kv[b]
        shown = min(ql, n)  # rows in front of the first position see nothing
        want = torch.zeros(ql, hq, d, dtype=torch.float64)
        bound = torch.zeros(ql, hq, d, dtype=torch.float64)
        if shown:
            want[ql - shown:], bound[ql - shown:] = reference(q[:, at[b] + ql - shown:at[b] + ql], k, v, scale, window, sinks)
        check(got[at[b]:at[b] + ql], want, bound, f"sequence {b} of {n} keys, {ql} rows")
    assert (got[at[-1]:] == 7.0).all(), "rows behind the last sequence are not touched"


# (sequence lengths, their rows): one to many tiles, ends inside a page and a tile, empty sequences, more rows than keys
SHAPES = [
    ([1], [1]),
    ([5], [5]),
    ([64, 1, 0, 65], [64, 1, 0, 1]),
    ([200, 33, 129], [7, 33, 2]),
    ([300], [40]),
    ([3, 700, 16], [5, 70, 0]),
]


@pytest.mark.parametrize("lens,q_lens", SHAPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (4, 4, 64, 32), (7, 1, 128, 64), (6, 2, 64, 128), (20, 1, 64, 16), (2, 1, 128, 1024)])
def test_chunks_match_the_definition(gpu_device, lens, q_lens, hq, hkv, d, page):
    _run(gpu_device, lens, q_lens, hq, hkv, d, page, seed=len(lens) + hq, extra_rows=3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (64, 64), (100, 3), (100, 1000), (5000, 4), (63, 130)])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 64), (128, 256)])
def test_windows_and_sinks_match_the_definition(gpu_device, window, sinks, d, page):
    _run(gpu_device, [400, 1, 77, 213], [130, 1, 77, 3], 4, 2, d, page, window, sinks, seed=window + sinks, extra_rows=1)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (7, 1, 128), (14, 2, 64), (4, 4, 64), (16, 1, 128), (18, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4), (33, 40), (1, 0)])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_single_tokens_match_the_definition(gpu_device, hq, hkv, d, window, sinks, page):
    lens = [1, 0, 31, 32, 33, 300, 1000, 129, 16]
    _run(gpu_device, lens, [1] * len(lens), hq, hkv, d, page, window, sinks, seed=hq, singles=True)


def test_single_tokens_of_long_caches(gpu_device):
    _run(gpu_device, [20011, 5, 9000], [1, 1, 1], 8, 2, 128, 16, seed=3, singles=True)
    _run(gpu_device, [20011, 5, 9000], [1, 1, 1], 4, 1, 64, 64, 4096, 100, seed=4, singles=True)


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 70), (1111, 3), (64, 2000), (100, 64)])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 32), (128, 64)])
def test_long_chunks(gpu_device, window, sinks, d, page):
    """Tables of more pages than a wave has lanes: walks that go from the sinks to a window far behind, begin and end anywhere, and pages
    that are missing on either side.  K's pool token by token, V's head by head, the table a slice of a wider one."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(window + page)
    hq, hkv, lens, q_lens = 4, 2, [5003, 2111, 40], [40, 61, 9]
    kp, vp, table, kv = make_pages(lens, hkv, d, page, gen)
    gone = [0, 66, lens[0] // page - 3]  # of the first sequence
    seen = torch.ones(lens[0], dtype=torch.bool)
    for i in gone:
        table[0, i] = -1
        seen[i * page:(i + 1) * page] = False
    at = starts(q_lens)
    q = torch.randn(at[-1], hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    wide = torch.full((3, table.shape[1] + 5), 1, dtype=torch.int32, device=gpu_device)
    wide[:, 2:-3] = table.to(gpu_device)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    args = [kp.to(gpu_device).transpose(1, 2).contiguous().transpose(1, 2), vp.to(gpu_device), wide[:, 2:-3], ints(lens), default_scale(d)]
    got = ops.paged_attention(q.contiguous().to(gpu_device), *args, cu_q=ints(at), window=window or None, sinks=sinks).cpu()
    ones = ops.paged_attention(q[:, [at[b + 1] - 1 for b in range(3)]].to(gpu_device), *args, window=window or None, sinks=sinks).cpu()
    for b in range(3):
        want, bound = reference(q[:, at[b]:at[b + 1]], *kv[b], default_scale(d), window, sinks, seen if b == 0 else None)
        check(got[at[b]:at[b + 1]], want, bound, f"sequence {b}")
        check(ones[b:b + 1], want[-1:], bound[-1:], f"last token of sequence {b}")


def test_more_kv_heads_than_workgroups(gpu_device):
    _run(gpu_device, [50, 33], [40, 1], 300, 300, 64, 16, 20, 3, seed=1)
    _run(gpu_device, [50, 33], [1, 1], 300, 300, 64, 16, seed=2, singles=True)


@pytest.mark.parametrize("batch", [63, 65, 300])
def test_many_sequences(gpu_device, batch):
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 90, (batch,), generator=gen).tolist()
    _run(gpu_device, lens, [1] * batch, 4, 2, 64, 16, seed=batch, singles=True)
    q_lens = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 6, (batch,), generator=gen).tolist())]
    _run(gpu_device, lens, q_lens, 4, 2, 64, 16, 40, 2, seed=batch)


def test_pools_kept_token_by_token(gpu_device):
    _run(gpu_device, [150, 40], [60, 1], 4, 2, 128, 32, seed=1, token_major=True)
    _run(gpu_device, [150, 40], [1, 1], 4, 2, 64, 16, seed=2, token_major=True, singles=True)


def test_large_logits(gpu_device):
    _run(gpu_device, [300, 90], [50, 90], 4, 2, 128, 16, seed=9, scale=3.0)
    _run(gpu_device, [300, 90], [1, 1], 4, 2, 128, 16, seed=9, scale=3.0, singles=True)


def _device(t, dev):
    return t.to(dev)


@pytest.mark.parametrize("singles", [False, True])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 32), (128, 128)])
def test_keys_without_a_page_are_not_seen(gpu_device, singles, d, page):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(5)
    hq, hkv, n = 4, 2, 5 * page + 3
    kp, vp, table, kv = make_pages([n, n, n], hkv, d, page, gen)
    seen = torch.ones(3, n, dtype=torch.bool)
    for b, i, entry in ((0, 1, -1), (0, 4, kp.shape[0]), (1, 0, 2 ** 31 - 1), (1, 5, -7)):
        table[b, i] = entry
        seen[b, i * page:(i + 1) * page] = False
    table[2] = -1
    seen[2] = False
    rows = 1 if singles else 20
    q = torch.randn(3 * rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    got = ops.paged_attention(q.to(gpu_device), kp.to(gpu_device), vp.to(gpu_device), table.to(gpu_device), ints([n] * 3), default_scale(d),
                              cu_q=None if singles else ints([0, rows, 2 * rows, 3 * rows])).cpu()
    for b in range(3):
        want, bound = reference(q[:, b * rows:(b + 1) * rows], *kv[b], default_scale(d), 0, 0, seen[b])
        check(got[b * rows:(b + 1) * rows], want, bound, f"sequence {b}")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("d", [64, 128])
def test_values_of_masked_keys_do_not_matter(gpu_device, bad, window, sinks, d):
    """A later token's value, and one that has left the window, may be anything: rows that do not see it are those of the definition, rows
    that do are not finite."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(11)
    hq, hkv, page, n, rows = 4, 2, 16, 150, 60
    kp, vp, table, kv = make_pages([n], hkv, d, page, gen)
    spoilt = [100, 149] + ([30] if window else [])
    for j in spoilt:
        kv[0][1][:, j] = bad
        vp[table[0, j // page], :, j % page] = bad
        kv[0][0][:, j] = bad if j == 30 else kv[0][0][:, j]
        kp[table[0, j // page], :, j % page] = kv[0][0][:, j]
    q = torch.randn(rows, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    got = ops.paged_attention(q.to(gpu_device), kp.to(gpu_device), vp.to(gpu_device), table.to(gpu_device), ints([n]), default_scale(d),
                              cu_q=ints([0, rows]), window=window or None, sinks=sinks).cpu()
    want, bound = reference(q, *kv[0], default_scale(d), window, sinks)
    positions = torch.arange(n - rows, n)
    clean = torch.ones(rows, dtype=torch.bool)
    for j in spoilt:
        sees = (positions >= j) & ((positions - j < window) | (j < sinks) if window else True)
        clean &= ~sees
    assert clean.any() and not clean.all()
    check(got[clean], want[clean], bound[clean], "rows that do not see the spoilt values")
    assert not torch.isfinite(got[~clean].float()).any(), "rows that see them"


def test_pools_beyond_32_bit_offsets(gpu_device):
    """Pages whose first element lies past 2^32 bytes and past 2^31 elements of the pool."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(2)
    hq, hkv, d, page, n = 4, 2, 128, 64, 200
    small_k, small_v, table, kv = make_pages([n, n], hkv, d, page, gen, slack=0)
    pages = (1 << 31) // (hkv * page * d) + 64  # 4.3e9 bytes
    at = [pages - 1, 0, pages - 30, pages // 2 + 1, pages - 7, 3, pages - 64, 9]
    kp, vp = (torch.zeros(pages, hkv, page, d, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    moved = torch.full_like(table, -1)
    for b in range(2):
        for i in range(table.shape[1]):
            to = at[b * 4 + i]
            moved[b, i] = to
            kp[to], vp[to] = small_k[table[b, i]].to(gpu_device), small_v[table[b, i]].to(gpu_device)
    q = torch.randn(2 * 9, hq, d, generator=gen).to(torch.bfloat16).transpose(0, 1)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    got = ops.paged_attention(q.to(gpu_device), kp, vp, moved.to(gpu_device), ints([n, n]), default_scale(d), cu_q=ints([0, 9, 18])).cpu()
    one = ops.paged_attention(q[:, [8, 17]].to(gpu_device), kp, vp, moved.to(gpu_device), ints([n, n]), default_scale(d)).cpu()
    for b in range(2):
        want, bound = reference(q[:, 9 * b:9 * b + 9], *kv[b], default_scale(d), 0, 0)
        check(got[9 * b:9 * b + 9], want, bound)
        check(one[b:b + 1], want[8:], bound[8:])
    # and the copy into them
    k_new, v_new = (torch.randn(3, hkv, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1) for _ in range(2))
    slots = torch.tensor([(pages - 2) * page + 5, 17, pages * page], dtype=torch.int64, device=gpu_device)
    ops.paged_cache_write(k_new, v_new, kp, vp, slots)
    assert torch.equal(kp[pages - 2, :, 5], k_new[:, 0]) and torch.equal(vp[0, :, 17], v_new[:, 1])


@pytest.mark.parametrize("singles", [False, True])
def test_a_captured_step_follows_new_lengths(gpu_device, singles):
    """Lengths, offsets and tables are read on the device: a replay with others gives the eager run's bits, replay after replay, and so do
    two graphs captured one after the other and replayed on two streams."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(8)
    hq, hkv, d, page, rows = 8, 2, 128, 16, 48
    sets = []
    for lens, q_lens in (([500, 90, 1000], [30, 1, 17]), ([1300, 3, 16], [1, 3, 16]), ([0, 2000, 45], [0, 40, 8])):
        if singles:
            q_lens = [1, 1, 1]
        kp, vp, table, _ = make_pages([2000] * 3, hkv, d, page, gen, slack=0)
        sets.append((kp, vp, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(starts(q_lens), dtype=torch.int32)))
    n = 3 if singles else rows
    qs = [torch.randn(n, hq, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1) for _ in sets]
    sets = [tuple(t.to(gpu_device) for t in s) for s in sets]

    def call(q, s, out):
        return ops.paged_attention(q, s[0], s[1], s[2], s[3], default_scale(d), cu_q=None if singles else s[4], out=out)

    eager = [call(q, s, torch.zeros(n, hq, d, dtype=torch.bfloat16, device=gpu_device)) for q, s in zip(qs, sets)]
    graphs = []
    for _ in range(2):
        live = tuple(t.clone() for t in sets[0])
        q_live, out = torch.empty(n, hq, d, dtype=torch.bfloat16, device=gpu_device).transpose(0, 1), torch.zeros(
            n, hq, d, dtype=torch.bfloat16, device=gpu_device)
        q_live.copy_(qs[0])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(q_live, live, out)
        graphs.append((graph, q_live, live, out))
    for i in (0, 1, 2, 1, 0):
        graph, q_live, live, out = graphs[0]
        q_live.copy_(qs[i])
        for a, b in zip(live, sets[i]):
            a.copy_(b)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), f"replay with set {i}"
        call(qs[1], sets[1], torch.zeros_like(out))  # the program's own work in between
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(6):
        for (graph, q_live, live, out), i, stream in zip(graphs, (turn % 3, (turn + 1) % 3), streams):
            with torch.cuda.stream(stream):
                q_live.copy_(qs[i])
                for a, b in zip(live, sets[i]):
                    a.copy_(b)
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), i in zip(graphs, (turn % 3, (turn + 1) % 3)):
            assert torch.equal(out, eager[i])


def test_another_stream_gives_the_same(gpu_device):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(4)
    kp, vp, table, _ = make_pages([900, 400], 2, 64, 32, gen)
    args = [t.to(gpu_device) for t in (kp, vp, table, torch.tensor([900, 400], dtype=torch.int32))]
    q = torch.randn(80, 4, 64, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1)
    cu = torch.tensor([0, 70, 80], dtype=torch.int32, device=gpu_device)
    here = ops.paged_attention(q, *args, 0.1, cu_q=cu)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = [ops.paged_attention(q, *args, 0.1, cu_q=cu) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(here, x) for x in there)


def test_device_values_out_of_range_are_held(gpu_device):
    """Lengths beyond the table, offsets beyond the rows: nothing is read or written out of place."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(6)
    hq, hkv, d, page = 4, 2, 64, 16
    kp, vp, table, kv = make_pages([100], hkv, d, page, gen, slack=0)
    q = torch.randn(10, hq, d, generator=gen).to(torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    pools = kp.to(gpu_device), vp.to(gpu_device)
    # offsets past the last row, in front of the first
    out = ops.paged_attention(q.transpose(0, 1).to(gpu_device), *pools, table.to(gpu_device), ints([100]), 0.1, cu_q=ints([-5, 1000])).cpu()
    want, bound = reference(q.transpose(0, 1), *kv[0], 0.1, 0, 0)
    check(out, want, bound)
    # a length beyond the table: what lies behind its last page is not there
    full = 7 * page
    for n in (5000, 2 ** 31 - 1):
        got = ops.paged_attention(q[:1].transpose(0, 1).to(gpu_device), *pools, table.to(gpu_device), ints([n]), 0.1, window=n).cpu()
        assert got.shape == (1, hq, d)
    assert (ops.paged_attention(q[:1].transpose(0, 1).to(gpu_device), *pools, table.to(gpu_device), ints([-3]), 0.1) == 0).all()
    assert full >= 100


def test_rows_of_no_request(gpu_device):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(7)
    kp, vp, table, _ = make_pages([40, 20], 2, 64, 16, gen)
    args = [t.to(gpu_device) for t in (kp, vp, table, torch.tensor([40, 20], dtype=torch.int32))]
    empty = torch.empty(4, 0, 64, dtype=torch.bfloat16, device=gpu_device)
    cu = torch.zeros(3, dtype=torch.int32, device=gpu_device)
    assert ops.paged_attention(empty, *args, 0.1, cu_q=cu).shape == (0, 4, 64)
    q = torch.randn(4, 6, 64, generator=gen).to(torch.bfloat16).to(gpu_device)
    out = torch.full((6, 4, 64), 3.0, dtype=torch.bfloat16, device=gpu_device)
    ops.paged_attention(q, *args, 0.1, cu_q=cu, out=out)
    assert (out == 3.0).all()


def test_refusals(gpu_device):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(7)
    kp, vp, table, _ = make_pages([40], 2, 64, 16, gen)
    kp, vp, table, lens = (t.to(gpu_device) for t in (kp, vp, table, torch.tensor([40], dtype=torch.int32)))
    q = torch.zeros(4, 1, 64, dtype=torch.bfloat16, device=gpu_device)
    ok = lambda **kw: ops.paged_attention(**{**dict(q=q, k_pages=kp, v_pages=vp, block_table=table, seq_lens=lens, softmax_scale=0.1), **kw})
    ok()
    for error, kw in [
        (AssertionError, dict(q=q.float())), (AssertionError, dict(k_pages=kp.float())), (ValueError, dict(q=q.cpu())),
        (ValueError, dict(q=q[0])), (ValueError, dict(v_pages=vp[:, :1])), (ValueError, dict(block_table=table.long())),
        (ValueError, dict(block_table=table.cpu())), (ValueError, dict(seq_lens=lens.long())), (ValueError, dict(seq_lens=lens.cpu())),
        (ValueError, dict(q=q.repeat(1, 2, 1))), (ValueError, dict(cu_q=lens)), (ValueError, dict(window=0)), (ValueError, dict(sinks=-1)),
        (ValueError, dict(softmax_scale=0.0)), (ValueError, dict(softmax_scale=float("nan"))), (ValueError, dict(q=q[:3])),
        (ValueError, dict(out=torch.empty(1, 4, 64, device=gpu_device))), (ValueError, dict(q=q[..., :32])),
        (NotImplementedError, dict(q=q[..., :32].contiguous(), k_pages=kp[..., :32].contiguous(), v_pages=vp[..., :32].contiguous())),
        (NotImplementedError, dict(k_pages=kp[:, :, :8], v_pages=vp[:, :, :8])),
        (NotImplementedError, dict(k_pages=kp.reshape(-1)[4:4 + 16 * 2 * 64].view(1, 2, 16, 64), v_pages=vp[:1]))]:
        with pytest.raises(error):
            ok(**kw)
