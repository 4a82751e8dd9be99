"""Block tables, slots and the copy into pages against plain Python, and a server's run of them together with the attention."""

import random

import pytest
import torch

from paged_reference import check, default_scale, reference

pytestmark = pytest.mark.gpu


def plan(lens, new, table, free, count, page, pages, tokens):
    """The definition, request by request."""
    table = [row[:] for row in table]
    width = len(table[0])
    stack = free[:max(0, min(count, len(free)))]
    slots, positions, cu = [], [], [0]
    missing = 0
    for b, (n, more) in enumerate(zip(lens, new)):
        n, more = max(n, 0), max(more, 0)
        for i in range(min(-(-n // page), width), min(-(-(n + more) // page), width)):
            if stack:
                entry = stack.pop()
                table[b][i] = entry if 0 <= entry < pages else -1
            else:
                table[b][i], missing = -1, missing + 1
        for p in range(n, n + more):
            entry = table[b][p // page] if p // page < width else -1
            slots.append(entry * page + p % page if 0 <= entry < pages else -1)
            positions.append(p)
        cu.append(cu[-1] + more)
    pad = max(0, tokens - len(slots))
    return (table, [max(a, 0) + max(b, 0) for a, b in zip(lens, new)], cu, (slots + [-1] * pad)[:tokens], (positions + [0] * pad)[:tokens],
            len(stack) - missing)


def _check_tables(dev, lens, new, page, width, free, count, pages, tokens, table=None, stride=None):
    from shareprefill_amd import ops

    if table is None:
        rng = random.Random(1)
        table = [[rng.randrange(pages) if i < -(-max(n, 0) // page) else -1 for i in range(width)] for n in lens]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    wide = torch.full((len(lens), stride or width), 77, dtype=torch.int32, device=dev)
    live = wide[:, :width]
    live.copy_(ints(table))
    got = ops.page_tables(ints(lens), ints(new), live, ints(free).reshape(-1), ints([count]), page, pages, tokens)
    want = plan(lens, new, table, free, count, page, pages, tokens)
    assert live.tolist() == want[0]
    assert (wide[:, width:] == 77).all()
    assert got.seq_lens.tolist() == want[1] and got.cu_new.tolist() == want[2]
    assert got.slots.tolist() == want[3] and got.positions.tolist() == want[4] and got.free_left.tolist() == [want[5]]


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("batch", [1, 7, 256, 257, 1000, 4096])
def test_tables_match_the_definition(gpu_device, page, batch):
    rng = random.Random(page + batch)
    lens = [rng.choice((0, 1, page - 1, page, page + 1, rng.randrange(5 * page))) for _ in range(batch)]
    new = [rng.choice((0, 1, 1, page, rng.randrange(40))) for _ in range(batch)]
    pages = 7 * batch + 10
    free = list(range(pages))
    rng.shuffle(free)
    total = sum(new)
    for tokens in {total, total + 300, max(total - 5, 0), 0}:
        _check_tables(gpu_device, lens, new, page, 9, free, len(free), pages, tokens, stride=12)


def test_tables_when_pages_or_rows_run_out(gpu_device):
    lens, new, page = [0, 15, 40, 16], [20, 3, 30, 1], 16
    for count in (0, 1, 3, 4, 6, 99, -4):
        _check_tables(gpu_device, lens, new, page, 6, [3, 9, 1, 4, 7, 2, 8], count, 10, 60)
    _check_tables(gpu_device, lens, new, page, 2, [3, 9, 1, 4, 7], 5, 10, 60)   # requests longer than their rows
    _check_tables(gpu_device, lens, new, page, 6, [3, 99, -5, 4, 7, 2], 6, 10, 60)  # entries of the stack that are no pages
    _check_tables(gpu_device, [-3, 5], [4, -9], page, 3, [1, 2], 2, 10, 8)
    _check_tables(gpu_device, [0, 0], [0, 0], page, 3, [], 0, 0, 4)
    _check_tables(gpu_device, [33], [3], page, 4, [1], 1, 5, 4, table=[[2, 3, 900, -1]])  # a table that names no page for what is cached


def test_tables_of_very_long_requests(gpu_device):
    """Sums of the lengths past 32 bits: what is within reach is right, nothing else is touched."""
    from shareprefill_amd import ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    table = torch.full((3, 4), -1, dtype=torch.int32, device=gpu_device)
    got = ops.page_tables(ints([0, 2 ** 31 - 1, 0]), ints([20, 2 ** 31 - 1, 5]), table, ints([5, 6, 7]), ints([3]), 16, 8, 40)
    assert table.tolist()[0] == [7, 6, -1, -1] and table.tolist()[1] == [-1] * 4
    assert got.slots.tolist()[:20] == [7 * 16 + i for i in range(16)] + [6 * 16 + i for i in range(4)]
    assert got.slots.tolist()[20:] == [-1] * 20


@pytest.mark.parametrize("hkv,d,page", [(8, 128, 16), (1, 8, 16), (3, 40, 64), (2, 64, 1024), (5, 256, 32)])
@pytest.mark.parametrize("tokens", [1, 5, 300])
@pytest.mark.parametrize("token_major", [True, False])
def test_write_puts_every_token_in_its_slot(gpu_device, hkv, d, page, tokens, token_major):
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 2
    kv = [torch.randn(tokens, hkv, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for _ in range(2)]
    if not token_major:
        kv = [x.contiguous() for x in kv]
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    slots[0] = -1
    if tokens > 2:
        slots[2] = pages * page
    shape = (pages, page, hkv, d) if token_major else (pages, hkv, page, d)
    before = [torch.randn(shape, generator=gen).to(torch.bfloat16) for _ in range(2)]
    live = [x.to(gpu_device) for x in before]
    view = (lambda x: x.transpose(1, 2)) if token_major else (lambda x: x)
    ops.paged_cache_write(*(x.to(gpu_device) for x in kv), *(view(x) for x in live), slots.to(gpu_device))
    for x, pool, got in zip(kv, before, live):
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                view(pool)[s // page, :, s % page] = x[:, t]
        assert torch.equal(got.cpu(), pool)


def test_a_write_of_more_than_one_launch(gpu_device):
    """2100 tokens of 64 heads x 65536 channels are more 16-byte pieces than a launch takes; one token's memory stands for all of them, and
    all but a few have no slot."""
    from shareprefill_amd import ops

    hkv, d, tokens = 64, 65536, 2100
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(hkv, 1, d, generator=gen).to(torch.bfloat16).to(gpu_device) for _ in range(2))
    pools = [torch.zeros(1, hkv, 16, d, dtype=torch.bfloat16, device=gpu_device) for _ in range(2)]
    slots = torch.full((tokens,), -1, dtype=torch.int64)
    for t, slot in ((0, 3), (2047, 4), (2048, 9), (2099, 15)):
        slots[t] = slot
    ops.paged_cache_write(k.expand(-1, tokens, -1), v.expand(-1, tokens, -1), *pools, slots.to(gpu_device))
    for pool, x in zip(pools, (k, v)):
        for i in range(16):
            assert torch.equal(pool[0, :, i], x[:, 0] if i in (3, 4, 9, 15) else torch.zeros_like(x[:, 0])), i


def test_write_of_nothing_and_refusals(gpu_device):
    from shareprefill_amd import ops

    make = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=gpu_device)
    slots = torch.zeros(3, dtype=torch.int64, device=gpu_device)
    pool = make(4, 2, 16, 64)
    ops.paged_cache_write(make(2, 0, 64), make(2, 0, 64), pool, pool, slots[:0])
    k = make(2, 3, 64)
    for error, args in [
        (ValueError, (k, k[:1], pool, pool, slots)), (ValueError, (k, k, pool[:, :1], pool[:, :1], slots)), (ValueError, (k, k, pool, pool, slots[:2])),
        (ValueError, (k, k, pool, pool, slots.int())), (ValueError, (k, k, pool, pool, slots.cpu())), (AssertionError, (k.half(), k, pool, pool, slots)),
        (AssertionError, (k, k, pool.half(), pool, slots)), (ValueError, (k.cpu(), k, pool, pool, slots)), (ValueError, (k, k, pool[0], pool, slots)),
        (NotImplementedError, (k, k, make(4, 2, 24, 64), make(4, 2, 24, 64), slots)), (NotImplementedError, (k[..., :4], k[..., :4], pool[..., :4], pool[..., :4], slots))]:
        with pytest.raises(error):
            ops.paged_cache_write(*args)


@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 4)])
@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 16), (14, 2, 64, 64)])
def test_a_server_run(gpu_device, hq, hkv, d, page, window, sinks):
    """Prompts in chunks, next tokens beside them, requests that end and others in their place: every step's outputs are those of the
    definition over what each request has seen so far."""
    from shareprefill_amd import PagedKVCache

    gen = torch.Generator().manual_seed(page)
    rng = random.Random(page)
    layers, room = 2, 5
    cache = PagedKVCache(layers, num_pages=-(-5 * 300 // page), num_kv_heads=hkv, head_dim=d, max_requests=room, max_tokens=320, page_size=page,
                         device=gpu_device)
    scale = default_scale(d)
    held = [[(torch.zeros(hkv, 0, d, dtype=torch.bfloat16),) * 2 for _ in range(layers)] for _ in range(room)]
    for step in range(9):
        singles = step in (4, 8)
        if step == 5:
            finished = torch.tensor([True, False, True, False, False], device=gpu_device)
            cache.release(finished)
            for r in (0, 2):
                held[r] = [(torch.zeros(hkv, 0, d, dtype=torch.bfloat16),) * 2 for _ in range(layers)]
        new = [1] * room if singles else [rng.choice((0, 1, 1, rng.randrange(2, 60))) for _ in range(room)]
        total = sum(new)
        tokens = total if singles else total + rng.randrange(4)
        tables = cache.begin_step() if singles else cache.begin_step(torch.tensor(new, dtype=torch.int32, device=gpu_device), tokens)
        assert tables.free_left.item() >= 0
        for layer in range(layers):
            q, k, v = (torch.randn(tokens, h, d, generator=gen).to(torch.bfloat16).transpose(0, 1) for h in (hq, hkv, hkv))
            cache.write(layer, k.to(gpu_device), v.to(gpu_device))
            out = cache.attend(layer, q.to(gpu_device), scale, window=window, sinks=sinks).cpu()
            at = 0
            for r, n in enumerate(new):
                held[r][layer] = tuple(torch.cat((old, x[:, at:at + n]), 1) for old, x in zip(held[r][layer], (k, v)))
                if n:
                    check(out[at:at + n], *reference(q[:, at:at + n], *held[r][layer], scale, window or 0, sinks), f"step {step} request {r}")
                at += n
    assert cache.lens.tolist() == [h[0][0].shape[1] for h in held]
    used = sum(-(-n // page) for n in cache.lens.tolist())
    assert cache.free_count.item() == cache.num_pages - used
    cache.release(torch.ones(room, dtype=torch.bool, device=gpu_device))
    assert cache.free_count.item() == cache.num_pages and (cache.block_table == -1).all()
    assert sorted(cache._stack[:cache.num_pages].tolist()) == list(range(cache.num_pages))


def test_a_captured_server_step(gpu_device):
    """A decode step -- tables, copies, attention -- recorded once and replayed: the cache advances by a token per replay."""
    from shareprefill_amd import PagedKVCache, ops

    gen = torch.Generator().manual_seed(3)
    hq, hkv, d, page, room = 8, 2, 128, 16, 3
    make = lambda h, n: torch.randn(n, h, d, generator=gen).to(torch.bfloat16).to(gpu_device).transpose(0, 1)
    cache = PagedKVCache(1, 64, hkv, d, room, 300, page, device=gpu_device)
    first = torch.tensor([30, 7, 50], dtype=torch.int32, device=gpu_device)
    held = []
    cache.begin_step(first, 87)
    k, v = make(hkv, 87), make(hkv, 87)
    cache.write(0, k, v)
    at = 0
    for n in (30, 7, 50):
        held.append((k[:, at:at + n].cpu(), v[:, at:at + n].cpu()))
        at += n
    q_in, k_in, v_in = (torch.zeros(room, h, d, dtype=torch.bfloat16, device=gpu_device).transpose(0, 1) for h in (hq, hkv, hkv))
    out = torch.zeros(room, hq, d, dtype=torch.bfloat16, device=gpu_device)
    state = [t.clone() for t in (cache.lens, cache.free_count, cache.block_table, cache.pools)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.begin_step()
        cache.write(0, k_in, v_in)
        cache.attend(0, q_in, default_scale(d), out=out)
    for t, s in zip((cache.lens, cache.free_count, cache.block_table, cache.pools), state):
        assert torch.equal(t, s), "a capture runs nothing"
    for step in range(20):
        q, k, v = make(hq, room), make(hkv, room), make(hkv, room)
        q_in.copy_(q), k_in.copy_(k), v_in.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for r in range(room):
            held[r] = tuple(torch.cat((old, x[:, r:r + 1].cpu()), 1) for old, x in zip(held[r], (k, v)))
            check(out[r:r + 1].cpu(), *reference(q[:, r:r + 1].cpu(), *held[r], default_scale(d), 0, 0), f"replay {step} request {r}")
    assert cache.lens.tolist() == [50, 27, 70]
    assert isinstance(cache.tables, ops.PageTables)


def test_refusals(gpu_device):
    from shareprefill_amd import PagedKVCache, ops

    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    table = torch.full((2, 4), -1, dtype=torch.int32, device=gpu_device)
    ok = lambda **kw: ops.page_tables(**{**dict(lens=ints(1, 2), new_lens=ints(1, 1), block_table=table, free_pages=ints(1, 2, 3), free_count=ints(3),
                                               page_size=16, num_pages=8, max_new_tokens=4), **kw})
    ok()
    for error, kw in [
        (ValueError, dict(lens=ints(1, 2).cpu())), (ValueError, dict(lens=ints(1, 2).long())), (ValueError, dict(new_lens=ints(1))),
        (ValueError, dict(block_table=table[:1])), (ValueError, dict(block_table=table.t())), (ValueError, dict(block_table=table.long())),
        (ValueError, dict(free_count=ints(1, 2))), (ValueError, dict(free_pages=ints(1).long())), (ValueError, dict(max_new_tokens=-1)),
        (ValueError, dict(lens=ints(), new_lens=ints(), block_table=table[:0])), (NotImplementedError, dict(page_size=24)),
        (NotImplementedError, dict(page_size=8))]:
        with pytest.raises(error):
            ok(**kw)
    with pytest.raises(NotImplementedError):
        many = torch.zeros(4097, dtype=torch.int32, device=gpu_device)
        ok(lens=many, new_lens=many, block_table=torch.zeros(4097, 1, dtype=torch.int32, device=gpu_device))
    cache = PagedKVCache(1, 4, 2, 64, 2, 64, 16, device=gpu_device)
    with pytest.raises(RuntimeError):
        cache.attend(0, torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=gpu_device), 0.1)
    with pytest.raises(ValueError):
        cache.begin_step(ints(1, 1))
    with pytest.raises(ValueError):
        cache.release(torch.zeros(3, dtype=torch.bool, device=gpu_device))
    with pytest.raises(ValueError):
        PagedKVCache(1, 0, 2, 64, 2, 64)
