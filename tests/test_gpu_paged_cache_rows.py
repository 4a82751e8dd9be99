"""Steps of PagedKVCache in which requests bring more tokens than the step has rows: the tokens that have none are left out of lengths, pages and
sight, and the requests go on from what they have (paged_reference.py holds the bound)."""

import pytest
import torch

from paged_reference import check, default_scale, reference

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 4, 2, 64, 16


class Server:
    """A cache and what each of its requests should hold."""

    def __init__(self, dev, requests, seed, window=None, sinks=0, num_pages=60):
        from shareprefill_amd import PagedKVCache

        self.dev, self.gen, self.window, self.sinks = dev, torch.Generator().manual_seed(seed), window, sinks
        self.cache = PagedKVCache(1, num_pages, HKV, D, requests, 200, PAGE, device=dev)
        self.cache.pools.fill_(float("nan"))  # whoever reads what nobody wrote is found out
        self.held = [(torch.zeros(HKV, 0, D, dtype=torch.bfloat16),) * 2 for _ in range(requests)]

    def rows(self, n):
        return [torch.randn(n, h, D, generator=self.gen).to(torch.bfloat16).transpose(0, 1) for h in (HQ, HKV, HKV)]

    def ints(self, *x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def verify(self, out, taken, at, q, k, v, what=""):
        """taken: new tokens of every request that count, at: their first row"""
        for r, (n, first) in enumerate(zip(taken, at)):
            self.held[r] = tuple(torch.cat((old, x[:, first:first + n]), 1) for old, x in zip(self.held[r], (k, v)))
            if n:
                check(out[first:first + n], *reference(q[:, first:first + n], *self.held[r], default_scale(D), self.window or 0, self.sinks),
                      f"{what} request {r}")
        assert self.cache.lens.tolist() == [h[0].shape[1] for h in self.held]
        used = sum(-(-h[0].shape[1] // PAGE) for h in self.held)
        assert self.cache.free_count.item() == self.cache.num_pages - used
        assert ((self.cache.block_table >= 0).sum().item()) == used

    def step(self, new, rows, what=""):
        taken, at, left = [], [], rows
        for n in new:
            at.append(rows - left)
            taken.append(min(max(n, 0), left))
            left -= taken[-1]
        tables = self.cache.begin_step(self.ints(*new), rows)
        assert tables.cu_new.tolist() == at + [rows - left]
        assert tables.free_left.item() >= 0
        q, k, v = self.rows(rows)
        self.cache.write(0, k.to(self.dev), v.to(self.dev))
        out = self.cache.attend(0, q.to(self.dev), default_scale(D), window=self.window, sinks=self.sinks).cpu()
        self.verify(out, taken, at, q, k, v, what)


@pytest.mark.parametrize("window,sinks", [(None, 0), (25, 2)])
def test_more_new_tokens_than_rows(gpu_device, window, sinks):
    server = Server(gpu_device, 4, 1, window, sinks)
    for i, (new, rows) in enumerate([((20, 30, 10, 0), 40), ((1, 10, 10, 5), 21), ((1, 1, 1, 1), 4), ((2 ** 31 - 1, 5, 5, 5), 10), ((3, 0, 17, 40), 60),
                                     ((5, 5, 5, 5), 0), ((0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1), 3), ((1, 1, 1, 1), 9)]):
        server.step(new, rows, f"step {i}")


def test_a_replayed_step_with_more_tokens_than_it_has_rows(gpu_device):
    server = Server(gpu_device, 3, 2)
    server.step((9, 30, 16), 55)
    cache, rows, dev = server.cache, 12, gpu_device
    new = server.ints(0, 0, 0)
    q_in, k_in, v_in = (torch.zeros(rows, h, D, dtype=torch.bfloat16, device=dev).transpose(0, 1) for h in (HQ, HKV, HKV))
    out = torch.zeros(rows, HQ, D, dtype=torch.bfloat16, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.begin_step(new, rows)
        cache.write(0, k_in, v_in)
        cache.attend(0, q_in, default_scale(D), out=out)
    for i, (more, taken) in enumerate([((5, 4, 3), (5, 4, 3)), ((5, 9, 3), (5, 7, 0)), ((13, 1, 1), (12, 0, 0)), ((0, 0, 20), (0, 0, 12)),
                                       ((1, 1, 1), (1, 1, 1))]):
        new.copy_(server.ints(*more))
        q, k, v = server.rows(rows)
        q_in.copy_(q), k_in.copy_(k), v_in.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        server.verify(out.cpu(), taken, [0, taken[0], taken[0] + taken[1]], q, k, v, f"replay {i}")


@pytest.mark.parametrize("batch", [1, 5, 257, 1000, 4096])
def test_tables_leave_out_what_has_no_row(gpu_device, batch):
    """page_tables with `truncate` is page_tables of the lengths that fit."""
    from shareprefill_amd import ops

    gen = torch.Generator().manual_seed(batch)
    dev = gpu_device
    lens = torch.randint(0, 60, (batch,), generator=gen).to(torch.int32)
    new = torch.where(torch.rand(batch, generator=gen) < 0.4, torch.randint(0, 40, (batch,), generator=gen), torch.ones((), dtype=torch.int64)).to(torch.int32)
    new[batch // 3] = -4
    table = torch.arange(batch * 8).view(batch, 8).to(torch.int32)
    free = (batch * 8 + torch.randperm(batch * 4, generator=gen)).to(torch.int32)
    total = int(new.clamp(min=0).sum())
    for rows in sorted({0, 1, total // 2, max(total - 1, 0), total, total + 70}):
        ends = new.clamp(min=0).cumsum(0).clamp(max=rows)
        fits = torch.cat((ends[:1], ends.diff())).to(torch.int32)
        results = []
        for lengths, kw in ((new, dict(truncate=True)), (fits, {})):
            live = table.clone().to(dev)
            t = ops.page_tables(lens.to(dev), lengths.to(dev), live, free.to(dev), torch.tensor([free.numel()], dtype=torch.int32, device=dev), 16,
                                batch * 12, rows, **kw)
            results.append((live, *t))
        assert all(torch.equal(a, b) for a, b in zip(*results)), rows
