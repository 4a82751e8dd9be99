"""The bound of an eviction's waits: a workgroup that has waited in vain writes nothing, and the request's length says so."""

import pytest
import torch

from test_gpu_evict import definition

pytestmark = pytest.mark.gpu


def test_waits_in_vain(gpu_device):
    """A bound of no looks at all: whoever has to wait gives up, whatever the others have done.  Requests that one chunk moves, or that keep everything, are done."""
    from shareprefill_amd import _lib, ops

    dev, page, hkv, d, budget, recent = gpu_device, 16, 2, 64, 300, 20
    lens, first = [1000, 310, 420, 500], [20, 0, 130, 0]  # kept rows, by chunks of 128: 320, none moves, none moves, 320
    gen = torch.Generator().manual_seed(1)
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=gen).to(torch.int32)
    table, at = torch.full((4, max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pools = [torch.randn(sum(need) + 2, hkv, page, d, generator=gen).to(torch.bfloat16) for _ in range(2)]
    pools.append(torch.rand(sum(need) + 2, hkv, page, generator=gen))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)

    def call(budget, polls, live):
        k, v, w = live
        lib, left = _lib.load(), torch.full((4,), 77, dtype=torch.int32, device=dev)
        tab, ln, fi = table.to(dev), ints(lens), ints(first)
        need_bytes = lib.sp_paged_evict_workspace_bytes(4, hkv, d, k.shape[0], page, table.shape[1])
        ws = torch.empty(need_bytes, dtype=torch.uint8, device=dev)
        st = lib.sp_paged_evict_bounded_bf16(_lib.EVICT_ARGS.pack(
            k.data_ptr(), v.data_ptr(), w.data_ptr(), tab.data_ptr(), ln.data_ptr(), fi.data_ptr(), left.data_ptr(), ws.data_ptr(), need_bytes, 4, hkv, d,
            k.shape[0], page, tab.shape[1], tab.stride(0), budget, recent, k.stride(0), k.stride(2), k.stride(1), v.stride(0), v.stride(2), v.stride(1),
            w.stride(0), w.stride(1), ops._stream_handle(dev)), polls)
        torch.cuda.synchronize()
        return st, left.tolist()

    for budget, lost in ((300, [0, 3]), (100, []), (0, [])):  # (at most 120 rows: one chunk)
        live = [x.to(dev) for x in pools]
        st, left = call(budget, 0, live)
        want, lengths = definition([x.clone() for x in pools], table, lens, first, budget, recent, page)
        assert st == 0 and left == [-1 if b in lost else n for b, n in enumerate(lengths)]
        for b in range(4):
            for j in range(lens[b] if b not in lost else first[b]):
                place = (int(table[b, j // page]), slice(None), j % page)
                for x, y in zip(live, want):
                    assert torch.equal(x[place].cpu(), y[place]), (budget, b, j)
        spare = order[-2:].long()
        for x, y in zip(live, pools):
            assert torch.equal(x.cpu()[spare], y[spare])
    live = [x.to(dev) for x in pools]
    want, lengths = definition([x.clone() for x in pools], table, lens, first, 300, recent, page)
    assert call(300, 1 << 20, live) == (0, lengths)
    for x, y in zip(live, want):
        assert torch.equal(x.cpu(), y)
    assert call(300, -1, live)[0] == -1
