"""Block tables for lengths whose sums pass 32 bits: what is within reach is right, nothing else is touched."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("new", [[TOP] * 6, [20, TOP, 5, TOP, TOP, 3], [20, 2 ** 30 - 1, 1, 2 ** 30 - 1, 2 ** 30, 7], [20] + [TOP] * 700])
def test_many_lengths_near_the_largest(gpu_device, new):
    from shareprefill_amd import ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    page, width, tokens, pages = 16, 4, 300, 5000
    table = torch.full((len(new), width), -1, dtype=torch.int32, device=gpu_device)
    got = ops.page_tables(ints([0] * len(new)), ints(new), table, ints(list(range(pages))), ints([pages]), page, pages, tokens)
    held = [min(n, 2 ** 30 - 1) for n in new]
    need = [min(-(-n // page), width) for n in held]
    stack, rows, slots = list(range(pages)), [], []
    for n, opened in zip(held, need):
        rows.append([stack.pop() for _ in range(opened)] + [-1] * (width - opened))
        slots += [rows[-1][p // page] * page + p % page if p < width * page else -1 for p in range(min(n, tokens - len(slots)))]
    assert table.tolist() == rows
    assert got.seq_lens.tolist() == held
    assert got.cu_new.tolist() == [min(sum(held[:i]), 2 ** 30) for i in range(len(new) + 1)]
    assert got.slots.tolist() == (slots + [-1] * tokens)[:tokens]
    assert got.free_left.tolist() == [pages - sum(need)]
