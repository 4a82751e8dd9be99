"""What PagedKVCache refuses before anything reaches the GPU."""

import pytest
import torch

from shareprefill_amd import PagedKVCache, ops


def test_attend_takes_the_steps_rows(monkeypatch):
    """Rows that are missing would move the others of their request to other positions: offsets are held to the rows there are, and a request's
    rows are its last ones."""
    cache = PagedKVCache(1, 4, 2, 64, 2, 32, 16, device="cpu")
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.int32)
    cache.tables = ops.PageTables(zeros(2), zeros(3), torch.zeros(7, dtype=torch.int64), zeros(7), zeros(1))
    taken = []
    monkeypatch.setattr(ops, "paged_attention", lambda q, *args, **kw: taken.append(q.shape[1]))
    cache.attend(0, torch.zeros(4, 7, 64, dtype=torch.bfloat16), 0.1)
    for rows in (6, 8, 0):
        with pytest.raises(ValueError, match="rows"):
            cache.attend(0, torch.zeros(4, rows, 64, dtype=torch.bfloat16), 0.1)
    assert taken == [7]
