"""What PagedKVCache and its tables refuse before anything reaches the GPU."""

import pytest
import torch

from shareprefill_amd import PagedKVCache, _lib, ops


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


@pytest.mark.parametrize("entry", ["sp_paged_tables", "sp_paged_tables_truncated"])
def test_both_tables_refuse_alike(entry):
    P = 1 << 20

    def tables(**kw):
        a = dict(lens=P, new=P, table=P, free=P, count=P, seq=P + 64, cu=P + 128, slots=P + 256, positions=P + 512, left=P + 1024, batch=4, page=16,
                 pages=50, width=9, stride=9, room=50, tokens=10, stream=0)
        a.update(kw)
        return getattr(_lib.load(), entry)(_lib.PAGED_TABLES_ARGS.pack(*a.values()))

    for code, kw in [(-1, dict(batch=0)), (-2, dict(batch=4097)), (-1, dict(lens=0)), (-1, dict(slots=0)), (-1, dict(stride=8)), (-1, dict(width=0)),
                     (-2, dict(page=17)), (-1, dict(tokens=-1)), (-2, dict(tokens=(1 << 30) + 1)), (-1, dict(room=-1)), (-1, dict(seq=P))]:
        assert tables(**kw) == code and f"{entry}:" in _lib.load().sp_last_error().decode(), kw
