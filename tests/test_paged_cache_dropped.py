"""How many keys evictions have taken from a request, which its positions count, where rows of a group begin behind its first row: on the CPU, no kernel
takes part in it."""

import pytest
import torch

from shareprefill_amd import ops
from test_paged_cache_groups import _cache, _fill, _mask


@pytest.fixture
def evicting(monkeypatch):
    """Evictions' lengths without the kernel that moves what stays."""

    def lengths(k_pages, v_pages, weights, block_table, seq_lens, budget, recent, first=None):
        mid = (seq_lens - torch.minimum(first, seq_lens) - recent).clamp(min=0)
        return seq_lens - mid + mid.clamp(max=budget)

    monkeypatch.setattr(ops, "paged_evict", lengths)
    return _cache(key_weights=True)


def test_rows_behind_an_ended_start_count_nothing(evicting):
    cache = evicting
    _fill(cache, 0, 6, 90)
    cache.evict(budget=20, recent=20)
    assert cache.lens.tolist()[0] == 40 and cache.dropped.tolist()[0] == 50
    cache.share(0, 32)
    assert cache.lens.tolist()[:3] == [40, 32, 32] and cache.dropped.tolist()[:3] == [50, 50, 50]
    finished = _mask(0, 1, 2)
    cache.release(finished)
    cache.join(finished)  # behind nothing
    assert cache.lens.tolist() == [0] * 6 and cache.dropped.tolist() == [0] * 6


def test_rows_that_join_later_count_what_the_start_has_lost(evicting):
    cache = evicting
    _fill(cache, 0, 6, 90)
    cache.evict(budget=20, recent=20)
    cache.share(0, 32)
    cache.release(_mask(1))
    cache.join(_mask(1))
    assert cache.lens.tolist()[:3] == [40, 32, 32] and cache.dropped.tolist()[:3] == [50, 50, 50]


def test_a_start_of_less_than_a_page_counts_nothing(evicting):
    cache = evicting
    _fill(cache, 0, 6, 90)
    cache.evict(budget=20, recent=20)
    cache.share(0, 10)
    assert cache.lens.tolist()[:3] == [40, 0, 0] and cache.dropped.tolist()[:3] == [50, 0, 0]


def test_a_start_in_front_of_all_that_went_counts_nothing(evicting):
    """Keys among the first ones of every eviction stand where they stood in the prompt."""
    cache = evicting
    _fill(cache, 0, 6, 90)
    _fill(cache, 3, 6, 90)
    cache.evict(budget=10, recent=10, sinks=40)
    cache.evict(budget=4, recent=4, sinks=33)
    assert cache.lens.tolist() == [41, 0, 0, 41, 0, 0] and cache.dropped.tolist() == [49, 0, 0, 49, 0, 0]
    cache.share(0, 33)  # 32 keys
    assert cache.lens.tolist()[:3] == [41, 32, 32] and cache.dropped.tolist()[:3] == [49, 0, 0]
    cache.evict(budget=0, recent=0, sinks=20, rows=_mask(3))
    assert cache.lens.tolist()[3] == 20 and cache.dropped.tolist()[3] == 70
    cache.share(1, 16)
    assert cache.dropped.tolist() == [49, 0, 0, 70, 0, 0]
    cache.release(_mask(3, 4))
    _fill(cache, 3, 6, 90)  # (another request: what an earlier one kept is none of its)
    cache.evict(budget=10, recent=10, sinks=2, rows=_mask(3))
    cache.share(1, 16)
    assert cache.lens.tolist()[3:5] == [22, 16] and cache.dropped.tolist()[3:5] == [68, 68]


def test_a_request_that_an_eviction_has_spoilt(monkeypatch):
    """One layer of it is enough; its first keys stay, its pages go back, and its release ends it."""
    cache = _cache(key_weights=True, num_layers=3)
    _fill(cache, 0, 6, 90)
    _fill(cache, 5, 5, 80)
    left = iter([[30, 0, 0, 0, 0, 80], [-1, 0, 0, 0, 0, 80], [30, 0, 0, 0, 0, 80]])
    monkeypatch.setattr(ops, "paged_evict", lambda *a, **kw: torch.tensor(next(left), dtype=torch.int32))
    cache.evict(budget=20, recent=2, sinks=8)
    assert cache.lens.tolist() == [8, 0, 0, 0, 0, 80] and cache.lost.tolist() == [True] + [False] * 5
    assert (cache.block_table[0] >= 0).sum() == 1 and cache.free_count.item() == 20 - 6 and cache.dropped.tolist()[0] == 82
    cache.release(_mask(0))
    assert cache.lost.tolist() == [False] * 6 and cache.free_count.item() == 20 - 5


def test_a_request_that_an_eviction_left_nothing_of_is_no_empty_row(evicting):
    cache = evicting
    _fill(cache, 0, 3, 40)
    _fill(cache, 1, 2, 30)
    cache.evict(budget=0, recent=0, rows=_mask(1))
    assert cache.lens.tolist()[:2] == [40, 0] and cache.dropped.tolist()[:2] == [0, 30]
    cache.share(0, 40)
    cache.join(_mask(1))
    assert cache.lens.tolist()[:3] == [40, 0, 32] and cache.dropped.tolist()[:3] == [0, 30, 0] and (cache.block_table[1] == -1).all()
    cache.release(_mask(1))
    cache.join(_mask(1))
    assert cache.lens.tolist()[:3] == [40, 32, 32] and cache.dropped.tolist()[:3] == [0, 0, 0]


def test_share_says_where_the_other_rows_begin():
    cache = _cache()
    _fill(cache, 0, 4, 60)
    assert [cache.share(0, n) for n in (0, 15, 16, 55)] == [0, 0, 16, 48]
    assert cache.lens.tolist()[:3] == [60, 16, 16]  # (rows that are no longer empty stay as they are)
