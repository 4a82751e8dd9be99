"""Bookkeeping of a cache whose requests share pages, on the CPU: no kernel takes part in it."""

import pytest
import torch

from shareprefill_amd.paged_cache import PagedKVCache


def _cache(**kw):
    return PagedKVCache(**{**dict(num_layers=1, num_pages=20, num_kv_heads=1, head_dim=64, max_requests=6, max_tokens=128, page_size=16, device="cpu",
                                  group_sizes=[3, 2]), **kw})


def _fill(cache, row, pages, length):
    """as page_tables does"""
    n = cache.free_count.item()
    cache.block_table[row, :pages] = cache._stack[n - pages:n].flip(0)
    cache.free_count -= pages
    cache.lens[row] = length


def _mask(*rows):
    m = torch.zeros(6, dtype=torch.bool)
    m[list(rows)] = True
    return m


def _whole(cache):
    """every page is on the stack or named"""
    free = cache._stack[:cache.free_count.item()].tolist()
    named = set(cache.block_table[cache.block_table >= 0].tolist())
    assert len(set(free)) == len(free) and not set(free) & named and len(free) + len(named) == cache.num_pages


def test_shared_pages_are_named_and_come_back_when_the_last_row_lets_go():
    cache = _cache()
    _fill(cache, 0, 4, 60)
    _fill(cache, 3, 2, 32)
    cache.share(0, 55)  # three whole pages
    cache.share(1, 32)
    assert cache.shared_lens.tolist() == [48, 32] and cache.lens.tolist() == [60, 48, 48, 32, 32, 0]
    assert torch.equal(cache.block_table[1, :3], cache.block_table[0, :3]) and (cache.block_table[1, 3:] == -1).all()
    assert cache.block_table[4, :2].tolist() == cache.block_table[3, :2].tolist() and (cache.block_table[5] == -1).all()
    _whole(cache)
    cache.release(_mask(1))
    assert cache.free_count.item() == 14 and (cache.block_table[1] == -1).all() and cache.shared_lens.tolist() == [48, 32]
    cache.join(_mask(0, 1, 5))  # (a first row and one of no group stay as they are)
    assert cache.lens.tolist() == [60, 48, 48, 32, 32, 0] and torch.equal(cache.block_table[1, :3], cache.block_table[0, :3])
    cache.release(_mask(0))  # the others go on with its shared pages
    assert cache.shared_lens.tolist() == [0, 32] and cache.free_count.item() == 15
    _whole(cache)
    cache.release(_mask(1, 2, 3, 4))  # each page once
    assert cache.free_count.item() == 20 and (cache.block_table == -1).all() and cache.lens.tolist() == [0] * 6
    _whole(cache)


def test_pages_go_back_in_the_order_of_the_table_with_and_without_groups():
    stacks = []
    for sizes in ([3, 2], None):
        cache = _cache(group_sizes=sizes)
        for row, pages in ((0, 3), (2, 1), (5, 4)):
            _fill(cache, row, pages, pages * 16)
        cache.release(_mask(0, 5))
        stacks.append(cache._stack[:cache.free_count.item()].tolist())
        _whole(cache)
    assert stacks[0] == stacks[1]


def test_refusals():
    for sizes in ([0], [7], [3, 4], [-1]):
        with pytest.raises(ValueError):
            _cache(group_sizes=sizes)
    cache = _cache()
    for call in (lambda: cache.share(2, 16), lambda: cache.share(-1, 16), lambda: cache.share(0, -1), lambda: cache.share(0, 129),
                 lambda: cache.join(torch.zeros(5, dtype=torch.bool)), lambda: cache.join(torch.zeros(6))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        cache.evict(4, 4)
    with pytest.raises(RuntimeError):
        cache.observe(0, torch.zeros(1, 1, 64), 0.1)


def test_keys_in_pages_of_several_requests_stay_apart_behind_the_end_of_a_first_row():
    cache = _cache()
    _fill(cache, 0, 4, 60)
    cache.dropped[0] = 7
    cache.share(0, 50)
    assert cache._held.tolist() == cache._joined.tolist() == [48, 48, 48, 0, 0, 0]
    assert cache.dropped.tolist() == [7, 7, 7, 0, 0, 0]  # (positions go on from the first row's)
    cache.release(_mask(0))
    assert cache._held.tolist() == [0, 48, 48, 0, 0, 0] and cache._joined.tolist() == [0] * 6 and cache.dropped.tolist() == [0, 7, 7, 0, 0, 0]
    _fill(cache, 0, 2, 32)
    cache.share(0, 16)  # the others are not empty: they keep what they have and are none of this start's
    assert cache.shared_lens.tolist() == [16, 0] and cache._joined.tolist() == [16, 0, 0, 0, 0, 0] and cache._held.tolist() == [16, 48, 48, 0, 0, 0]
    assert cache.lens.tolist() == [32, 48, 48, 0, 0, 0] and cache.dropped.tolist() == [0, 7, 7, 0, 0, 0]
    assert not set(cache.block_table[0, :2].tolist()) & set(cache.block_table[1, :3].tolist())
    cache.release(_mask(2))
    cache.join(_mask(1, 2))
    assert cache.lens.tolist() == [32, 48, 16, 0, 0, 0] and cache._joined.tolist() == [16, 0, 16, 0, 0, 0]
    _whole(cache)
    cache.release(_mask(0, 1, 2))
    assert cache.free_count.item() == 20 and cache._held.tolist() == [0] * 6


def test_more_requests_than_groups_and_weights_take():
    for kw in (dict(group_sizes=[2]), dict(group_sizes=None, key_weights=True)):
        with pytest.raises(ValueError, match="1024"):
            _cache(max_requests=1025, **kw)
    assert _cache(max_requests=1025, group_sizes=None).max_requests == 1025
