"""A cache without groups and weights gives pages back in as many operations as it needs, on the CPU."""

import torch
from torch.utils._python_dispatch import TorchDispatchMode

from test_paged_cache_groups import _cache, _fill, _mask


class _Count(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.n = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.n += not func.is_view
        return func(*args, **(kwargs or {}))


def test_what_only_groups_and_weights_need_is_left_out():
    counts = {}
    for name, kw in (("plain", dict(group_sizes=None)), ("weights", dict(group_sizes=None, key_weights=True)), ("groups", {})):
        cache = _cache(**kw)
        _fill(cache, 1, 3, 40)
        _fill(cache, 4, 2, 20)
        finished = _mask(1)
        with _Count() as ops:
            cache.release(finished)
        counts[name] = ops.n
        assert cache.free_count.item() == 18 and cache.lens.tolist() == [0, 0, 0, 0, 20, 0]
    # one each: >=, &, cumsum, +, -, where and its scalar, a cast, the pages put back, the count, the entries, the lengths
    assert counts["plain"] <= 12 < counts["weights"] < counts["groups"]
