"""Calls whose launches would have more threads than a launch can have are refused on the host, before anything is launched; no pointer here is followed."""

from test_shared_refusals import _evict, _message


def test_evictions_of_too_many_heads():
    assert _evict(batch=4096, hkv=1024, workspace_bytes=1 << 60) == -2 and "too large" in _message()
