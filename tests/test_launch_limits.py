"""Calls whose launches would have more threads than a launch can have are refused on the host, before anything is launched; no pointer here is followed."""

from test_shared_refusals import _evict, _message, _shared, _weigh


def test_evictions_of_too_many_heads():
    assert _evict(batch=4096, hkv=1024, workspace_bytes=1 << 60) == -2 and "too large" in _message()


def test_attention_and_weights_of_too_many_rows():
    """The joining launches have a thread for four channels of a row, or a wave a row."""
    many = dict(batch=4, cu_q=1 << 20, workspace_bytes=1 << 60)
    assert _shared(tokens=1 << 24, weights=0, hq=8, **many) == -2 and "too many" in _message()
    assert _shared(tokens=1 << 25, weights=0, hq=8, d=64, k_stride_slot=64, v_stride_slot=64, **many) == -2 and "too many" in _message()
    assert _weigh(tokens=1 << 23, hq=8, **many) == -2 and "too many" in _message()
    assert _weigh(tokens=(1 << 26) - 1, hq=1, hkv=1, **many) == -2 and "too many" in _message()  # (a quarter of a workgroup)
