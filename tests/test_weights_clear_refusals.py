"""What sp_paged_weights_clear refuses, through the C ABI: the checks run on the host before any GPU call; no pointer here is followed."""

import pytest

from shareprefill_amd import _lib

P = 1 << 20


@pytest.mark.parametrize("code,kw", [
    (-1, dict(tokens=-1)), (-1, dict(hkv=0)), (-1, dict(num_pages=-1)), (-2, dict(page_size=24)), (-2, dict(page_size=2048)), (-1, dict(weights=0)),
    (-1, dict(slots=0)), (-2, dict(hkv=65537)), (-2, dict(num_pages=1 << 31)), (-2, dict(tokens=(1 << 29) + 1)), (0, dict(tokens=0, slots=0)),
    (0, dict(num_pages=0, weights=0))])
def test_refusals(code, kw):
    a = dict(weights=P, slots=P, tokens=5, hkv=2, num_pages=50, page_size=16, w_stride_page=32, w_stride_h=16, stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    assert _lib.load().sp_paged_weights_clear(*a.values()) == code
    assert code == 0 or "sp_paged_weights_clear" in _lib.load().sp_last_error().decode()
