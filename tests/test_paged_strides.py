"""Strides of axes of length one say nothing: the paged and windowed operators take any there, and refuse them where the axis is longer.  Through
the C ABI with nothing that could launch: what passes the strides' check is refused for its missing workspace or its size."""

import pytest

from test_paged_refusals import P, _message, _paged, _window

from shareprefill_amd import _lib


@pytest.mark.parametrize("axis,strides", [
    (dict(tokens=1, batch=1), ["q_stride_n"]), (dict(hq=1, hkv=1), ["q_stride_h", "k_stride_h", "v_stride_h"]), (dict(hkv=1), ["k_stride_h", "v_stride_h"]),
    (dict(num_pages=1), ["k_stride_page", "v_stride_page"])])
@pytest.mark.parametrize("stride", [1, 3, 132, -7])
def test_paged_attention(axis, strides, stride):
    for name in strides:
        assert _paged(**axis, **{name: stride}, workspace=0) == -4, (name, _message())
        assert _paged(**{name: stride}, workspace=0) == -2, name


@pytest.mark.parametrize("axis,strides", [
    (dict(batch=1), ["q_stride_b", "k_stride_b", "v_stride_b"]), (dict(n=1), ["q_stride_n"]), (dict(hq=1, hkv=1), ["q_stride_h", "k_stride_h", "v_stride_h"]),
    (dict(n=1, n_keys=1), ["q_stride_n", "k_stride_n", "v_stride_n"])])
@pytest.mark.parametrize("stride", [1, 3, 132, -7])
def test_window_attention(axis, strides, stride):
    for name in strides:
        assert _window(**axis, **{name: stride}, workspace=0) == -4, (name, _message())
        assert _window(**{name: stride}, workspace=0) == -2, name


@pytest.mark.parametrize("axis,strides", [
    (dict(tokens=1), ["k_n", "v_n"]), (dict(hkv=1), ["k_h", "v_h", "kp_h", "vp_h"]), (dict(pages=1), ["kp_p", "vp_p"])])
@pytest.mark.parametrize("stride", [1, 3, 250, -7])
def test_cache_write(axis, strides, stride):
    def write(**kw):
        a = dict(k=P, v=P, kp=P, vp=P, slots=P, tokens=5, hkv=2, d=128, pages=9, page=16, k_n=256, k_h=128, v_n=256, v_h=128, kp_p=4096, kp_n=128,
                 kp_h=2048, vp_p=4096, vp_n=128, vp_h=2048, stream=0)
        a.update(kw)
        return _lib.load().sp_paged_cache_write_bf16(_lib.PAGED_WRITE_ARGS.pack(*a.values()))

    # (refused for another size, which is looked at behind the strides)
    beyond = dict(hkv=65537) if "hkv" not in axis else dict(tokens=1 << 41)
    for name in strides:
        assert write(**{**axis, **beyond, name: stride}) == -2 and "too many" in _message(), name
        assert write(**{name: stride}) == -2 and "aligned" in _message(), name


def test_python_takes_a_table_of_one_page_a_request_in_any_order(monkeypatch):
    import torch

    from shareprefill_amd import ops

    table = torch.zeros(1, 5, dtype=torch.int32).t()
    assert table.stride(1) != 1
    ops._check_table(table, 5, table.device)
    with pytest.raises(ValueError):
        ops._check_table(torch.zeros(3, 5, dtype=torch.int32).t(), 5, table.device)
