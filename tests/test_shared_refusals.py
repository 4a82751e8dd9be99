"""What the entry points for shared starts, key weights and eviction refuse, through the C ABI: the checks run on the host before any GPU call, so
they need no GPU, and no pointer here is followed."""

import pytest

from shareprefill_amd import _lib

P = 1 << 20  # an address, 16-byte aligned


def _shared(**kw):
    a = dict(q=P, k_pages=P, v_pages=P, block_table=P, seq_lens=P, cu_q=0, shared_lens=P, cu_groups=P, joined=0, weights=P, out=P, workspace=P, workspace_bytes=1 << 40,
             tokens=4, batch=4, groups=2, hq=8, hkv=2, d=128, num_pages=50, page_size=16, table_width=9, table_stride=9, q_stride_n=1024, q_stride_h=128,
             k_stride_page=4096, k_stride_slot=128, k_stride_h=2048, v_stride_page=4096, v_stride_slot=128, v_stride_h=2048, w_stride_page=32, w_stride_h=16,
             softmax_scale=0.1, stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().sp_shared_attn_bf16(_lib.SHARED_ATTN_ARGS.pack(*a.values()))


def _weigh(**kw):
    a = dict(q=P, k_pages=P, block_table=P, seq_lens=P, cu_q=P, first=0, weights=P, workspace=P, workspace_bytes=1 << 40, tokens=100, batch=4, hq=8, hkv=2,
             d=128, num_pages=50, page_size=16, table_width=9, table_stride=9, accumulate=0, q_stride_n=1024, q_stride_h=128, k_stride_page=4096,
             k_stride_slot=128, k_stride_h=2048, w_stride_page=32, w_stride_h=16, softmax_scale=0.1, stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().sp_paged_key_weights_bf16(_lib.KEY_WEIGHTS_ARGS.pack(*a.values()))


def _evict(**kw):
    a = dict(k_pages=P, v_pages=P, weights=P, block_table=P, seq_lens=P, first=0, new_lens=P + 64, workspace=P, workspace_bytes=1 << 40, batch=4, hkv=2,
             d=128, num_pages=50, page_size=16, table_width=9, table_stride=9, budget=30, recent=4, k_stride_page=4096, k_stride_slot=128,
             k_stride_h=2048, v_stride_page=4096, v_stride_slot=128, v_stride_h=2048, w_stride_page=32, w_stride_h=16, stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().sp_paged_evict_bf16(_lib.EVICT_ARGS.pack(*a.values()))


def _message():
    return _lib.load().sp_last_error().decode()


@pytest.mark.parametrize("code,kw", [
    (-1, dict(hq=7)), (-1, dict(hkv=0)), (-2, dict(d=96)), (-2, dict(d=256)), (-1, dict(softmax_scale=0.0)), (-1, dict(softmax_scale=float("nan"))),
    (-1, dict(batch=0)), (-2, dict(batch=1025, tokens=1025)), (-1, dict(tokens=-1)), (-1, dict(table_width=0)), (-1, dict(num_pages=0)),
    (-2, dict(page_size=24)), (-2, dict(page_size=2048)), (-2, dict(page_size=8)), (-2, dict(table_width=1 << 27)), (-1, dict(block_table=0)),
    (-1, dict(seq_lens=0)), (-1, dict(q=0)), (-1, dict(k_pages=0)), (-2, dict(q=P + 8)), (-2, dict(k_pages=P + 2)), (-2, dict(k_stride_slot=132)),
    (-2, dict(q_stride_h=130)), (-4, dict(workspace=0)), (-4, dict(workspace=P + 8)), (-4, dict(workspace_bytes=100)), (-2, dict(num_pages=1 << 31))])
def test_attention_and_weights_refuse(code, kw):
    assert _shared(**kw) == code and "sp_shared_attn_bf16" in _message(), _message()
    tokens = dict(kw)
    if "tokens" in tokens:
        tokens["tokens"] = min(tokens["tokens"], 100)
    assert _weigh(**tokens) == code and "sp_paged_key_weights_bf16" in _message(), _message()


@pytest.mark.parametrize("code,kw", [
    (-1, dict(groups=-1)), (-1, dict(groups=5)), (-1, dict(shared_lens=0)), (-1, dict(cu_groups=0)), (-1, dict(tokens=3)), (-2, dict(cu_q=P)),
    (-2, dict(hq=34)), (-1, dict(out=0)), (-2, dict(out=P + 4)), (-2, dict(v_stride_slot=1 << 25)), (-2, dict(k_stride_slot=-128)), (-1, dict(v_pages=0)),
    (-2, dict(v_stride_page=4097)), (-2, dict(tokens=1 << 29, batch=4, cu_q=P, weights=0))])
def test_shared_attention_refuses(code, kw):
    assert _shared(**kw) == code, _message()


@pytest.mark.parametrize("code,kw", [(-1, dict(cu_q=0)), (-1, dict(weights=0)), (-2, dict(tokens=1 << 29))])
def test_key_weights_refuse(code, kw):
    assert _weigh(**kw) == code, _message()


@pytest.mark.parametrize("code,kw", [
    (-1, dict(batch=0)), (-2, dict(batch=4097)), (-1, dict(hkv=0)), (-1, dict(budget=-1)), (-1, dict(recent=-1)), (-2, dict(d=4)), (-2, dict(d=0)),
    (-2, dict(page_size=24)), (-2, dict(table_width=1 << 27)), (-1, dict(k_pages=0)), (-1, dict(v_pages=0)), (-1, dict(weights=0)), (-1, dict(block_table=0)),
    (-1, dict(seq_lens=0)), (-1, dict(new_lens=0)), (-1, dict(new_lens=P)), (-1, dict(first=P + 64)), (-2, dict(k_pages=P + 8)), (-2, dict(v_stride_slot=4)),
    (-4, dict(workspace=0)), (-4, dict(workspace_bytes=100)), (-2, dict(num_pages=1 << 29)), (-2, dict(d=65544))])
def test_eviction_refuses(code, kw):
    assert _evict(**kw) == code and "sp_paged_evict_bf16" in _message(), _message()


def test_nothing_to_do_is_no_error():
    assert _shared(tokens=0, batch=1, groups=0, cu_q=P, weights=0, q=0, out=0, workspace=0, workspace_bytes=0) == 0
    assert _weigh(tokens=0, q=0, workspace=0, workspace_bytes=0) == 0


def test_workspaces_of_calls_that_are_refused_are_none():
    lib = _lib.load()
    assert lib.sp_shared_attn_workspace_bytes(4, 4, 2, 8, 3, 128, 1, 0) == 0 and lib.sp_shared_attn_workspace_bytes(4, 2000, 2, 8, 2, 128, 1, 0) == 0
    assert lib.sp_paged_key_weights_workspace_bytes(4, 0, 8, 2) == 0 and lib.sp_paged_evict_workspace_bytes(0, 2, 128, 50, 16, 9) == 0
    assert lib.sp_shared_attn_workspace_bytes(4, 4, 2, 8, 2, 128, 1, 800) > lib.sp_shared_attn_workspace_bytes(4, 4, 2, 8, 2, 128, 1, 0) > 0
    assert lib.sp_paged_evict_workspace_bytes(4, 2, 128, 50, 16, 9) == 8 * 2 * 50 * 16 + 8 * 3 * 4 + 4 * 256
