"""What the entry points of the paged cache and the window refuse, through the C ABI: the checks run on the host before any GPU call, so
they need no GPU, and no pointer here is followed."""

import ctypes
import re

import pytest

from shareprefill_amd import _lib

P = 1 << 20  # an address, 16-byte aligned


def _paged(**kw):
    a = dict(q=P, k_pages=P, v_pages=P, block_table=P, seq_lens=P, cu_q=P, out=P, workspace=P, workspace_bytes=1 << 40, tokens=100, batch=4, hq=8,
             hkv=2, d=128, num_pages=50, page_size=16, table_width=9, table_stride=9, window=0, sinks=0, q_stride_n=1024, q_stride_h=128,
             k_stride_page=4096, k_stride_slot=128, k_stride_h=2048, v_stride_page=4096, v_stride_slot=128, v_stride_h=2048, softmax_scale=0.1,
             stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().sp_paged_attn_bf16(_lib.PAGED_ATTN_ARGS.pack(*a.values()))


def _window(**kw):
    a = dict(q=P, k=P, v=P, out=P, workspace=P, workspace_bytes=1 << 40, batch=2, n=10, n_keys=30, hq=8, hkv=2, d=128, window=0, sinks=0,
             q_stride_b=10240, q_stride_n=1024, q_stride_h=128, k_stride_b=8192, k_stride_n=128, k_stride_h=4096, v_stride_b=8192, v_stride_n=128,
             v_stride_h=4096, softmax_scale=0.1, stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().sp_window_attn_bf16(_lib.WINDOW_ATTN_ARGS.pack(*a.values()))


def _message():
    return _lib.load().sp_last_error().decode()


@pytest.mark.parametrize("code,kw", [
    (-1, dict(hq=7)), (-1, dict(hkv=0)), (-1, dict(softmax_scale=0.0)), (-1, dict(softmax_scale=float("nan"))), (-1, dict(window=-1)),
    (-1, dict(sinks=-1)), (-2, dict(d=96)), (-2, dict(d=256))])
def test_both_attentions_refuse(code, kw):
    assert _paged(**kw) == code and "sp_paged_attn_bf16" in _message()
    assert _window(**kw) == code and "sp_window_attn_bf16" in _message()


@pytest.mark.parametrize("code,kw", [
    (-1, dict(batch=0)), (-2, dict(batch=4097)), (-1, dict(tokens=-1)), (-1, dict(cu_q=0)), (-1, dict(q=0)), (-1, dict(block_table=0)),
    (-1, dict(seq_lens=0)), (-1, dict(out=0)), (-1, dict(num_pages=0)), (-1, dict(table_width=0)), (-2, dict(page_size=24)), (-2, dict(page_size=8)),
    (-2, dict(page_size=2048)), (-2, dict(table_width=1 << 27)), (-2, dict(tokens=1 << 31)), (-2, dict(q=P + 8)), (-2, dict(k_pages=P + 2)),
    (-2, dict(out=P + 4)), (-2, dict(k_stride_slot=132)), (-2, dict(v_stride_slot=1 << 25)), (-2, dict(k_stride_slot=-128)),
    (-2, dict(q_stride_h=130)), (-2, dict(v_stride_page=4097)), (-4, dict(workspace=0)), (-4, dict(workspace=P + 8)), (-4, dict(workspace_bytes=1000))])
def test_paged_attention_refuses(code, kw):
    assert _paged(**kw) == code, _message()


@pytest.mark.parametrize("code,kw", [
    (-1, dict(batch=0)), (-2, dict(batch=5000)), (-1, dict(n=-1)), (-1, dict(n=31)), (-2, dict(n_keys=(1 << 30) + 1)), (-1, dict(q=0)), (-1, dict(v=0)),
    (-2, dict(k=P + 8)), (-2, dict(k_stride_n=4)), (-2, dict(v_stride_n=1 << 24)), (-2, dict(q_stride_b=3)), (-4, dict(workspace=0))])
def test_window_attention_refuses(code, kw):
    assert _window(**kw) == code, _message()


def test_nothing_to_do_is_no_error():
    assert _paged(tokens=0, q=0, out=0, workspace=0, workspace_bytes=0) == 0
    assert _window(n=0, q=0, out=0, workspace=0, workspace_bytes=0) == 0
    lib = _lib.load()
    assert lib.sp_paged_attn_workspace_bytes(0, 4, 8, 2, 128, 0) == 0 == lib.sp_window_attn_workspace_bytes(0, 4, 4, 8, 2, 128)
    assert lib.sp_paged_attn_workspace_bytes(4, 4, 7, 2, 128, 1) == 0


def test_tables_and_writes_refuse():
    lib = _lib.load()

    def tables(**kw):
        a = dict(lens=P, new=P, table=P, free=P, count=P, seq=P + 64, cu=P + 128, slots=P + 256, positions=P + 512, left=P + 1024, batch=4, page=16,
                 pages=50, width=9, stride=9, room=50, tokens=10, stream=0)
        a.update(kw)
        return lib.sp_paged_tables(_lib.PAGED_TABLES_ARGS.pack(*a.values()))

    for code, kw in [(-1, dict(batch=0)), (-2, dict(batch=4097)), (-1, dict(lens=0)), (-1, dict(free=0)), (-1, dict(slots=0)), (-1, dict(stride=8)),
                     (-1, dict(width=0)), (-2, dict(page=17)), (-2, dict(page=2048)), (-1, dict(tokens=-1)), (-1, dict(room=-1)),
                     (-2, dict(width=1 << 27, stride=1 << 27)), (-1, dict(left=P)), (-1, dict(seq=P))]:
        assert tables(**kw) == code, (kw, _message())

    def write(**kw):
        a = dict(k=P, v=P, kp=P, vp=P, slots=P, tokens=5, hkv=2, d=128, pages=9, page=16, k_n=256, k_h=128, v_n=256, v_h=128, kp_p=4096, kp_n=128,
                 kp_h=2048, vp_p=4096, vp_n=128, vp_h=2048, stream=0)
        a.update(kw)
        return lib.sp_paged_cache_write_bf16(_lib.PAGED_WRITE_ARGS.pack(*a.values()))

    for code, kw in [(-1, dict(k=0)), (-1, dict(slots=0)), (-1, dict(tokens=-1)), (-1, dict(hkv=0)), (-2, dict(d=12)), (-2, dict(page=48)),
                     (-2, dict(kp=P + 8)), (-2, dict(vp_h=2047)), (-2, dict(k_n=250)), (-2, dict(tokens=1 << 45))]:
        assert write(**kw) == code, (kw, _message())
    assert write(tokens=0) == 0 and write(pages=0) == 0


def test_argument_structs_are_those_of_the_header():
    header = open(_lib.__file__.replace("shareprefill_amd/_lib.py", "include/shareprefill_hip.h")).read()
    for name, packed in (("sp_paged_tables_args", _lib.PAGED_TABLES_ARGS), ("sp_paged_write_args", _lib.PAGED_WRITE_ARGS),
                         ("sp_paged_attn_args", _lib.PAGED_ATTN_ARGS), ("sp_window_attn_args", _lib.WINDOW_ATTN_ARGS)):
        body = header[header.index("typedef struct %s {" % name):header.index("} %s;" % name)].split("{")[1]
        size, kinds = 0, ""
        for line in re.findall(r"([^;]+);", body):
            line = line.strip()
            names = [n.strip() for n in re.sub(r"^(const\s+)?(void|int32_t|int64_t|uint64_t|double|sp_stream_t)\s*", "", line).split(",")]
            kind = "P" if "*" in line or line.startswith("sp_stream_t") else {"uint64_t": "Q", "int64_t": "q", "double": "d"}[line.split()[0]]
            kinds += kind * len(names)
            size += 8 * len(names)
        assert packed.size == size
        expanded = "".join((c * int(n or 1)) for n, c in re.findall(r"(\d*)([PQqd])", packed.format))
        assert expanded == kinds
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_cpu_tensors_are_refused():
    import torch

    from shareprefill_amd import PagedKVCache, ops

    q = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    pool = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_attention(q, pool, pool, table, lens, 0.1)
    with pytest.raises(ValueError, match="GPU"):
        ops.window_attention(q[None], q[None], q[None], 0.1)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_cache_write(q, q, pool, pool, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        PagedKVCache(1, 4, 2, 64, 1, 32, 16, device="cpu").begin_step()
