"""The paged-cache operators without a GPU: what the C ABI refuses before it
touches a device, workspace sizes, and the Python checks."""
import ctypes

import pytest
import torch

# 16-byte aligned, never dereferenced: every call fails validation first.
P = ctypes.c_void_p(0x10000)


def record(fp8lin, **kw):
    from fp8lin._lib import PagedCacheRecord
    d = dict(k=0x10000, v=0x20000, k_page=16 * 2 * 64, k_slot=2 * 64, k_head=64, v_page=16 * 2 * 64, v_slot=2 * 64, v_head=64, pages=4,
             page_size=16, kv_heads=2, head_dim=64, fp8=0, k_scale=None, v_scale=None)
    d.update(kw)
    return PagedCacheRecord(**d)


BAD_CACHES = [
    (dict(k=None), 2), (dict(v=0), 2), (dict(k=0x10002), 2),
    (dict(page_size=8), 1), (dict(page_size=24), 1), (dict(page_size=0), 1), (dict(page_size=-16), 1), (dict(page_size=1 << 21), 1),
    (dict(pages=0), 1), (dict(kv_heads=0), 1), (dict(head_dim=0), 1), (dict(head_dim=8192, k_slot=16384, v_slot=16384), 1),
    (dict(k_slot=56), 2), (dict(v_slot=-128), 2), (dict(v_head=60), 2), (dict(k_page=-2048), 2), (dict(k_slot=1 << 28), 2),
    (dict(fp8=1), 2), (dict(fp8=1, k_scale=0x100), 2), (dict(k_scale=0x100), 2), (dict(fp8=1, k_scale=0x100, v_scale=0x100, k_head=72), 2),
]


def attention(L, rec, **kw):
    d = dict(q=P, q_token=256, q_head=64, gate=None, gate_token=0, gate_head=0, table=P, table_ld=8, width=8, offsets=P, lengths=P,
             requests=3, tokens=5, heads=4, max_count=2, causal=1, scale=0.125, out=P, out_token=256, out_head=64, workspace=P,
             workspace_bytes=1 << 40, stream=None)
    d.update(kw)
    return L.fp8lin_paged_attention(ctypes.byref(rec) if rec is not None else None, *d.values())


@pytest.mark.parametrize("change,code", BAD_CACHES, ids=str)
def test_bad_caches(fp8lin, change, code):
    L, rec = fp8lin.lib(), record(fp8lin, **change)
    assert L.fp8lin_paged_append(ctypes.byref(rec), P, 128, 64, P, 128, 64, P, 3, None) == code
    assert attention(L, rec) == code
    assert L.fp8lin_last_error()


@pytest.mark.parametrize("change,code", [
    (dict(q=None), 2), (dict(table=None), 2), (dict(offsets=None), 2), (dict(lengths=None), 2), (dict(out=None), 2),
    (dict(heads=3), 1), (dict(heads=0), 1), (dict(heads=-2), 1), (dict(tokens=-1), 1), (dict(tokens=1 << 30), 1), (dict(requests=0), 1),
    (dict(requests=8193), 1), (dict(width=0), 1), (dict(width=(1 << 26) + 1), 1), (dict(table_ld=7), 1), (dict(scale=0.0), 2),
    (dict(scale=-1.0), 2), (dict(scale=float("nan")), 2), (dict(scale=float("inf")), 2), (dict(scale=1e-60), 2),
    (dict(tokens=1 << 10, heads=1 << 20, width=1 << 24), 1), (dict(workspace_bytes=64), 4), (dict(workspace=None), 4), (dict(workspace=ctypes.c_void_p(0x10008)), 4),
    (dict(tokens=0, q=None, out=None, workspace=None, workspace_bytes=0), 0),
], ids=str)
def test_attention_validation(fp8lin, change, code):
    assert attention(fp8lin.lib(), record(fp8lin), **change) == code


def test_attention_null_cache_and_head_dims(fp8lin):
    L = fp8lin.lib()
    assert attention(L, None) == 2
    for dim in (32, 96, 192, 512):
        wide = record(fp8lin, head_dim=dim, k_slot=2 * dim, v_slot=2 * dim, k_head=dim, v_head=dim)
        assert attention(L, wide) == 3


def test_append_validation(fp8lin):
    L, rec = fp8lin.lib(), record(fp8lin)
    call = L.fp8lin_paged_append
    assert call(None, P, 128, 64, P, 128, 64, P, 3, None) == 2
    assert call(ctypes.byref(rec), None, 128, 64, P, 128, 64, P, 3, None) == 2
    assert call(ctypes.byref(rec), P, 128, 64, P, 128, 64, None, 3, None) == 2
    assert call(ctypes.byref(rec), P, 128, 64, P, 128, 64, P, -1, None) == 1
    assert call(ctypes.byref(rec), None, 128, 64, None, 128, 64, None, 0, None) == 0  # no tokens: no-op
    odd = record(fp8lin, head_dim=60, k_slot=128, v_slot=128)
    assert call(ctypes.byref(odd), P, 128, 64, P, 128, 64, P, 3, None) == 3


@pytest.mark.parametrize("at,value,code", [
    (0, None, 2), (1, None, 2), (2, None, 2), (4, None, 2), (11, None, 2), (12, None, 2), (13, None, 2), (14, None, 2), (15, None, 2),
    (17, None, 2), (3, 3, 1), (16, 3, 1), (5, -1, 1), (7, 0, 1), (7, 8193, 1), (8, 0, 1), (8, 1 << 27, 1), (9, 17, 1), (9, 8, 1),
    (10, -1, 1), 
])
def test_layout_validation(fp8lin, at, value, code):
    Q = ctypes.c_void_p(0x20000)
    args = [P, P, P, 8, P, 10, None, 3, 8, 16, 4, P, P, P, P, Q, 8, P, P, 1 << 20, None]
    args[at] = value
    assert fp8lin.lib().fp8lin_paged_layout(*args) == code


def test_layout_in_place(fp8lin):
    args = [P, P, P, 8, P, 10, None, 3, 8, 16, 4, P, P, P, P, P, 9, P, P, 1 << 20, None]
    call = fp8lin.lib().fp8lin_paged_layout
    assert call(*args) == 2  # another stride
    args[16] = 8
    assert call(*args[:18], None, 0, None) == 4 and call(*args[:18], P, 20, None) == 4


@pytest.mark.parametrize("at,value,code", [
    (0, None, 2), (6, None, 2), (7, None, 2), (8, None, 2), (13, None, 2), (14, None, 2), (2, 99, 1), (4, 99, 1), (5, -1, 1), (10, 0, 1),
    (10, 8193, 1), (11, -1, 1), (12, 0, 1), (12, 1 << 31, 1), (15, None, 4), (16, 8, 4),
])
def test_verify_validation(fp8lin, at, value, code):
    args = [P, 0, 100, P, 100, 5, P, P, P, None, 2, 7, 100, P, P, P, 1 << 30, None]
    args[at] = value
    assert fp8lin.lib().fp8lin_verify_drafts(*args) == code


def test_workspace_sizes(fp8lin):
    L = fp8lin.lib()
    assert L.fp8lin_paged_attention_workspace_bytes(12, 2, 256, 1) < L.fp8lin_paged_attention_workspace_bytes(12, 2, 256, 1000)
    assert L.fp8lin_paged_attention_workspace_bytes(12, 5, 256, 1) == 0
    assert L.fp8lin_paged_attention_workspace_bytes(0, 1, 256, 1) == 0
    sizes = L.fp8lin_paged_layout_workspace_bytes
    assert sizes(0, 1) == 0 and sizes(7, 1) > 0 and sizes(7, 0) == 0 and sizes(3000, 0) > 0
    assert L.fp8lin_verify_drafts_workspace_bytes(3, 10, 1000) > 0
    assert L.fp8lin_verify_drafts_workspace_bytes(3, 10, 0) == 0 and L.fp8lin_verify_drafts_workspace_bytes(0, 10, 10) == 0


def test_python_refuses_host_tensors(fp8lin):
    i32 = torch.zeros(3, dtype=torch.int32)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    x = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: fp8lin.paged_layout(i32, i32, torch.zeros(3, 4, dtype=torch.int32), i32, 5, 16),
                 lambda: fp8lin.paged_append(x, x, torch.zeros(5, dtype=torch.int64), cache, cache),
                 lambda: fp8lin.paged_attention(x, cache, cache, torch.zeros(3, 4, dtype=torch.int32), i32, i32),
                 lambda: fp8lin.verify_drafts(torch.zeros(5, 9), torch.zeros(5, dtype=torch.int64), torch.zeros(5), i32)):
        with pytest.raises(fp8lin.Fp8linError):
            call()
