"""Sizes past what the paged-cache kernels count in 32 bits, without a GPU: refused before anything is launched."""
import ctypes

import pytest

from test_paged import P, record


@pytest.mark.parametrize("tokens,kv_heads,head_dim", [
    (1, 1 << 20, 4096), (1, (1 << 31) - 1, 64), (1 << 30, 1 << 30, 4096), ((1 << 31) - 1, 1 << 19, 4096 - 16), (1, 1 << 23, 256),
    (1 << 24, 8, 256), ((1 << 31) - 1, 1, 64), ((1 << 29) - 1, 1, 64),
])
def test_append_of_too_many_values(fp8lin, tokens, kv_heads, head_dim):
    """Head strides of 0 (expanded caches and inputs) reach any number of heads."""
    rec = record(fp8lin, kv_heads=kv_heads, head_dim=head_dim, k_head=0, v_head=0, k_slot=head_dim, v_slot=head_dim, k_page=0, v_page=0)
    assert fp8lin.lib().fp8lin_paged_append(ctypes.byref(rec), P, 0, 0, P, 0, 0, P, tokens, None) == 1


@pytest.mark.parametrize("rows", [1 << 24, (1 << 31) - 1])
def test_verify_of_too_many_rows(fp8lin, rows):
    L = fp8lin.lib()
    A = 1 << 50  # apart, whatever their sizes
    at = [ctypes.c_void_p(i * A) for i in range(1, 8)]
    assert L.fp8lin_verify_drafts(at[0], 0, 100, None, 0, 0, at[1], at[2], at[3], None, 2, rows, 100, at[4], at[5], at[6], 1 << 45, None) == 1
    assert L.fp8lin_verify_drafts_workspace_bytes(2, rows, 100) == 0
    assert L.fp8lin_verify_drafts_workspace_bytes(2, (1 << 24) - 1, 100) > 0
