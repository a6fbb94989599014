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
