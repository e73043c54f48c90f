"""Limits of the operators around the sparse attention that are checked without a GPU."""

import pytest

from flash_topk_attn_v2 import _lib


@pytest.mark.parametrize("B,H,Hk,N,D", [(1 << 30, 4096, 4096, 1 << 29, 64), (1 << 30, 1 << 20, 1 << 16, 1 << 20, 64),
                                        ((1 << 31) - 1, 1 << 20, 1 << 20, 1 << 20, 256), (1 << 28, 1 << 16, 1, 1 << 19, 16)])
def test_sizes_whose_products_wrap(B, H, Hk, N, D):
    """Sizes of no real tensor: refused, where a 64-bit product wrapped to zero was divided by."""
    L, z, x = _lib.lib(), _lib.i64arr((0, 0, 0)), 4096  # an address that nothing reads
    assert L.fta_window_attn_bwd_workspace_size(B, H, Hk, N, D, 3, 0, 4) == 0
    assert L.fta_cache_attn_workspace_size(B, H, Hk, min(N, 1 << 20), 10, D, 0, 3, 0) == 0
    assert L.fta_qk_norm_rope_bwd_workspace_size(B, H, Hk, N, D) == 0
    rc = L.fta_window_attn_fwd(x, z, x, z, x, z, 0, B, H, Hk, N, D, None, 3, 0, 4, 0.1, x, z, x, None)
    assert rc == _lib.FTA_ERR_UNSUPPORTED
    rc = L.fta_cache_attn(x, z, x, z, x, z, 0, B, H, Hk, min(N, 1 << 20), 10, D, x, None, z, None, z, 0, 3, 0, 0.1, x, z, x,
                          None, 0, None)
    assert rc == _lib.FTA_ERR_UNSUPPORTED
    rc = L.fta_qk_norm_rope(x, z, x, z, 0, B, H, Hk, N, D, None, None, 2, x, x, N, 16, None, 0, 1e-6, 0, x, z, x, z, None)
    assert rc == _lib.FTA_ERR_UNSUPPORTED
