"""Calls whose grids no launch takes are refused as unsupported, before any HIP call (no GPU needed)."""
import ctypes

import pytest

import busfill as bf
from test_ops_abi import FAKE, cache, refused, route, rows


@pytest.mark.parametrize("T", [1 << 26, (1 << 31) - 1])
def test_route_of_too_many_rows(T):
    a = route(T=T)
    refused(lambda: bf.lib().bf_moe_route(ctypes.byref(a), None), f"T={T}", bf.ERR_UNSUPPORTED)


@pytest.mark.parametrize("name", ["bf_kv4_store", "bf_kv4_load"])
@pytest.mark.parametrize("dim,T", [(256, 1 << 29), (128, 1 << 30), (96, 1431655766)])
def test_store_and_load_of_too_many_tokens(name, dim, T):
    refused(rows(name, cache(head_dim=dim, kv_heads=1), T=T, ldk=256, ldv=256), f"T={T}", bf.ERR_UNSUPPORTED)
