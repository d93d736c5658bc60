"""More of what the 8-bit paged cache's entry points refuse, without a GPU."""
from __future__ import annotations

P = 0x1000  # a fake non-null, aligned address; never dereferenced


def test_reserve_refuses_more_columns_than_it_can_count(pkg):
    """Its requests' columns are numbered in 32 bits."""
    lib, n, width = pkg.load(), 1 << 20, 1 << 10
    ws = pkg.kv8_pages_workspace(10, n)
    for requests, w in ((n, width + 1), (1 << 11, (1 << 19) + 1)):
        assert lib.gptoss_kv8_reserve(None, requests, P, P, n, P, P, w, 10, P, P, P, ws, 0) == pkg.ERR_UNSUPPORTED
