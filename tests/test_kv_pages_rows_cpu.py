"""What giving back pages refuses of caches and counts, before anything touches a device."""
import ctypes

from test_kv_pages_cpu import BAD, BAD_CACHES, PTR, _cache, _lib, _runner


def test_free_with_caches():
    L = _lib()
    ok = dict(block_table=PTR, num_held=PTR, kv_len=PTR, free_pages=PTR, num_free=PTR, shares=PTR, workspace=PTR, table_stride=8, batch=2, table_width=8,
              page_size=16, free_capacity=4, num_pages=4)
    run = _runner("msa_pages_free", L.MsaPagesFreeArgs, ok)
    for kw in [dict(num_caches=-1), dict(num_caches=1), dict(cache=_cache(), shares=0), dict(num_shared=PTR, shares=0)] + [dict(cache=_cache(**c)) for c in BAD_CACHES]:
        assert run(**kw) == BAD, kw


def test_workspace_of_the_rows():
    size = _lib().lib.msa_pages_free_workspace_bytes
    assert size(1000, 5) >= 4 * (1000 + 1 + 5 * 1000 + 1) and size(1, 1 << 20) >= 4 * ((1 << 10) + 1 + 5 + 1)
    assert ctypes.c_int64(size((1 << 31) - 1, (1 << 31) - 1)).value > 1 << 50
