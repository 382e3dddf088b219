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


def test_sizes_at_the_end_of_32_bits():
    """Loops of the kernels would step past it."""
    L = _lib()
    most, large = (1 << 31) - 1, -4
    table = dict(block_table=PTR, num_held=PTR, free_pages=PTR, num_free=PTR, workspace=PTR, free_capacity=4)
    fork = _runner("msa_pages_fork", L.MsaPagesForkArgs, dict(table, kv_len=PTR, parents=PTR, children=PTR, shares=PTR, count=1, num_pages=4, page_size=16, batch=2,
                                                              table_width=8, table_stride=most))
    free = _runner("msa_pages_free", L.MsaPagesFreeArgs, dict(table, kv_len=PTR, table_stride=8, table_width=0, page_size=16, num_pages=4, batch=2))
    compact = _runner("msa_pages_compact", L.MsaPagesCompactArgs, dict(table, src=PTR, dst=PTR, num_moved=PTR, num_pages=4, page_size=1, batch=2, table_width=8,
                                                                       table_stride=most))
    for run, kw in [(fork, dict(table_width=most)), (fork, dict(table_width=most - 1000)), (free, dict(batch=most)), (free, dict(batch=most - 1000)),
                    (compact, dict(num_pages=most)), (compact, dict(num_pages=most - 1000)), (compact, dict(batch=most)), (compact, dict(table_width=most))]:
        assert run(**kw) == large, kw
