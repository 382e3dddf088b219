"""What the operators on pages of a cache, and the attention call that merges its partials, refuse before anything touches a device."""
import ctypes

import pytest
import torch

BAD, UNSUPPORTED, TOO_LARGE = -1, -2, -4
PTR = 1 << 20                                                   # an address that no call gets to use


def _lib():
    from msa_for_sail import _lib
    return _lib


def _cache(**kw):
    L = _lib()
    return L.MsaPageCache(**{**dict(base=PTR, stride_page=4096, stride_part=1024, parts=4, part_bytes=1024, token_bytes=64), **kw})


def _runner(name, struct, ok):
    L = _lib()
    fn = getattr(L.lib, name)

    def run(**kw):
        cache = kw.pop("cache", None)
        args = {**ok, **kw}
        if cache is not None:
            args.update(caches=ctypes.addressof(cache), num_caches=1)
        return fn(ctypes.byref(struct(**args)), None)
    assert fn(None, None) == BAD
    return run


BAD_CACHES = [dict(base=0), dict(parts=0), dict(part_bytes=0), dict(part_bytes=-1), dict(token_bytes=-2), dict(token_bytes=65)]


def test_copy_arguments():
    L = _lib()
    run = _runner("msa_pages_copy", L.MsaPagesCopyArgs, dict(src=PTR, dst=PTR, count=0, num_pages=4, page_size=16))
    assert run() == 0 and run(cache=_cache()) == 0 and run(src=0, dst=0) == 0               # no entries: nothing to launch
    assert run(count=5) == 0                                                                # nor without caches
    for kw in [dict(count=-1), dict(num_caches=-1), dict(num_caches=1), dict(num_pages=-1), dict(page_size=0), dict(count=1, src=0, cache=_cache()),
               dict(count=1, dst=0, cache=_cache())] + [dict(cache=_cache(**c)) for c in BAD_CACHES]:
        assert run(**kw) == BAD, kw
    assert run(cache=_cache(parts=(1 << 31) - 1, part_bytes=1 << 20, token_bytes=0)) == TOO_LARGE


def test_fork_arguments():
    L = _lib()
    assert L.lib.msa_pages_fork_workspace_bytes(-1, 0) == BAD and L.lib.msa_pages_fork_workspace_bytes(0, -1) == BAD
    assert L.lib.msa_pages_fork_workspace_bytes(3, 2) == 4 * (3 + 14) and L.lib.msa_pages_fork_workspace_bytes((1 << 31) - 1, (1 << 31) - 1) > 1 << 35
    ok = dict(block_table=PTR, num_held=PTR, kv_len=PTR, parents=PTR, children=PTR, free_pages=PTR, num_free=PTR, shares=PTR, num_missing=PTR, workspace=PTR,
              table_stride=8, count=2, num_pages=4, page_size=16, batch=2, table_width=8, free_capacity=4)
    run = _runner("msa_pages_fork", L.MsaPagesForkArgs, ok)
    for kw in [dict(count=-1), dict(batch=-1), dict(table_width=-1), dict(table_stride=7), dict(free_capacity=-1), dict(page_size=0), dict(num_pages=-1),
               dict(num_caches=1), dict(num_free=0), dict(workspace=0), dict(parents=0), dict(children=0), dict(num_held=0), dict(kv_len=0),
               dict(block_table=0), dict(free_pages=0), dict(shares=0)] + [dict(cache=_cache(**c)) for c in BAD_CACHES]:
        assert run(**kw) == BAD, kw
    assert run(count=(1 << 24) + 1) == TOO_LARGE


def test_free_arguments():
    L = _lib()
    assert L.lib.msa_pages_free_workspace_bytes(-1, 0) == BAD and L.lib.msa_pages_free_workspace_bytes(0, -1) == BAD
    assert L.lib.msa_pages_free_workspace_bytes(0, 0) > 0
    ok = dict(block_table=PTR, num_held=PTR, kv_len=PTR, free_pages=PTR, num_free=PTR, workspace=PTR, table_stride=8, batch=2, table_width=8, page_size=16,
              free_capacity=4, num_pages=4, window=3, sink_tokens=1)
    run = _runner("msa_pages_free", L.MsaPagesFreeArgs, ok)
    for kw in [dict(batch=-1), dict(table_width=-1), dict(table_stride=7), dict(page_size=0), dict(free_capacity=-1), dict(num_pages=-1), dict(window=-1),
               dict(window=0), dict(sink_tokens=-1), dict(num_free=0), dict(workspace=0), dict(free_pages=0), dict(num_held=0), dict(kv_len=0),
               dict(block_table=0)]:
        assert run(**kw) == BAD, kw
    assert run(batch=1 << 20, table_width=1 << 12, table_stride=1 << 12) == TOO_LARGE


def test_compact_arguments():
    L = _lib()
    assert L.lib.msa_pages_compact_workspace_bytes(-1) == BAD and L.lib.msa_pages_compact_workspace_bytes(0) > 0
    ok = dict(block_table=PTR, num_held=PTR, free_pages=PTR, num_free=PTR, src=PTR, dst=PTR, num_moved=PTR, workspace=PTR, table_stride=8, num_pages=4,
              page_size=1, batch=2, table_width=8, free_capacity=4)
    run = _runner("msa_pages_compact", L.MsaPagesCompactArgs, ok)
    for kw in [dict(batch=-1), dict(table_width=-1), dict(table_stride=7), dict(free_capacity=-1), dict(page_size=0), dict(num_pages=-1), dict(num_caches=1),
               dict(num_free=0), dict(workspace=0), dict(num_moved=0), dict(free_pages=0), dict(src=0), dict(dst=0), dict(num_held=0),
               dict(block_table=0)] + [dict(cache=_cache(**c)) for c in BAD_CACHES[:5]]:
        assert run(**kw) == BAD, kw


def test_no_cpu_path():
    import msa_for_sail as msa
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    one = i(0)
    for call in [lambda: msa.kv_pages_copy(torch.zeros(4, 8), one, one), lambda: msa.kv_pages_copy([], one, one),
                 lambda: msa.kv_pages_fork(table, i(0, 0), i(0, 0), one, one, i(1, 2), one, i(0, 0, 0, 0)),
                 lambda: msa.kv_pages_free(table, i(0, 0), i(0, 0), i(1, 2), one),
                 lambda: msa.kv_pages_compact(table, i(0, 0), i(1, 2), one, num_pages=4)]:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_attention_with_partials_of_its_own_call():
    L = _lib()
    ok = dict(q=PTR, k=PTR, v=PTR, out=PTR, partial_o=PTR, partial_lse=PTR, qo_start=PTR, kv_len=PTR, qo_offset=PTR, kv_page_indptr=PTR, kv_indices=PTR, work=PTR,
              q_stride_tok=1024, q_stride_head=128, k_stride_page=32768, k_stride_head=16384, k_stride_tok=128, v_stride_page=32768, v_stride_head=16384,
              v_stride_tok=128, out_stride_tok=1024, out_stride_head=128, kv_extent=4, total_q=0, num_qo_heads=8, num_kv_heads=2, batch=1, num_work=0,
              block_m=16, pack=4, page_size=128, num_splits=2, decode_rows=4, q_dtype=L.MSA_DT_BF16, kv_dtype=L.MSA_DT_BF16, flags=L.FLAG_OUT_O, sm_scale=1,
              out_scale=1, window=100, sink_tokens=4)
    run = lambda dtype=L.MSA_DT_BF16, **kw: L.lib.msa_fmha_fwd_merged(ctypes.byref(L.MsaFmhaParams(**{**ok, **kw})), None, dtype, None)
    assert run() == 0 and run(L.MSA_DT_F32) == 0 and run(window=0, sink_tokens=0) == 0       # no rows: nothing to launch
    assert L.lib.msa_fmha_fwd_merged(None, None, L.MSA_DT_BF16, None) == BAD
    for kw in [dict(partial_o=0), dict(partial_lse=0), dict(out=0), dict(num_splits=0), dict(q=0), dict(window=-1), dict(q_stride_tok=1028), dict(total_q=-1)]:
        assert run(**kw) == BAD, kw
    assert run(L.MSA_DT_E4M3) == UNSUPPORTED
