"""An attention call that merges its partials refuses what its merge would, before anything is launched."""
import ctypes

import pytest

BAD, UNSUPPORTED, TOO_LARGE = -1, -2, -4
PTR = 1 << 20


def _run(dtype, **kw):
    from msa_for_sail import _lib as L
    ok = dict(q=PTR, k=PTR, v=PTR, out=PTR, partial_o=PTR, partial_lse=PTR, qo_start=PTR, kv_len=PTR, qo_offset=PTR, kv_page_indptr=PTR, kv_indices=PTR, work=PTR,
              q_stride_tok=1024, q_stride_head=128, k_stride_page=32768, k_stride_head=16384, k_stride_tok=128, v_stride_page=32768, v_stride_head=16384,
              v_stride_tok=128, out_stride_tok=1024, out_stride_head=128, kv_extent=4, total_q=0, num_qo_heads=8, num_kv_heads=2, batch=1, num_work=0,
              block_m=16, pack=4, page_size=128, num_splits=2, decode_rows=4, q_dtype=L.MSA_DT_BF16, kv_dtype=L.MSA_DT_BF16, flags=L.FLAG_OUT_O, sm_scale=1,
              out_scale=1, window=100, sink_tokens=4)
    return L.lib.msa_fmha_fwd_merged(ctypes.byref(L.MsaFmhaParams(**{**ok, **kw})), None, getattr(L, dtype), None)


@pytest.mark.parametrize("dtype,size", [("MSA_DT_BF16", 2), ("MSA_DT_F32", 4)])
def test_rows_of_the_result(dtype, size):
    step = 16 // size
    assert _run(dtype) == 0 and _run(dtype, out=PTR + 16, out_stride_tok=1024 + step, out_stride_head=128 + step) == 0
    for kw in [dict(out=PTR + 8), dict(out=PTR + size), dict(out_stride_tok=1024 + step // 2), dict(out_stride_head=128 + step // 2), dict(out_stride_head=129),
               dict(partial_o=PTR + 8)]:
        assert _run(dtype, **kw) == BAD, kw
    assert _run(dtype, total_q=1 << 28, num_work=1) == TOO_LARGE


def test_the_number_of_sms():
    assert _run("MSA_DT_BF16", num_sms=20) == 0 and _run("MSA_DT_BF16", num_sms=-1) == BAD
