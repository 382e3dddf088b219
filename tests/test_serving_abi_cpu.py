"""What the serving operators refuse before anything touches a device, and the frequencies of a rope plan."""
import ctypes
import math
from fractions import Fraction

import pytest
import torch

BAD, UNSUPPORTED, TOO_LARGE = -1, -2, -4
PTR = 1 << 20                                                   # a multiple of 16 that no call gets to use


def _lib():
    from msa_for_sail import _lib
    return _lib


def _rope_args(**kw):
    L = _lib()
    a = L.MsaNormRopeArgs(q=PTR, k=PTR, v=PTR, q_out=PTR, k_cache=PTR, v_cache=PTR, slot_map=PTR, positions=PTR, turns=PTR, axis=PTR,
                          q_stride_tok=1024, q_stride_head=128, k_stride_tok=256, k_stride_head=128, v_stride_tok=256, v_stride_head=128,
                          q_out_stride_tok=1024, q_out_stride_head=128, k_cache_stride_page=18432, k_cache_stride_head=9216, v_cache_stride_page=18432,
                          v_cache_stride_head=9216, tokens=0, num_qo_heads=8, num_kv_heads=2, rotary=64, norm=1, weight_dtype=L.MSA_DT_F32,
                          q_out_dtype=L.MSA_DT_BF16, cache_dtype=L.MSA_DT_KV4, page_size=128, num_pages=4, eps=1e-6, q_scale=1, k_scale=1, v_scale=1)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


def test_norm_rope_arguments():
    L = _lib()
    run = lambda **kw: L.lib.msa_norm_rope(ctypes.byref(_rope_args(**kw)), None)
    assert run() == 0 and L.lib.msa_norm_rope(None, None) == BAD            # no tokens: nothing to launch
    for kw in [dict(tokens=-1), dict(q=0, k=0, v=0), dict(q_out=0), dict(q=PTR + 2), dict(q_stride_tok=1028), dict(k_stride_head=4), dict(v_cache=0),
               dict(slot_map=0), dict(page_size=0), dict(num_pages=-1), dict(k_cache=PTR + 8), dict(k_cache_stride_page=8), dict(k=0), dict(v=0),
               dict(positions=0), dict(turns=0), dict(axis=0), dict(num_qo_heads=0), dict(num_kv_heads=0), dict(q_weight=PTR + 4), dict(q_weight_stride=4)]:
        assert run(**kw) == BAD, kw
    for kw in [dict(rotary=16), dict(rotary=160), dict(rotary=-32), dict(page_size=64), dict(cache_dtype=9), dict(q_out_dtype=L.MSA_DT_F32),
               dict(weight_dtype=L.MSA_DT_E4M3)]:
        assert run(**kw) == UNSUPPORTED, kw
    bf16 = dict(cache_dtype=L.MSA_DT_BF16, k_cache_stride_tok=128, v_cache_stride_tok=128, page_size=16)
    assert run(**bf16) == 0
    assert run(**{**bf16, "v_cache_stride_tok": 130}) == BAD


def test_kv4_read_arguments():
    L = _lib()
    ok = dict(cache=PTR, out=PTR, slot_map=PTR, stride_page=18432, stride_head=9216, rows=0, num_kv_heads=2, num_pages=3)
    run = lambda **kw: L.lib.msa_kv4_read(ctypes.byref(L.MsaKv4ReadArgs(**{**ok, **kw})), None)
    assert run() == 0 and run(whole_pages=1) == 0
    for kw in [dict(cache=0), dict(out=0), dict(slot_map=0), dict(rows=-1), dict(num_kv_heads=0), dict(num_pages=-1), dict(cache=PTR + 8), dict(out=PTR + 8),
               dict(stride_page=24), dict(stride_head=72)]:
        assert run(**kw) == BAD, kw
    assert run(num_kv_heads=70000) == TOO_LARGE


def test_page_table_arguments():
    L = _lib()
    assert L.lib.msa_page_tables(None, None) == BAD and L.lib.msa_page_tables_workspace_bytes(-1) == BAD
    assert L.lib.msa_page_tables_workspace_bytes(0) > 0
    ok = dict(qo_len=PTR, kv_len=PTR, block_table=PTR, kv_indices=PTR, kv_page_indptr=PTR, slot_map=PTR, positions=PTR, workspace=PTR, table_stride=4, batch=2,
              table_width=4, page_size=128, max_total_q=2, max_total_pages=8)
    run = lambda **kw: L.lib.msa_page_tables(ctypes.byref(L.MsaPageTablesArgs(**{**ok, **kw})), None)
    for kw in [dict(qo_len=0), dict(kv_len=0), dict(block_table=0), dict(kv_indices=0), dict(kv_page_indptr=0), dict(slot_map=0), dict(positions=0),
               dict(workspace=0), dict(table_stride=3), dict(batch=-1), dict(table_width=-1), dict(page_size=0), dict(max_total_q=-1), dict(max_total_pages=-1),
               dict(num_held=PTR), dict(free_pages=PTR), dict(num_free=PTR), dict(num_held_out=PTR), dict(num_free_out=PTR), dict(free_capacity=-1),
               dict(num_held=PTR, num_free=PTR, free_capacity=3)]:
        assert run(**kw) == BAD, kw


def test_merge_of_many_splits_arguments():
    L = _lib()
    ok = dict(po=PTR, pl=PTR, spr=None, out=PTR, dt=L.MSA_DT_BF16, lse=None, S=2, T=0, H=4, st=512, sh=128)
    run = lambda **kw: (lambda a: L.lib.msa_lse_merge_many(a["po"], a["pl"], a["spr"], a["out"], a["dt"], a["lse"], a["S"], a["T"], a["H"], a["st"], a["sh"],
                                                             1.0, None))({**ok, **kw})
    assert run() == 0
    for kw in (dict(po=None), dict(pl=None), dict(out=None), dict(S=0), dict(T=-1), dict(H=0), dict(T=1, po=PTR + 8), dict(T=1, out=PTR + 4),
               dict(T=1, st=514), dict(T=1, sh=130)):
        assert run(**kw) == BAD, kw
    assert run(dt=L.MSA_DT_E4M3) == UNSUPPORTED


def test_attention_arguments_of_a_4_bit_cache():
    L = _lib()
    ok = dict(q=PTR, k=PTR, v=PTR, out=PTR, qo_start=PTR, kv_len=PTR, qo_offset=PTR, kv_page_indptr=PTR, kv_indices=PTR, work=PTR, q_stride_tok=1024,
              q_stride_head=128, k_stride_page=18432, k_stride_head=9216, v_stride_page=18432, v_stride_head=9216, out_stride_tok=1024, out_stride_head=128,
              kv_extent=4, total_q=0, num_qo_heads=8, num_kv_heads=2, batch=1, num_work=0, block_m=16, pack=4, page_size=128, num_splits=1, decode_rows=4,
              q_dtype=L.MSA_DT_BF16, kv_dtype=L.MSA_DT_KV4, flags=L.FLAG_OUT_O, sm_scale=1, out_scale=1)
    run = lambda **kw: L.lib.msa_fmha_fwd(ctypes.byref(L.MsaFmhaParams(**{**ok, **kw})), None)
    assert run() == 0
    for kw in [dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(qo_start=0), dict(kv_len=0), dict(qo_offset=0), dict(kv_page_indptr=0), dict(kv_indices=0),
               dict(flags=0), dict(num_work=1, work=0), dict(num_splits=2), dict(partial_o=PTR), dict(num_kv_heads=3), dict(pack=3), dict(k=PTR + 8),
               dict(k_stride_page=9224), dict(v_stride_head=72), dict(q_stride_tok=1020), dict(out_stride_head=4), dict(total_q=1, kv_extent=0),
               dict(pack=4, block_m=16, num_qo_heads=64, num_kv_heads=1, decode_rows=0, flags=L.FLAG_OUT_O | L.FLAG_SPARSE),
               dict(flags=L.FLAG_OUT_O | L.FLAG_SPARSE)]:
        assert run(**kw) == BAD, kw
    for kw in [dict(page_size=64), dict(page_size=0), dict(flags=L.FLAG_OUT_SCORE), dict(flags=L.FLAG_OUT_O | L.FLAG_OUT_SCORE), dict(block_m=256),
               dict(q_dtype=L.MSA_DT_F32)]:
        assert run(**kw) == UNSUPPORTED, kw
    # the entry point with the library's own scratch has no 4-bit form
    p = L.MsaFmhaParams(**{**ok, "kv_start": PTR})
    assert L.lib.msa_fmha_fwd_split_static(ctypes.byref(p), None, None) == UNSUPPORTED


@pytest.mark.parametrize("base,rotary", [(10000.0, 128), (5e6, 64), (1e3, 32)])
def test_rope_plan_frequencies(base, rotary):
    """turns / 2^64 is the frequency in turns: the angle of any position is off by less than 2^31 x 2^-53 turns of the frequency's own
    rounding."""
    import msa_for_sail as msa
    plan = msa.rope_plan(rotary, base=base, device="cpu")
    assert plan["turns"].dtype == torch.int64 and plan["axis"].tolist() == [0] * (rotary // 2)
    for i, t in enumerate(plan["turns"].tolist()):
        f = base ** (-2 * i / rotary)
        exact = Fraction(f) / (2 * Fraction(math.pi))
        assert abs(Fraction(t % (1 << 64), 1 << 64) - exact) < Fraction(1, 1 << 52)
    plan = msa.rope_plan(rotary, inv_freq=[-0.5] * (rotary // 2), sections=[3, rotary // 2 - 3], device="cpu")
    assert plan["turns"][0] < 0 and plan["axis"].tolist() == [0] * 3 + [1] * (rotary // 2 - 3) and plan["axes"] == 2


def test_rope_plan_refusals():
    import msa_for_sail as msa
    for kw in [dict(rotary_dim=16), dict(rotary_dim=0), dict(rotary_dim=160), dict(rotary_dim=64, inv_freq=[1.0]), dict(rotary_dim=64, sections=[1, 2]),
               dict(rotary_dim=64, sections=[-1, 33]), dict(rotary_dim=32, inv_freq=[float("inf")] * 16)]:
        with pytest.raises(ValueError):
            msa.rope_plan(device="cpu", **kw)


def test_no_cpu_path():
    import msa_for_sail as msa
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    c = torch.zeros(1, 1, 128, 72, dtype=torch.uint8)
    for f in [lambda: msa.paged_kv_tables(i, i, i[None], max_total_q=1), lambda: msa.qk_norm_rope(x, x, None, None),
              lambda: msa.kv_cache_append(x, x, c, c, i), lambda: msa.kv4_read(c, i), lambda: msa.fmha_sail(x, c, c, (False, 0, 1, {}, None), kv_indices=i)]:
        with pytest.raises(RuntimeError):
            f()
