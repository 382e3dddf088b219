"""Plans of windowed attention: the tiles of each work item, and what is refused."""
import ctypes
import random

import numpy as np
import pytest
import torch

BAD, UNSUPPORTED = -1, -2
PTR = 1 << 20


def _lib():
    from msa_for_sail import _lib
    return _lib


def _plan(ql, kl, off, hq, hk, block_m, pack, splits, window, sinks):
    L = _lib()
    a_q, a_k, a_o = (np.asarray(v, np.int32) for v in (ql, kl, off))
    host = np.empty((1 << 16, 8), np.int32)
    spr = np.zeros(max(1, sum(ql)), np.int32)
    most = ctypes.c_int32()
    args = L.MsaPlanArgs(a_q.ctypes.data, a_k.ctypes.data, a_o.ctypes.data, len(ql), hq, hk, block_m, pack, splits, 148, 0, window, sinks)
    n = L.check(L.lib.msa_plan_dense(ctypes.byref(args), host.ctypes.data, len(host), spr.ctypes.data, ctypes.byref(most)), "plan")
    return host[:n]


@pytest.mark.parametrize("block_m,pack", [(16, 4), (64, 4), (128, 1), (256, 1)])
@pytest.mark.parametrize("splits", [-128, 1, 3])
def test_tiles_of_an_item_are_those_that_its_rows_see(block_m, pack, splits):
    rng = random.Random(block_m + splits)
    for _ in range(60):
        b = rng.randint(1, 4)
        ql = [rng.choice([0, 1, 3, rng.randint(1, 600)]) for _ in range(b)]
        kl = [rng.choice([0, 1, 128, rng.randint(0, 5000)]) for _ in range(b)]
        off = [rng.choice([k - q, k - q, 0, rng.randint(-700, 6000)]) for q, k in zip(ql, kl)]
        window, sinks = rng.choice([1, 2, 127, 128, 129, 1000, (1 << 31) - 1]), rng.choice([0, 1, 128, 129, 700, (1 << 31) - 1])
        items = _plan(ql, kl, off, 4 * pack, 4, block_m, pack, splits, window, sinks)
        seen = {}
        for batch, head0, row0, tb, te, split, rows, skip in items.tolist():
            assert skip >= 0 and 0 <= tb <= te
            first = -(-sinks // 128)
            tiles = seen.setdefault((batch, head0, row0, rows), [])
            tiles += [t if t < first else t + skip for t in range(tb, te)]
        groups = 4 * pack // pack
        step = block_m // pack * pack
        assert len(seen) == sum(-(-n * pack // step) for n in ql) * groups
        for (batch, _, row0, rows), tiles in seen.items():
            lo, hi = row0 // pack + off[batch], (row0 + rows - 1) // pack + off[batch]
            j = np.arange(kl[batch])
            see = (j <= hi) & ((j > lo - window) | (j < sinks))
            want = set((np.nonzero(see)[0] // 128).tolist())
            assert sorted(tiles) == sorted(set(tiles))
            assert want <= set(tiles)
            # none but tiles that some row sees, and the last one where the keys between sinks and window are nobody's
            assert len(tiles) <= len(want) + (0 if rows == 1 else 1)


def _refuse(**kw):
    import msa_for_sail as msa
    i = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        msa.fmha_sail_plan(i, i, 8, num_kv_heads=2, device="cuda:0", **kw)


@pytest.mark.parametrize("kw", [
    dict(window_size=0), dict(window_size=-2), dict(window_size=1 << 31), dict(num_sink_tokens=1), dict(window_size=5, num_sink_tokens=-1),
    dict(window_size=5, num_sink_tokens=1 << 31), dict(window_size=5, causal=False), dict(window_size=5, output_maxscore=True, page_size=128),
    dict(window_size=5, kv_block_num=16, page_size=128), dict(window_size=5, use_kv4_cache=True, page_size=128)])
def test_plans_that_are_refused(kw):
    _refuse(**kw)


def test_arguments_of_the_library():
    L = _lib()
    ok = dict(q=PTR, k=PTR, v=PTR, out=PTR, qo_start=PTR, kv_len=PTR, qo_offset=PTR, kv_page_indptr=PTR, kv_indices=PTR, work=PTR, q_stride_tok=1024,
              q_stride_head=128, k_stride_page=32768, k_stride_head=16384, k_stride_tok=128, v_stride_page=32768, v_stride_head=16384, v_stride_tok=128,
              out_stride_tok=1024, out_stride_head=128, kv_extent=4, total_q=0, num_qo_heads=8, num_kv_heads=2, batch=1, num_work=0, block_m=16, pack=4,
              page_size=128, num_splits=1, decode_rows=4, q_dtype=L.MSA_DT_BF16, kv_dtype=L.MSA_DT_BF16, flags=L.FLAG_OUT_O, sm_scale=1, out_scale=1,
              window=100, sink_tokens=4)
    run = lambda **kw: L.lib.msa_fmha_fwd(ctypes.byref(L.MsaFmhaParams(**{**ok, **kw})), None)
    assert run() == 0 and run(sink_tokens=0) == 0
    for kw in [dict(window=-1), dict(sink_tokens=-1), dict(window=0, sink_tokens=1)]:
        assert run(**kw) == BAD, kw
    for kw in [dict(max_score=PTR, max_k_tiles=4, flags=L.FLAG_OUT_O | L.FLAG_OUT_SCORE), dict(max_score=PTR, max_k_tiles=4, flags=L.FLAG_OUT_SCORE),
               dict(kv_block_indexes=PTR, token_batch=PTR, kv_block_num=4, flags=L.FLAG_OUT_O | L.FLAG_SPARSE), dict(kv_dtype=L.MSA_DT_KV4)]:
        assert run(**kw) == UNSUPPORTED, kw
    for kw in [dict(window=-1), dict(window=0, sink_tokens=1), dict(window=1, sink_tokens=-1)]:
        a = L.MsaPlanDeviceArgs(qo_len=PTR, kv_len=PTR, batch=0, num_qo_heads=8, num_kv_heads=2, block_m=16, pack=4, num_splits=1, row_tiles=1, **kw)
        assert L.lib.msa_plan_device(ctypes.byref(a), None) == BAD, kw
        with pytest.raises(RuntimeError):
            _plan([1], [1], [0], 8, 2, 16, 4, 1, kw.get("window", 0), kw.get("sink_tokens", 0))


def test_a_windowed_call_from_its_parameter_line():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "msa-for-sail_b200", "benchmarks", "run_msa.py")
    spec = importlib.util.spec_from_file_location("run_msa", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    for q, k, off, window, sinks in [(3, 500, 497, 100, 4), (200, 700, 500, 64, 30), (5, 5, 0, 3, 9), (4, 100, 300, 50, 2), (3, 10, -2, 4, 0), (2, 50, 0, 1, 0)]:
        cfg = m.parse_format(f"[MSA] --format=seqlen_q:[{q}],seqlen_k:[{k}],qo_offset:[{off}],num_qo_heads:4,kv_block_num:0,window_size:{window},num_sink_tokens:{sinks}.")
        assert cfg["window_size"] == window and m.parse_format(m.format_line(cfg)) == cfg
        place = np.arange(q)[:, None] + off
        j = np.arange(k)[None]
        see = (j <= place) & ((j > place - window) | (j < sinks))
        flops, nbytes = m.flops_and_bytes(cfg)
        assert flops == 4 * 512 * int(see.sum())
        # from the first query's window to the last query: one stretch of keys, and the sinks
        lo, hi = max(0, off - window + 1), max(0, min(k, q + off))
        assert nbytes == 2 * q * 4 * 128 * 2 + int(((j < hi) & ((j >= lo) | (j < sinks))).sum()) * 4 * 128 * 2 * 2
    assert "window_size" not in m.format_line(m.parse_format("--format=seqlen_q:[2],seqlen_k:[256],num_qo_heads:4"))
