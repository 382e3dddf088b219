"""Page tables that end before the lengths do (lengths on the device may outgrow a table of fixed size): the places behind the end are the
last page, in every kernel and on every cache.  A short table gives what a full one gives whose last places are that page, bit for bit."""
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
KEYS, PAGES, KEPT = 600, 5, 2


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(kind, g, P, hk, page):
    if kind == "kv4":
        return [ref.random_kv4(g, P, hk).to(DEV) for _ in range(2)]
    x = [torch.randn(P, hk, page, 128, generator=g).to(DEV) for _ in range(2)]
    return [t.to(torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn) for t in x]


def _plan(rows, hq, hk, page=128, kbn=-1, scores=False, splits=1, keys=KEYS, **kw):
    import msa_for_sail as msa
    ws = msa.allocate_graph_workspace(1, hq, num_kv_heads=hk, page_size=page, num_kv_splits=splits, kv_block_num=kbn, max_qo_len=rows)
    return msa.fmha_sail_plan(_i32([rows]), _i32([keys]), hq, num_kv_heads=hk, page_size=page, kv_block_num=kbn, num_kv_splits=splits, graph_safe=True,
                              output_maxscore=scores, max_total_q=rows, max_qo_len_override=rows, qo_len_uniform_override=True, max_kv_len_override=700,
                              qo_offset=_i32([keys - rows]), given_workspace=ws, **kw)


# rows, query heads, page, selected pages, scores, splits
CASES = {"decode": (1, 16, 128, -1, False, 2), "decode of 4 tokens": (4, 16, 128, -1, False, 1), "prompt": (200, 4, 128, -1, False, 1),
         "prompt in splits": (60, 4, 128, -1, False, 2), "pages of 64": (3, 16, 64, -1, False, 1), "scores of one row": (1, 2, 128, -1, True, 1),
         "scores of a prompt": (200, 4, 128, -1, True, 1), "scores of many rows": (8, 16, 128, -1, True, 1), "selected": (3, 16, 128, 3, False, 2)}


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "kv4"])
@pytest.mark.parametrize("case", list(CASES))
def test_a_short_table_reads_as_its_last_page(kind, case):
    import msa_for_sail as msa
    from msa_for_sail import api
    rows, hq, page, kbn, scores, splits = CASES[case]
    if kind == "kv4" and page != 128:
        pytest.skip("pages of a 4-bit cache have 128 tokens")
    hk = 2
    g = torch.Generator().manual_seed(11)
    pages = -(-KEYS // page)
    k, v = _cache(kind, g, pages + 3, hk, page)
    q = torch.randn(rows, hq, 128, generator=g).to(torch.bfloat16).to(DEV)
    table = torch.randperm(pages + 3, generator=g)[:pages].to(torch.int32).to(DEV)
    if kind == "e4m3" and rows > 128:
        q = q.to(torch.float8_e4m3fn)
    sel = dict(kv_block_indexes=_i32([0, 2, pages - 1]).expand(rows, hk, 3).contiguous()) if kbn > 0 else {}
    plan = _plan(rows, hq, hk, page, kbn, scores, splits, use_kv4_cache=kind == "kv4")
    full = table.clone()
    full[KEPT:] = table[KEPT - 1]
    kw = dict(output_o=False) if scores else {}
    run = lambda t: [x.clone() for x in msa.fmha_sail(q, k, v, plan, kv_indices=t, **kw, **sel) if x is not None]
    got = run(table[:KEPT].clone())
    api.last_status()                                           # (the build with bounds checks reports the places past the end)
    want = run(full)
    other = run(table)
    assert len(got) == len(want) == 1
    assert torch.equal(got[0], want[0]) and not torch.equal(want[0], other[0])


def test_a_short_table_of_a_plan_with_pages_first():
    """Sparse prefill page by page: a host-made plan, whose table is as long as its pages, or shorter where nobody selects the rest."""
    import msa_for_sail as msa
    g = torch.Generator().manual_seed(12)
    k, v = _cache("bf16", g, 9, 2, 128)
    q = torch.randn(300, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    plan = msa.fmha_sail_plan(torch.tensor([300]), torch.tensor([900]), 8, num_kv_heads=2, page_size=128, kv_block_num=4)
    assert plan[3]["sparse_tc_preferred"]
    table = _i32([3, 7, 1, 0, 8, 2, 4, 6])
    blocks = _i32([0, 1, 2, -1]).expand(300, 2, 4).contiguous()
    want = msa.fmha_sail(q, k, v, plan, kv_indices=table, kv_block_indexes=blocks)[0]
    assert torch.equal(msa.fmha_sail(q, k, v, plan, kv_indices=table[:3].clone(), kv_block_indexes=blocks)[0], want)
    last = _i32([3, 7, 7, 7, 7, 7, 7, 7])
    want = msa.fmha_sail(q, k, v, plan, kv_indices=last, kv_block_indexes=blocks)[0]
    assert torch.equal(msa.fmha_sail(q, k, v, plan, kv_indices=table[:2].clone(), kv_block_indexes=blocks)[0], want)


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "kv4"])
def test_tables_with_too_few_places_and_attention(kind):
    """paged_kv_tables counts the pages that its flat table has no place for; attention over such a table stays in the cache."""
    import msa_for_sail as msa
    g = torch.Generator().manual_seed(13)
    k, v = _cache(kind, g, 12, 2, 128)
    ql, kl = _i32([1, 200]), _i32([300, 700])
    block_table = torch.randperm(12, generator=g).view(2, 6).to(torch.int32).to(DEV)
    q = torch.randn(201, 8, 128, generator=g).to(torch.bfloat16).to(DEV)

    def run(places):
        tabs = msa.paged_kv_tables(ql, kl, block_table, max_total_q=201, max_total_pages=places)
        ws = msa.allocate_graph_workspace(2, 8, num_kv_heads=2, page_size=128, max_qo_len=200)
        plan = msa.fmha_sail_plan(ql, kl, 8, num_kv_heads=2, page_size=128, num_kv_splits=1, graph_safe=True, max_total_q=201, max_qo_len_override=200,
                                  qo_len_uniform_override=False, max_kv_len_override=700, qo_offset=_i32([-1, -1]), given_workspace=ws,
                                  use_kv4_cache=kind == "kv4")
        return msa.fmha_sail(q, k, v, plan, kv_indices=tabs["kv_indices"])[0].clone(), int(tabs["num_missing"])
    want, none = run(9)
    got, missing = run(4)
    assert none == 0 and missing == 5
    assert torch.equal(got[0], want[0]) and torch.isfinite(got.float()).all()


@pytest.mark.parametrize("kind", ["bf16", "kv4"])
@pytest.mark.parametrize("ql,hq,scores,splits", [([1, 1, 1, 1], 16, False, 1), ([1, 1, 1, 1], 16, False, 2), ([3, 4, 2, 3], 16, False, 1), ([2, 150, 200, 1], 4, False, 1),
                                                 ([20, 30, 25, 4], 4, False, 2), ([1, 1, 1, 1], 2, True, 1), ([40, 150, 3, 9], 4, True, 1)])
def test_tokens_past_the_rows_of_a_plan(kind, ql, hq, scores, splits):
    """Query lengths on the device may sum to more than max_total_q, as paged_kv_tables counts in num_missing: what is past it is in no sequence.
    The rows that there are get what they get from lengths that end there, and nothing around q, the result and the scores is touched."""
    import msa_for_sail as msa
    g = torch.Generator().manual_seed(14)
    hk, kl = 2, [300, 500, 260, 129]
    T = sum(ql[:2]) + (ql[2] + 1) // 2                          # ends inside the third sequence, or behind it
    cut = [min(n, max(0, T - sum(ql[:i]))) for i, n in enumerate(ql)]
    k, v = _cache(kind, g, 14, hk, 128)
    table = torch.randperm(14, generator=g)[:sum(-(-n // 128) for n in kl)].to(torch.int32).to(DEV)
    q = torch.randn(T + 512, hq, 128, generator=g).to(torch.bfloat16).to(DEV)
    off = _i32([a - b for a, b in zip(kl, ql)])
    tabs = msa.paged_kv_tables(_i32(ql), _i32(kl), torch.zeros(4, 4, dtype=torch.int32, device=DEV), max_total_q=T)
    assert int(tabs["num_missing"]) == sum(ql) - T

    def run(lens):
        ws = msa.allocate_graph_workspace(4, hq, num_kv_heads=hk, page_size=128, max_qo_len=max(ql), num_kv_splits=splits)
        plan = msa.fmha_sail_plan(_i32(lens), _i32(kl), hq, num_kv_heads=hk, page_size=128, num_kv_splits=splits, graph_safe=True, output_maxscore=scores,
                                  max_total_q=T, max_qo_len_override=max(ql), qo_len_uniform_override=False, max_kv_len_override=500, qo_offset=off,
                                  given_workspace=ws, use_kv4_cache=kind == "kv4")
        assert plan[3]["qo_segment_offsets"].tolist() == [min(T, sum(ql[:i])) for i in range(5)]
        if scores:
            ms = torch.full((hq + 1, plan[3]["max_k_tiles"], T), -float("inf"), device=DEV)
            msa.fmha_sail(q[:T], k, v, plan, kv_indices=table, output_o=False, max_score=ms[:hq])
            assert (ms[hq] == -float("inf")).all()
            return ms[:hq], None
        out, lse = torch.full((T + 512, hq, 128), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((T + 512, hq), 7.0, device=DEV)
        msa.fmha_sail(q[:T], k, v, plan, kv_indices=table, out=out[:T], lse=lse[:T])
        assert (out[T:] == 7).all() and (lse[T:] == 7).all()
        return out[:T], lse[:T]
    want, got = run(cut), run(ql)
    assert torch.equal(got[0], want[0]) and (scores or torch.equal(got[1], want[1]))
    assert scores or not (got[0] == 7).all(2).any()


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "kv4"])
@pytest.mark.parametrize("most,hq,scores,splits", [(1, 16, False, 1), (2, 16, False, 2), (3, 16, False, 1), (8, 32, False, 1), (2, 16, True, 1), (1, 2, True, 1)])
def test_more_tokens_than_a_plan_has_rows_for(kind, most, hq, scores, splits):
    """A sequence with more tokens than max_qo_len_override: as many as fill its row tiles are worked on, the rows of the rest stay as they were."""
    import msa_for_sail as msa
    g = torch.Generator().manual_seed(15)
    hk, kl, ql = 2, [300, 500], [40, 1]
    k, v = _cache(kind, g, 9, hk, 128)
    table = torch.randperm(9, generator=g)[:7].to(torch.int32).to(DEV)
    q = torch.randn(41, hq, 128, generator=g).to(torch.bfloat16).to(DEV)
    off = _i32([200, 499])

    def run(lens, q, most):
        T = q.shape[0]
        ws = msa.allocate_graph_workspace(2, hq, num_kv_heads=hk, page_size=128, max_qo_len=40, num_kv_splits=splits)
        plan = msa.fmha_sail_plan(_i32(lens), _i32(kl), hq, num_kv_heads=hk, page_size=128, num_kv_splits=splits, graph_safe=True, output_maxscore=scores,
                                  max_total_q=T, max_qo_len_override=most, qo_len_uniform_override=False, max_kv_len_override=500, qo_offset=off,
                                  given_workspace=ws, use_kv4_cache=kind == "kv4")
        if scores:
            ms = torch.full((hq, plan[3]["max_k_tiles"], T), 7.0, device=DEV)
            msa.fmha_sail(q, k, v, plan, kv_indices=table, output_o=False, max_score=ms)
            return ms.movedim(2, 0)
        out = torch.full((T, hq, 128), 7.0, dtype=torch.bfloat16, device=DEV)
        msa.fmha_sail(q, k, v, plan, kv_indices=table, out=out)
        return out
    want = run([most, 1], torch.cat([q[:most], q[40:]]), most)
    got = run(ql, q, most)
    assert torch.equal(got[:most], want[:most]) and torch.equal(got[40], want[most])
    if splits == 1:                                             # (a merge takes the rows of every token)
        assert (got[39] == 7).all()
