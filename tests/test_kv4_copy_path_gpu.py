"""Attention over a 4-bit cache where it runs on bf16 copies of the pages: queries of more than 128 rows, page scores, pages that many tokens
share.  What holds for the kernels that read 4 bits holds here too."""
import pytest
import torch

import serving_ref as ref
from test_kv4_attention_gpu import DEV, P_BF16, Batch

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _empty_batch():
    """A call without a token, and one whose sequences have no key: neither has a page to read."""
    import msa_for_sail as msa
    k, v = (torch.zeros(3, 2, 128, 72, dtype=torch.uint8, device=DEV) for _ in range(2))
    return msa, k, v, torch.empty(0, dtype=torch.int32, device=DEV)


def test_a_table_shorter_than_a_host_made_plan():
    import msa_for_sail as msa
    b = Batch(101, [200, 1], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    for n in (4, 0):
        with pytest.raises(ValueError, match="kv_indices must have the 5 pages"):
            msa.fmha_sail(q, k, v, b.plan(), kv_indices=table[:n].clone())
    out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table)
    ref.check_attention(out, None, b.want(), P_BF16, "the whole table")


def test_a_call_without_tokens():
    msa, k, v, none = _empty_batch()
    plan = msa.fmha_sail_plan(torch.tensor([0, 0]), torch.tensor([300, 200]), 16, num_kv_heads=2, page_size=128, use_kv4_cache=True)
    out, _ = msa.fmha_sail(torch.empty(0, 16, 128, dtype=torch.bfloat16, device=DEV), k, v, plan, kv_indices=none)
    assert out.shape == (0, 16, 128)


def test_offsets_of_any_type_and_stride():
    """An override may be int64, or every second entry of a tensor: it is what it says, entry by entry."""
    import msa_for_sail as msa
    b = Batch(102, [140, 3], [300, 200], 8, 2, offsets=[100, 150])
    q, k, v, table = b.cuda()
    plan = msa.fmha_sail_plan(torch.tensor(b.qo), torch.tensor(b.kv), 8, num_kv_heads=2, page_size=128, use_kv4_cache=True)
    wide = torch.tensor([100, -7, 150, -7], device=DEV)
    for off in (wide[::2], wide[::2].to(torch.int32), wide.to(torch.int32)[::2]):
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table, q_offset_override=off)
        ref.check_attention(out, None, b.want(), P_BF16, "offsets")
    with pytest.raises(ValueError, match="q_offset_override must be"):
        msa.fmha_sail(q, k, v, plan, kv_indices=table, q_offset_override=wide[:1])


def _paths(seed=103):
    """(name, batch, plan, what the call adds) of every way to the copies."""
    prompt = Batch(seed, [200, 1], [300, 200], 16, 2)
    shared = Batch(seed + 1, [300], [900], 8, 2)
    few = Batch(seed + 2, [9, 2], [500, 260], 64, 4)
    return [("prompt", prompt, prompt.plan(), {}), ("scores", prompt, prompt.plan(output_maxscore=True), dict(output_o=False)),
            ("shared pages", shared, shared.plan(kv_block_num=4), dict(kv_block_indexes=shared.blocks(4).to(DEV))), ("9 tokens", few, few.plan(), {})]


def _results(x):
    return [t.clone() for t in x if t is not None]


def _dirty():
    """What the allocator hands out next holds NaN, as memory that others have used may."""
    torch.cuda.empty_cache()
    junk = torch.full((1 << 27,), float("nan"), dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    del junk


@pytest.mark.parametrize("i", range(4))
def test_a_number_that_is_no_page(i):
    """Checked, it is refused; else it is the nearest page, never memory that nobody wrote."""
    import msa_for_sail as msa
    from msa_for_sail import api
    name, b, plan, kw = _paths()[i]
    q, k, v, table = b.cuda()
    for bad, near in ((10 ** 6, k.shape[0] - 1), (-3, 0), (k.shape[0], k.shape[0] - 1)):
        wrong, right = table.clone(), table.clone()
        wrong[1], right[1] = bad, near
        want = _results(msa.fmha_sail(q, k, v, plan, kv_indices=right, check_input_valid=True, **kw))
        _dirty()
        got = _results(msa.fmha_sail(q, k, v, plan, kv_indices=wrong, **kw))
        api.last_status()                                       # (the build with bounds checks reports the number)
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and len(got) == len(want) == 1, name
        with pytest.raises(AssertionError, match="outside"):
            msa.fmha_sail(q, k, v, plan, kv_indices=wrong, check_input_valid=True, **kw)


def test_copies_of_the_pages_that_count():
    """Entries behind the number that the device has are not copied; numbers that are no pages are the nearest ones."""
    from msa_for_sail import cache
    c = ref.random_kv4(torch.Generator().manual_seed(6), 7, 3).to(DEV)
    want = ref.kv4_values(c)
    pages, used = _i32([6, -1, 2, 7, 10 ** 6, 4, -1, 5]), _i32([99, 6])
    got = cache.unpack_pages(c, pages, used[1:].data_ptr()).double().cpu()
    assert torch.equal(got[:6], want[[6, 0, 2, 6, 6, 4]])
    assert torch.equal(cache.unpack_pages(c, pages).double().cpu(), want[[6, 0, 2, 6, 6, 4, 0, 5]])
    assert torch.equal(cache.unpack_pages(c, pages[:3], used.data_ptr()).double().cpu(), want[[6, 0, 2]])


@pytest.mark.parametrize("what", ["pages", "table"])
def test_the_checked_build_reports_what_the_copies_clamp(what):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, os.path.join(here, "checked_kv4_child.py"), what], capture_output=True, text=True, timeout=600,
                       env=dict(os.environ, MSA_BOUNDS_CHECK="1"))
    assert r.returncode == 0 and "CHECKED_KV4_OK" in r.stdout, r.stdout[-2000:] + "\n--- stderr ---\n" + r.stderr[-3000:]


@pytest.mark.parametrize("rows,scores,splits", [(200, False, 1), (40, False, 2), (200, True, 1), (1, True, 1), (3, True, 1)])
def test_an_empty_table_has_no_keys(rows, scores, splits):
    """As on the kernels that read 4 bits: zeros, an LSE and scores of -inf; rows behind the last sequence stay as they were."""
    import msa_for_sail as msa
    hq, pad = 4, 3
    k, v = (ref.random_kv4(torch.Generator().manual_seed(7), 6, 2).to(DEV) for _ in range(2))
    q = torch.ones(rows + pad, hq, 128, dtype=torch.bfloat16, device=DEV)
    ws = msa.allocate_graph_workspace(1, hq, num_kv_heads=2, page_size=128, max_qo_len=rows + pad, num_kv_splits=splits)
    plan = msa.fmha_sail_plan(_i32([rows]), _i32([600]), hq, num_kv_heads=2, page_size=128, num_kv_splits=splits, graph_safe=True, output_maxscore=scores,
                              max_total_q=rows + pad, max_qo_len_override=rows, qo_len_uniform_override=True, max_kv_len_override=600, qo_offset=_i32([-1]),
                              given_workspace=ws, use_kv4_cache=True)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    if scores:
        _, ms = msa.fmha_sail(q, k, v, plan, kv_indices=none, output_o=False)
        assert (ms == -float("inf")).all()
        return
    out, lse = torch.full((rows + pad, hq, 128), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((rows + pad, hq), 7.0, device=DEV)
    msa.fmha_sail(q, k, v, plan, kv_indices=none, out=out, lse=lse)
    assert (out[:rows] == 0).all() and (lse[:rows] == -float("inf")).all()
    if splits == 1:
        assert (out[rows:] == 7).all() and (lse[rows:] == 7).all()


def test_sequences_without_a_key():
    import msa_for_sail as msa
    msa, k, v, none = _empty_batch()
    plan = msa.fmha_sail_plan(torch.tensor([200, 5]), torch.tensor([0, 0]), 16, num_kv_heads=2, page_size=128, use_kv4_cache=True)
    lse = torch.empty(205, 16, device=DEV)
    out, _ = msa.fmha_sail(torch.ones(205, 16, 128, dtype=torch.bfloat16, device=DEV), k, v, plan, kv_indices=none, lse=lse)
    assert (out == 0).all() and (lse == -float("inf")).all()


def _one_value(x, **kw):
    return torch.tensor([x], device=DEV, **kw)


@pytest.mark.parametrize("path", ["prompt", "tokens", "shared pages", "scores"])
@pytest.mark.parametrize("hk", [1, 2])
def test_scales_stay_on_the_device(path, hk):
    """One value for all heads, or one per head, of every scale: nothing is read back, so a graph sees what they become."""
    import msa_for_sail as msa
    hq = 8 * hk
    b = Batch(110, *{"prompt": ([200, 1], [300, 200]), "tokens": ([1, 1], [300, 200]), "shared pages": ([300], [600]), "scores": ([140], [300])}[path],
              hq, hk, q_dtype=torch.float8_e4m3fn if path in ("prompt", "tokens") else torch.bfloat16)
    q, k, v, table = b.cuda()
    kw, want_kw = {}, {}
    plan = b.plan(**{"shared pages": dict(kv_block_num=2), "scores": dict(output_maxscore=True)}.get(path, {}))
    if path == "shared pages":
        blocks = b.blocks(2)
        kw, want_kw = dict(kv_block_indexes=blocks.to(DEV)), dict(blocks=blocks)
    if path == "scores":
        kw = dict(output_o=False)
    scales = dict(q_scale=_one_value(0.5), k_scale=_one_value(1.5), v_scale=torch.rand(hk, device=DEV) + 0.5, o_scale=_one_value(2.0))
    run = lambda: [x for x in msa.fmha_sail(q, k, v, plan, kv_indices=table, **scales, **kw) if x is not None][0]
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    scales["q_scale"].fill_(0.75), scales["k_scale"].fill_(0.25), scales["v_scale"].mul_(3.0), scales["o_scale"].fill_(0.125)
    graph.replay()
    torch.cuda.synchronize()
    if path == "scores":                                        # largest raw products: no scale enters
        plain = msa.fmha_sail(q, k, v, plan, kv_indices=table, **kw)[1]
        assert torch.equal(got, plain)
        return
    want = b.want(k_scale=torch.full((hk,), 0.75 * 0.25), v_scale=scales["v_scale"] * 0.125, **want_kw)
    ref.check_attention(got, None, want, P_BF16, path)


@pytest.mark.parametrize("path", ["prompt", "tokens"])
def test_every_form_of_a_scale(path):
    """Floats, one value in host memory (fp64 too), one value and one per head on the device: the same attention."""
    import msa_for_sail as msa
    b = Batch(111, [200 if path == "prompt" else 2], [300], 8, 2)
    q, k, v, table = b.cuda()
    plan = b.plan()
    want = b.want(k_scale=torch.full((2,), 0.5 * 0.25), v_scale=torch.full((2,), 4.0 * 0.5))
    forms = [lambda x: x, lambda x: torch.tensor(x), lambda x: torch.tensor([x], dtype=torch.float64), _one_value, lambda x: _one_value(x, dtype=torch.bfloat16),
             lambda x: torch.full((2,), x, device=DEV), lambda x: torch.full((2,), x), lambda x: torch.full((4,), x, device=DEV)[::2]]
    for i, f in enumerate(forms):
        lse = torch.empty(b.T, 8, device=DEV)
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table, q_scale=f(0.5), k_scale=f(0.25), v_scale=f(4.0), o_scale=f(0.5), lse=lse)
        ref.check_attention(out, lse, want, P_BF16, f"{path}, form {i}")
    for name in ("q_scale", "k_scale", "v_scale", "o_scale"):
        with pytest.raises(AssertionError, match="must have 2 entries"):
            msa.fmha_sail(q, k, v, plan, kv_indices=table, **{name: torch.ones(3, device=DEV)})
    # one value in host memory does not stop a capture
    graph, one = torch.cuda.CUDAGraph(), torch.tensor(0.5)
    first = msa.fmha_sail(q, k, v, plan, kv_indices=table, k_scale=one)[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table, k_scale=one)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


@pytest.mark.parametrize("kind", ["kv4", "bf16"])
def test_first_prompt_of_a_process_inside_a_capture(kind, monkeypatch):
    """The word that kernels report to is not made inside a capture, where it would belong to the graph and hold anything until a replay."""
    import msa_for_sail as msa
    from msa_for_sail import api
    b = Batch(112, [200, 1], [300, 200], 8, 2)
    q, k, v, table = b.cuda()
    if kind == "bf16":
        k, v = (ref.kv4_values(x).nan_to_num(0.0).to(torch.bfloat16).to(DEV) for x in (b.k, b.v))
    plan = b.plan()
    msa.fmha_sail(q, k, v, plan, kv_indices=table)
    torch.cuda.synchronize()
    monkeypatch.setattr(api, "_STATUS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table)
    assert not api._STATUS
    first, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table)    # before any replay
    ref.check_attention(first, None, b.want(), P_BF16, "eager")
    graph.replay()
    torch.cuda.synchronize()
    ref.check_attention(out, None, b.want(), P_BF16, "captured")


@pytest.mark.parametrize("kind", ["kv4", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("sparse", [False, True])
def test_fp32_rows_behind_the_last_sequence(kind, n, sparse):
    """An fp32 result of an unsplit call: rows behind the last sequence of a padded batch stay as they were, bit for bit, and what is between
    the rows of a wider buffer too."""
    import msa_for_sail as msa
    qo, pad, hq = [n, 1, 0], 4, 16
    b = Batch(113, qo, [500, 130, 0], hq, 2)
    q, k, v, table = b.cuda()
    if kind == "bf16":
        k, v = (ref.kv4_values(x).nan_to_num(0.0).to(torch.bfloat16).to(DEV) for x in (b.k, b.v))
    T = b.T + pad
    q = torch.cat([q, torch.full((pad, hq, 128), float("nan"), dtype=torch.bfloat16, device=DEV)])
    blocks = torch.cat([b.blocks(3), torch.zeros(pad, 2, 3, dtype=torch.int32)])
    kbn = 3 if sparse else -1
    ws = msa.allocate_graph_workspace(3, hq, num_kv_heads=2, page_size=128, num_kv_splits=1, kv_block_num=kbn, max_qo_len=n + 2)
    off = _i32([-1] * 3)

    def run(out):
        plan = msa.fmha_sail_plan(_i32(qo), _i32(b.kv), hq, num_kv_heads=2, page_size=128, kv_block_num=kbn, num_kv_splits=1, graph_safe=True, max_total_q=T,
                                  max_qo_len_override=n, qo_len_uniform_override=False, max_kv_len_override=600, qo_offset=off, given_workspace=ws,
                                  use_kv4_cache=kind == "kv4")
        msa.fmha_sail(q, k, v, plan, kv_indices=table, out=out, **(dict(kv_block_indexes=blocks.to(DEV)) if sparse else {}))

    was = torch.randn(T, hq + 3, 128, device=DEV)
    wide = was.clone()
    run(wide[:, 1:1 + hq])
    ref.check_attention(wide[:b.T, 1:1 + hq], None, b.want(**(dict(blocks=blocks[:b.T]) if sparse else {})), P_BF16, "real rows")
    assert torch.equal(wide[b.T:], was[b.T:]) and torch.equal(wide[:, 0], was[:, 0]) and torch.equal(wide[:, 1 + hq:], was[:, 1 + hq:])


@pytest.mark.parametrize("path", ["tokens", "prompt", "selected", "another cache"])
@pytest.mark.parametrize("on_device", [False, True])
def test_partials_are_those_of_a_call(path, on_device):
    """A plan for a 4-bit cache holds no partials; whatever runs with it, the copies and a cache of another type too, brings its own."""
    import msa_for_sail as msa
    qo, kv = {"prompt": ([40, 1], [900, 700])}.get(path, ([1, 2], [900, 700]))
    b = Batch(114, qo, kv, 16, 4)
    q, k, v, table = b.cuda()
    blocks, kbn = (b.blocks(32), 32) if path == "selected" else (None, -1)       # (fewer pages are not cut: a merge costs more)
    if path == "another cache":
        k, v = (ref.kv4_values(x).nan_to_num(0.0).to(torch.bfloat16).to(DEV) for x in (b.k, b.v))
    if on_device:
        ws = msa.allocate_graph_workspace(2, 16, num_kv_heads=4, page_size=128, max_qo_len=max(qo), kv_block_num=kbn, num_kv_splits=1)
        plan = msa.fmha_sail_plan(_i32(qo), _i32(kv), 16, num_kv_heads=4, page_size=128, kv_block_num=kbn, num_kv_splits=4, graph_safe=True, max_total_q=b.T,
                                  max_qo_len_override=max(qo), qo_len_uniform_override=False, max_kv_len_override=900, qo_offset=_i32([-1, -1]),
                                  given_workspace=ws, use_kv4_cache=True)
    else:
        plan = b.plan(num_kv_splits=4, kv_block_num=kbn)
    assert plan[3]["num_kv_splits"] > 1 and plan[3]["workspace_o"] is None and plan[3]["workspace_lse"] is None
    lse = torch.empty(b.T, 16, device=DEV)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.empty(b.T, 16, 128, dtype=dtype, device=DEV)
        msa.fmha_sail(q, k, v, plan, kv_indices=table, out=out, lse=lse, **(dict(kv_block_indexes=blocks.to(DEV)) if blocks is not None else {}))
        want = b.want(**(dict(blocks=blocks) if blocks is not None else {}))
        # The decode kernel of a bf16 cache adds up the weights as it has rounded them, each by half a step (2^-8) at most, so their sum is
        # within 2^-8 of the exact one and its logarithm within -log(1 - 2^-8) < 2^-8 + 2^-16.
        ref.check_attention(out, None if path == "another cache" else lse, want, P_BF16, path)
        assert path != "another cache" or ((lse.double().cpu() - want[1]).abs() <= want[3] + 2.0 ** -15 + 2.0 ** -21 * want[1].abs() + 2.0 ** -8 + 2.0 ** -16).all()
