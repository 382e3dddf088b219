"""Windowed attention as a server runs it: pages given back behind the window, requests forked, pages of new tokens, the cache write and the attention
over it in one captured step; and what a windowed call refuses."""
import copy
import math
import os
import subprocess
import sys

import pytest
import torch

import window_ref as ref
from test_window_gpu import BF, DEV, E4, SCALE, Case, _i32, kernels  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,tokens,page", [(BF, 1, 128), (E4, 1, 128), (BF, 3, 32), (E4, 2, 64), (BF, 20, 128)])
def test_a_captured_server_step(dtype, tokens, page):
    """Requests of many lengths, some of them forked or ended between the replays.  The pool has just the pages that the windows need."""
    import msa_for_sail as msa
    from msa_for_sail import api
    B, hq, hk, window, sinks, steps, longest = 7, 8, 2, 200, 10, 60, 2000
    width = -(-longest // page)
    held_most = -(-sinks // page) + (window + tokens) // page + 2
    P = B * held_most + -(-900 // page)
    g = torch.Generator(device=DEV).manual_seed(tokens * 1000 + page)
    kc, vc = (torch.zeros(P, hk, page, 128, device=DEV).to(dtype) for _ in range(2))
    table, held, kv, ql = torch.full((B, width), -1, dtype=torch.int32, device=DEV), _i32([0] * B), _i32([0] * B), _i32([0] * B)
    free, num_free, shares = torch.arange(P - 1, -1, -1, dtype=torch.int32, device=DEV), _i32([P]), _i32([0] * P)
    T = B * tokens
    q, k, v = (torch.zeros(T, h, 128, dtype=BF, device=DEV) for h in (hq, hk, hk))
    out = torch.zeros(T, hq, 128, dtype=BF, device=DEV)
    missing = _i32([0])
    spaces = {n: msa.allocate_graph_workspace(B, hq, hk, max_qo_len=n, page_size=page, num_kv_splits=1) for n in (700, tokens)}

    def step(max_total, max_q, q, k, v, out, ql):
        msa.kv_pages_free(table, held, kv, free, num_free, shares, window_size=window, num_sink_tokens=sinks, page_size=page)
        kv.add_(ql)
        t = msa.paged_kv_tables(ql, kv, table, held, free, num_free, max_total_q=max_total, page_size=page, num_held_out=held, num_free_out=num_free)
        missing.add_(t["num_missing"])
        msa.kv_cache_append(k, v, kc, vc, t["slot_map"], page_size=page)
        plan = msa.fmha_sail_plan(ql, kv, hq, num_kv_heads=hk, page_size=page, window_size=window, num_sink_tokens=sinks, graph_safe=True,
                                  max_total_q=max_total, max_qo_len_override=max_q, qo_len_uniform_override=False, max_kv_len_override=longest, num_kv_splits=1,
                                  given_workspace=spaces[max_q])
        msa.fmha_sail(q, kc, vc, plan, kv_indices=t["kv_indices"], out=out)

    keys, values = [torch.zeros(0, hk, 128, dtype=BF, device=DEV) for _ in range(B)], [torch.zeros(0, hk, 128, dtype=BF, device=DEV) for _ in range(B)]

    def run(lens, fn, q, k, v, out):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=DEV, generator=g))
        at = 0
        for b, n in enumerate(lens):
            keys[b], values[b] = torch.cat([keys[b], k[at:at + n]]), torch.cat([values[b], v[at:at + n]])
            at += n
        out.fill_(5.0)
        fn()
        torch.cuda.synchronize()
        assert api.last_status() == 0 and missing.item() == 0
        places = [torch.arange(len(x) - n, len(x)) for x, n in zip(keys, lens)]
        ref.check(out[:at], None, ref.attention(q[:at], [x.to(dtype) for x in keys], [x.to(dtype) for x in values], places, window, sinks, SCALE),
                  2 ** -8, 2 ** -8 if dtype is E4 else 0.0, str(lens))
        assert (out[at:] == 5).all()

    # prompts
    lens = [700, 150, 1, 333, 0, 0, 0]
    ql.copy_(_i32(lens))
    n = sum(lens)
    big = [torch.zeros(n, h, 128, dtype=BF, device=DEV) for h in (hq, hk, hk, hq)]
    run(lens, lambda: step(n, 700, *big, ql), *big)
    # the first captured call is preceded by one that does nothing
    ql.zero_()
    step(T, tokens, q, k, v, out, ql)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(T, tokens, q, k, v, out, ql)
    for it in range(steps):
        if it in (5, 20, 40):                               # two further samples of a request; those that ended before give their rows
            kids, parent = [4, 5, 6][:2 + (it == 20)], {5: 0, 20: 1, 40: 4}[it]
            kids = [c for c in kids if c != parent]
            for c in kids:
                kv[c] = 0
            msa.kv_pages_free(table, held, kv, free, num_free, shares, window_size=window, num_sink_tokens=sinks, page_size=page)
            lost = msa.kv_pages_fork(table, held, kv, _i32([parent] * len(kids)), _i32(kids), free, num_free, shares, (kc, vc), page_size=page)
            assert lost.item() == 0
            for c in kids:
                keys[c], values[c] = keys[parent], values[parent]
        if it == 30:                                        # a request ends and another begins in its row, a drafted token is rejected
            kv[2], keys[2], values[2] = 0, keys[2][:0], values[2][:0]
            kv[3] -= 1
            keys[3], values[3] = keys[3][:-1], values[3][:-1]
        lens = [tokens if len(x) else 0 for x in keys]
        if it == 31:
            lens[2] = 1
        if it % 7 == 3:
            lens = [n - (b % 2) * (n > 1) for b, n in enumerate(lens)]
        ql.copy_(_i32(lens))
        run(lens, graph.replay, q, k, v, out)
    assert kv.tolist() == [len(x) for x in keys]
    # everything ends: the pool is whole again
    kv.zero_()
    msa.kv_pages_free(table, held, kv, free, num_free, shares, page_size=page)
    assert num_free.item() == P and sorted(free.tolist()) == list(range(P)) and not shares.any() and (table == -1).all()


@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
@pytest.mark.parametrize("layout,page", [("ragged", 0), ("hnd", 16), ("hnd", 32), ("nhd", 48), ("hnd", 100), ("nhd", 96), ("hnd", 256), ("hnd", 128)])
def test_pages_of_any_size(types, layout, page):
    """Page sizes with and without whole units of the streaming kernel, rows that need one, two and four of its row tiles, and more than it has."""
    for hq, hk, n in ((8, 1, 1), (12, 1, 1), (16, 2, 3), (32, 1, 1), (10, 2, 5), (32, 1, 3)):
        Case([n] * 3, [700, 130 + n, 2049], hq, hk, 300, 20, layout, page, *types).check()


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_scores_times_nothing(kernels, n):
    """A factor of 0 is the mean of what a row sees; so is one of a head whose keys were all zeros when they were quantised."""
    import msa_for_sail as msa
    for types in ((BF, BF), (BF, E4), (E4, E4)):
        c = Case([n], [1000], 8, 2, 130, 3, "hnd", 128, *types)
        out, _ = msa.fmha_sail(c.q, c.k, c.v, c.plan(), kv_indices=c.table, sm_scale=0.0)
        want = ref.attention(c.q, c.ks, c.vs, c.places, 130, 3, 0.0)
        ref.check(out, None, want, 2 ** -8)
        scale = torch.tensor([0.0, 1.0], device=DEV)
        out, _ = msa.fmha_sail(c.q, c.k, c.v, c.plan(), kv_indices=c.table, k_scale=scale)
        mixed = types[0] is not types[1]
        ref.check(out, None, ref.attention(c.q, c.ks, c.vs, c.places, 130, 3, SCALE, scale), 2 ** -8, 2 ** -8 if mixed else 0.0)


def test_copies_of_a_plan():
    """A plan is what its tensors hold now, whatever calls were made with it or with the plan it was copied from."""
    c = Case([1, 2], [900, 500], 8, 2, 200, 4)
    plan = c.plan()
    want = c.check(plan=plan)
    for other in (copy.deepcopy(plan), copy.copy(plan)):
        assert torch.equal(c.check(plan=other), want)
    other = copy.deepcopy(plan)
    for p in plan:
        if isinstance(p, dict):
            for t in p.values():
                if isinstance(t, torch.Tensor):
                    t.zero_()
    assert torch.equal(c.check(plan=other), want)


def test_refused_calls():
    import msa_for_sail as msa
    c = Case([1, 2], [300, 500], 8, 2, 200, 4)
    plan = c.plan()
    T = 3
    ok = dict(q=c.q, k=c.k, v=c.v, kv_indices=c.table)

    def call(**kw):
        a = {**ok, **kw}
        return msa.fmha_sail(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("plan", plan), **a)

    kv4 = torch.zeros(8, 2, 128, 72, dtype=torch.uint8, device=DEV)
    nothing = torch.empty(0, device=DEV)
    bad = [
        dict(q_offset_override=3), dict(max_score=torch.zeros(8, 4, T, device=DEV)), dict(kv_block_indexes=_i32([[[0]]])), dict(output_o=False),
        dict(v=None), dict(k=kv4, v=kv4), dict(k=c.k.half(), v=c.v.half()), dict(q=c.q.half()), dict(q=c.q.float()), dict(k=c.k.to(E4)),
        dict(q=c.q.to(E4)), dict(q=c.q[:2]), dict(q=c.q[:, :4]), dict(q=c.q[0]), dict(q=c.q[..., :64]), dict(v=c.v[:, :1]), dict(k=c.k[:, :1], v=c.v[:, :1]),
        dict(kv_indices=None), dict(kv_indices=c.table.long()), dict(kv_indices=c.table[None]), dict(kv_indices=c.table.cpu()),
        dict(k=c.k.cpu(), v=c.v.cpu()), dict(out=torch.empty(T, 8, 128, dtype=torch.float16, device=DEV)), dict(out=torch.empty(T, 8, 64, dtype=BF, device=DEV)),
        dict(out=torch.empty(T, 8, 128, dtype=BF)), dict(out=torch.empty(T, 128, 8, dtype=BF, device=DEV).transpose(1, 2)),
        dict(lse=torch.empty(T, 8, dtype=BF, device=DEV)), dict(lse=torch.empty(T, 7, device=DEV)), dict(lse=torch.empty(8, T, device=DEV).T),
        dict(sm_scale=-0.1), dict(sm_scale=math.nan), dict(sm_scale=math.inf), dict(k_scale=-1.0), dict(q=c.q.transpose(1, 2).contiguous().transpose(1, 2)[..., ::2]),
        dict(k=c.k.view(-1, 128, 2, 128)[:, :64], v=c.v.view(-1, 128, 2, 128)[:, :64]), dict(out=nothing)]
    for kw in bad:
        with pytest.raises((ValueError, RuntimeError, AssertionError)):
            call(**kw)
    # rows that do not start on 16 bytes
    wide = torch.zeros(T, 8, 136, dtype=BF, device=DEV)
    for kw in (dict(q=wide[..., 1:129]), dict(out=wide[..., 2:130]), dict(q=torch.zeros(T, 8, 132, dtype=BF, device=DEV)[..., :128])):
        with pytest.raises(RuntimeError):
            call(**kw)
    torch.cuda.synchronize()
    out, _ = call()                                             # nothing was left behind
    ref.check(out, None, c.want(), 2 ** -8)
    # a ragged plan and a paged cache, and the other way round
    r = Case([1, 2], [300, 500], 8, 2, 200, 4, "ragged", 0)
    with pytest.raises(ValueError):
        call(plan=r.plan())
    with pytest.raises(ValueError):
        msa.fmha_sail(r.q, r.k, r.v, plan)


def test_checked_build():
    """Windows on the bounds-checked library: results, and a page number that is reported and clamped."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, os.path.join(here, "checked_window_child.py")], capture_output=True, text=True, timeout=600,
                       env=dict(os.environ, MSA_BOUNDS_CHECK="1"))
    assert r.returncode == 0 and "CHECKED_WINDOW_OK" in r.stdout, r.stdout[-3000:] + "\n--- stderr ---\n" + r.stderr[-3000:]


@pytest.mark.parametrize("batch,hk,page", [(1, 1, 128), (1, 2, 32), (3, 1, 0), (5, 4, 128), (24, 2, 128), (40, 4, 64), (148, 1, 128)])
def test_few_items(batch, hk, page):
    """Uncut items, which the CTAs of clusters share where they are few, and the same cut: one to 128 tiles, ends anywhere, rows that see nothing."""
    import msa_for_sail as msa
    layout = "hnd" if page else "ragged"
    for i, (types, g, n, window, sinks) in enumerate([((BF, BF), 4, 1, 300, 5), ((E4, E4), 8, 2, 129, 0), ((BF, E4), 16, 1, 2500, 70), ((BF, BF), 16, 2, 1, 1), ((BF, BF), 1, 1, 16000, 0)]):
        lens = [n + (37 * b * (b + i)) % (900 if batch > 8 else 4000) for b in range(batch)]
        offs = [k - n for k in lens]
        if batch > 2:
            offs[1] = -n                                        # stands for the default
            lens[2] = 0
            offs[2] = 10
        c = Case([n] * batch, lens, g * hk, hk, window, sinks, layout, page, *types, offsets=offs, seed=batch + i)
        out = c.check(num_kv_splits=1)
        c.check()
        c.check(num_kv_splits=3)
        assert torch.equal(c.check(num_kv_splits=1), out)


def test_nothing_runs_while_a_status_is_set():
    """The word says that a wait ran out: whole clusters and single CTAs return, and leave the output."""
    from msa_for_sail import _lib, api
    import msa_for_sail as msa
    for batch in (1, 40):
        for types in ((BF, BF), (BF, E4), (E4, E4)):
            c = Case([1] * batch, [1500] * batch, 32, 4, 1000, 4, "hnd", 128, *types)
            plan = c.plan(num_kv_splits=1)
            out = torch.full((batch, 32, 128), 7.0, dtype=BF, device=DEV)
            api._status_word(c.q.device).fill_(_lib.STATUS_TIMEOUT)
            msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table, out=out)
            assert (out == 7).all() and api.last_status() == _lib.STATUS_TIMEOUT
            c.check(plan=plan)


@pytest.mark.parametrize("splits", [1, 3])
def test_two_graphs_of_one_plan_at_a_time(splits):
    import msa_for_sail as msa
    cases = [Case([1] * 3, [3000, 900, 5000], 32, 4, 1500, 4, seed=s) for s in (1, 2)]
    plan = cases[0].plan(num_kv_splits=splits)                  # both have its lengths
    outs = [torch.zeros(3, 32, 128, dtype=BF, device=DEV) for _ in cases]
    graphs, streams = [], [torch.cuda.Stream() for _ in cases]
    for c, out in zip(cases, outs):
        msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(20):
                msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table, out=out)
        graphs.append(g)
    for out in outs:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, out in zip(cases, outs):
        ref.check(out, None, c.want(), 2 ** -8)


def test_splits_without_a_workspace():
    """The entry point whose partials are the library's own takes windows too."""
    import ctypes
    import msa_for_sail as msa
    from msa_for_sail import _lib
    for args in ((32, 4, 1, "hnd", 128, BF, BF), (40, 1, 2, "nhd", 128, BF, E4), (8, 2, 1, "ragged", 0, E4, E4)):
        hq, hk, n, layout, page, qt, ct = args
        c = Case([n] * 3, [2000, 700, 90], hq, hk, 600, 5, layout, page, qt, ct)
        plan = c.plan(num_kv_splits=3)
        got = []
        merged = _lib.lib.msa_fmha_fwd_merged
        _lib.lib.msa_fmha_fwd_merged = lambda p, *a: got.append((_lib.MsaFmhaParams.from_buffer_copy(p._obj), a)) or merged(p, *a)
        try:
            want, _ = msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table)
        finally:
            _lib.lib.msa_fmha_fwd_merged = merged
        (p, a), = got
        out = torch.zeros_like(want)
        p.out, p.partial_o, p.partial_lse = out.data_ptr(), None, None
        assert _lib.lib.msa_fmha_fwd_split_static(ctypes.byref(p), a[0], torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        mixed = qt is not ct
        ref.check(out, None, c.want(), 2 ** -8, 2 ** -8 if mixed else 0.0, str(args))
        ref.check(want, None, c.want(), 2 ** -8, 2 ** -8 if mixed else 0.0, str(args))
