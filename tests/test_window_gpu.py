"""Attention with a sliding window and sink tokens against its definition in 64 bits."""
import itertools
import math
import random

import pytest
import torch

import window_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _i32(v, device=DEV):
    return torch.tensor(v, dtype=torch.int32, device=device)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


class Case:
    """A batch, its cache in a layout, and what its sequences' queries see."""

    def __init__(self, ql, kl, hq, hk, window, sinks, layout="hnd", page=128, q_dtype=torch.bfloat16, kv_dtype=torch.bfloat16, offsets=None,
                 nan_unseen=True, seed=1, head_scales=False, v_mean=0.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.ql, self.kl, self.hq, self.hk, self.window, self.sinks, self.page = ql, kl, hq, hk, window, sinks, page
        self.offsets = offsets
        offs = [k - q if offsets is None or offsets[i] < 0 else offsets[i] for i, (q, k) in enumerate(zip(ql, kl))]     # (negative: the default)
        self.places = [torch.arange(n) + o for n, o in zip(ql, offs)]
        self.q = _randn(g, q_dtype, sum(ql), hq, 128)
        self.scales = {}
        if head_scales:
            self.scales = dict(k_scale=torch.rand(hk, device=DEV, generator=g) + 0.5, v_scale=torch.rand(hk, device=DEV, generator=g) + 0.5)
        self.ks = [_randn(g, kv_dtype, n, hk, 128) for n in kl]
        self.vs = [(torch.randn(n, hk, 128, device=DEV, generator=g) + v_mean).to(kv_dtype) for n in kl]
        ks, vs = [k.clone() for k in self.ks], [v.clone() for v in self.vs]
        if nan_unseen:                                      # keys that no query of the sequence sees hold no numbers
            for k, v, place, n in zip(ks, vs, self.places, kl):
                j = torch.arange(n)
                see = ((j[None] <= place[:, None]) & ((j[None] > place[:, None] - window) | (j[None] < sinks))).any(0).to(DEV)
                for x in (k, v):
                    x[~see] = torch.full((1, 1, 128), math.nan, device=DEV).to(kv_dtype)
        if layout == "ragged":
            self.page_size, self.table = -1, None
            self.k, self.v = (torch.cat(x) if x else torch.empty(0, hk, 128, dtype=kv_dtype, device=DEV) for x in (ks, vs))
        else:
            self.page_size = page
            need = [-(-n // page) for n in kl]
            pages = sum(need) + 3
            order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:sum(need)]
            shape = (pages, hk, page, 128) if layout == "hnd" else (pages, page, hk, 128)
            self.k, self.v = (torch.full(shape, math.nan, device=DEV).to(kv_dtype) for _ in range(2))
            entries, at = [], 0
            for k, v, n, place in zip(ks, vs, kl, self.places):
                lo = max(0, int(place[0]) - window + 1) if len(place) else n
                for i in range(-(-n // page)):
                    phys = int(order[at])
                    at += 1
                    rows = slice(i * page, min(n, (i + 1) * page))
                    for c, x in ((self.k, k), (self.v, v)):
                        dst = c[phys].transpose(0, 1) if layout == "hnd" else c[phys]
                        dst.view(dst.dtype)[:rows.stop - rows.start] = x[rows]
                    # a page that nobody sees was given back: its entry is no page of this sequence any more
                    gone = (i + 1) * page <= lo and i * page >= sinks
                    entries.append(0 if gone and i % 2 else phys)
            self.table = _i32(entries or [0])[:len(entries)]

    def plan(self, **kw):
        import msa_for_sail as msa
        off = {} if self.offsets is None else dict(qo_offset=_i32(self.offsets, "cpu"))
        return msa.fmha_sail_plan(_i32(self.ql, "cpu"), _i32(self.kl, "cpu"), self.hq, num_kv_heads=self.hk, page_size=self.page_size,
                                  window_size=self.window, num_sink_tokens=self.sinks, **off, **kw)

    def want(self):
        return ref.attention(self.q, self.ks, self.vs, self.places, self.window, self.sinks, SCALE, self.scales.get("k_scale"), self.scales.get("v_scale"))

    def check(self, plan=None, **kw):
        import msa_for_sail as msa
        from msa_for_sail import api
        plan = self.plan(**kw) if plan is None else plan
        T = self.q.shape[0]
        lse = torch.full((T, self.hq), 7.0, device=DEV)
        out, score = msa.fmha_sail(self.q, self.k, self.v, plan, kv_indices=self.table, lse=lse, **self.scales)
        assert score is None and api.last_status() == 0
        # half a step of bf16 weights, or of pairs of e4m3 values, which queries in bf16 become over an e4m3 cache too
        mixed = self.q.dtype != self.k.dtype
        ref.check(out, lse, self.want(), 2 ** -8, 2 ** -8 if mixed else 0.0, f"{self.ql} {self.kl} {self.window} {self.sinks}")
        return out


@pytest.fixture(params=["chosen", "generic", "tcgen05"])
def kernels(request):
    """The kernels that a call takes by itself, the generic one, and the tcgen05 ones wherever they can."""
    from msa_for_sail import api
    old = api._USE_TC, api._FORCE_TC, api._USE_DECODE_TC
    if request.param != "chosen":
        api._USE_TC = api._FORCE_TC = api._USE_DECODE_TC = request.param == "tcgen05"
    yield request.param
    api._USE_TC, api._FORCE_TC, api._USE_DECODE_TC = old


LAYOUTS = [("ragged", 0), ("hnd", 128), ("nhd", 128), ("hnd", 16), ("nhd", 64)]
BF, E4 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("layout,page", LAYOUTS)
@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (100, 4), (128, 128), (129, 0), (300, 200), (5000, 64)])
def test_decode(layout, page, types, window, sinks):
    kl = [1, 127, 128, 129, 700, 1500, 256, 0, 301]
    ql = [1] * 7 + [0, 1]
    Case(ql, kl, 16, 2, window, sinks, layout, page, *types, head_scales=types[1] == E4).check()


@pytest.mark.parametrize("heads", [(64, 8), (64, 4), (16, 1), (8, 8), (6, 2), (32, 1)])
@pytest.mark.parametrize("tokens", [1, 2, 4, 7, 32])
@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
def test_a_few_tokens(heads, tokens, types):
    kl = [tokens, 1000, 384, 2049]
    Case([tokens] * 4, kl, *heads, 200, 5, "hnd", 128, *types).check()


@pytest.mark.parametrize("layout,page", LAYOUTS)
@pytest.mark.parametrize("types", [(BF, BF), (E4, E4), (BF, E4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 1), (127, 4), (128, 128), (300, 0), (513, 200), (10000, 7)])
def test_prompts(kernels, layout, page, types, window, sinks):
    Case([700, 129, 1, 256, 0, 300], [700, 1000, 500, 256, 40, 333], 8, 2, window, sinks, layout, page, *types).check()


@pytest.mark.parametrize("types", [(BF, BF), (E4, E4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (200, 300), (1000, 0), (4096, 4), (300, 32), (300, 33), (500, 160), (500, 250), (64, 128)])
def test_a_chunk_behind_a_long_prefix(kernels, types, window, sinks):
    Case([1000], [9001], 4, 1, window, sinks, "hnd", 128, *types).check()


@pytest.mark.parametrize("n", [1, 3, 140, 300])
@pytest.mark.parametrize("layout,page", [("hnd", 128), ("ragged", 0), ("hnd", 16)])
@pytest.mark.parametrize("types", [(BF, BF), (E4, E4), (BF, E4)])
def test_places_before_and_behind_the_keys(kernels, n, layout, page, types):
    """Offsets of the caller's own: rows before the first key see nothing, rows far behind the last one the sinks alone."""
    kl = [500, 500, 500, 500, 0, 130]
    Case([n] * 6, kl, 8, 2, 100, 40, layout, page, *types, offsets=[700, 450, 5000000, 0, 10, 200]).check()
    out = Case([n] * 2, [400, 50], 8, 2, 100, 0, layout, page, *types, offsets=[2000000, 1000]).check()
    assert not out.any()


@pytest.mark.parametrize("splits", [-1, 1, 2, 5, 64])
@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
def test_splits(splits, types):
    for ql, kl in (([1] * 3, [9000, 100, 3001]), ([4, 2, 1], [5000, 4000, 129])):
        Case(ql, kl, 16, 2, 2500, 130, "hnd", 128, *types).check(num_kv_splits=splits)


@pytest.mark.parametrize("kw", [dict(ql=[1], kl=[3000], hq=16, hk=2), dict(ql=[700], kl=[900], hq=4, hk=1)])
def test_a_window_wider_than_the_keys_is_no_window(kw):
    import msa_for_sail as msa
    c = Case(window=(1 << 31) - 1, sinks=0, nan_unseen=False, **kw)
    got = c.check()
    plan = msa.fmha_sail_plan(_i32(c.ql, "cpu"), _i32(c.kl, "cpu"), c.hq, num_kv_heads=c.hk, page_size=128)
    plain, _ = msa.fmha_sail(c.q, c.k, c.v, plan, kv_indices=c.table)
    assert (got.float() - plain.float()).abs().max() <= 2 ** -7 * plain.float().abs().max()


def test_strides_scales_and_outputs(kernels):
    import msa_for_sail as msa
    for types in ((BF, BF), (BF, E4), (E4, E4)):
        for ql, kl in (([1, 1], [700, 2000]), ([300, 200], [700, 2000])):
            c = Case(ql, kl, 8, 2, 333, 9, "hnd", 128, *types, head_scales=types[1] == E4)
            want = c.check()
            T = sum(ql)
            wide = torch.zeros(T, 3, 8, 256, device=DEV).to(types[0])
            wide[:, 1, :, 128:] = c.q
            big = torch.zeros(c.k.shape[0], 2, 4, 128, 128, device=DEV).to(types[1])
            big[:, 0, 1:3], big[:, 1, 1:3] = c.k, c.v
            out = torch.full((T, 8, 384), 3.0, dtype=torch.bfloat16, device=DEV)
            msa.fmha_sail(wide[:, 1, :, 128:], big[:, 0, 1:3], big[:, 1, 1:3], c.plan(), kv_indices=c.table, out=out[..., 128:256], **c.scales)
            assert torch.equal(out[..., 128:256], want)
            assert (out[..., :128] == 3).all() and (out[..., 256:] == 3).all()
            f32 = torch.empty(T, 8, 128, device=DEV)
            msa.fmha_sail(c.q, c.k, c.v, c.plan(), kv_indices=c.table, out=f32, **c.scales)
            assert (f32 - want.float()).abs().max() <= 2 ** -8 * want.float().abs().max()
            # scales as floats, and all four of them
            got, _ = msa.fmha_sail(c.q, c.k, c.v, c.plan(), kv_indices=c.table, sm_scale=SCALE / 4, q_scale=2.0, k_scale=2.0, v_scale=0.5, o_scale=4.0)
            plain, _ = msa.fmha_sail(c.q, c.k, c.v, c.plan(), kv_indices=c.table)
            assert (got.float() - 2 * plain.float()).abs().max() <= 2 ** -7 * got.float().abs().max()


def _device_plan(c, max_q, T, splits=1, **kw):
    import msa_for_sail as msa
    ws = msa.allocate_graph_workspace(len(c.ql), c.hq, c.hk, max_qo_len=max_q, page_size=max(c.page_size, 0), num_kv_splits=splits)
    return msa.fmha_sail_plan(_i32(c.ql), _i32(c.kl), c.hq, num_kv_heads=c.hk, page_size=c.page_size, window_size=c.window, num_sink_tokens=c.sinks,
                              num_kv_splits=splits, graph_safe=True, max_total_q=T, max_qo_len_override=max_q, qo_len_uniform_override=False,
                              max_kv_len_override=max(c.kl), given_workspace=ws, **kw)


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("layout,page", [("hnd", 128), ("ragged", 0), ("nhd", 16)])
@pytest.mark.parametrize("types", [(BF, BF), (BF, E4), (E4, E4)])
def test_device_made_plans(kernels, splits, layout, page, types):
    for ql, kl, max_q in (([1, 1, 0, 1], [900, 3000 - 7, 10, 128], 1), ([4, 1, 2, 0], [900, 2501, 10, 0], 4), ([300, 1, 140, 0], [900, 2501, 140, 5], 400)):
        c = Case(ql, kl, 8, 2, 257, 3, layout, page, *types)
        c.check(plan=_device_plan(c, max_q, sum(ql), splits))


@pytest.mark.parametrize("max_q", [1, 300])
def test_a_captured_step_sees_new_lengths(max_q):
    import msa_for_sail as msa
    c = Case([max_q, max_q, max_q], [1000, 2000, 400], 8, 2, 300, 4)
    ql, kl = _i32(c.ql), _i32(c.kl)
    T = 3 * max_q
    ws = msa.allocate_graph_workspace(3, 8, 2, max_qo_len=max_q, page_size=128, num_kv_splits=2)
    out = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(64, dtype=torch.int32, device=DEV)
    kc, vc = (torch.zeros(64, 2, 128, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros_like(c.q)

    def step():
        plan = msa.fmha_sail_plan(ql, kl, 8, num_kv_heads=2, page_size=128, window_size=300, num_sink_tokens=4, num_kv_splits=2, graph_safe=True,
                                  max_total_q=T, max_qo_len_override=max_q, qo_len_uniform_override=False, max_kv_len_override=4096, given_workspace=ws)
        msa.fmha_sail(q, kc, vc, plan, kv_indices=table, out=out)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for ql_, kl_ in (([max_q] * 3, [1000, 2000, 400]), ([1, 0, max_q], [129, 50, 3001]), ([0, 1, 1], [0, 1, 2500])):
        d = Case(ql_, kl_, 8, 2, 300, 4, seed=sum(kl_))
        ql.copy_(_i32(ql_)), kl.copy_(_i32(kl_))
        kc[:d.k.shape[0]], vc[:d.v.shape[0]], q[:d.q.shape[0]] = d.k, d.v, d.q
        table[:d.table.shape[0]] = d.table
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        n = sum(ql_)
        ref.check(out[:n], None, d.want(), 2 ** -8, what=str((ql_, kl_)))


def test_mixed_batches_are_planned_in_parts():
    c = Case([1, 2, 300, 150], [800, 3001, 300, 900], 8, 2, 200, 10)
    c.check(split_prefill_decode=True)


def test_two_streams_and_another_current_device():
    import msa_for_sail as msa
    c = Case([1] * 8, [4000 + 100 * i for i in range(8)], 16, 2, 1000, 4)
    plan = [c.plan() for _ in range(2)]
    want = c.check()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [None, None]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i], _ = msa.fmha_sail(c.q, c.k, c.v, plan[i], kv_indices=c.table)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_rows_behind_the_last_sequence_are_left_as_they_were(kernels):
    import msa_for_sail as msa
    for types in ((BF, BF), (BF, E4), (E4, E4)):
        for max_q, ql in ((1, [1, 0, 1]), (300, [300, 0, 20])):
            c = Case(ql, [900, 20, 2000], 8, 2, 150, 2, "hnd", 128, *types)
            T = sum(ql)
            q = torch.cat([c.q, torch.ones(9, 8, 128, device=DEV).to(types[0])])
            out = torch.full((T + 9, 8, 128), 3.0, dtype=torch.bfloat16, device=DEV)
            msa.fmha_sail(q, c.k, c.v, _device_plan(c, max_q, T + 9), kv_indices=c.table, out=out)
            assert (out[T:] == 3).all()
            ref.check(out[:T], None, c.want(), 2 ** -8, 2 ** -8 if types[0] != types[1] else 0.0)


def test_random_batches(kernels):
    rng = random.Random(5)
    for i in range(30):
        b = rng.choice([1, 2, 5])
        top = rng.choice([1, 3, 40, 400])
        ql = [rng.randint(0, top) for _ in range(b)]
        kl = [n + rng.choice([0, 1, rng.randint(0, 3000)]) for n in ql]
        hq, hk = rng.choice([(8, 2), (16, 1), (4, 4), (12, 4)])
        types = rng.choice([(BF, BF), (BF, E4), (E4, E4)])
        layout, page = rng.choice(LAYOUTS)
        window, sinks = rng.choice([1, 17, 128, 300, 1024]), rng.choice([0, 1, 30, 128, 500])
        if sum(ql):
            Case(ql, kl, hq, hk, window, sinks, layout, page, *types, seed=i).check()


def test_large_values_and_infinities_outside_the_window(kernels):
    """What a query does not see may be anything, and a far larger score outside the window is not a maximum."""
    for types in ((BF, BF), (BF, E4), (E4, E4)):
        for n in (1, 200):
            c = Case([n], [1500], 4, 1, 130, 2, "hnd", 128, *types, nan_unseen=False)
            want = c.check()
            lo = 1500 - n - 130 + 1
            for i in range(2, lo):
                page, row = int(c.table[i // 128]), i % 128
                if (i // 128 + 1) * 128 <= lo and i // 128 > 0 and (i // 128) % 2:
                    continue
                c.k[page, :, row] = torch.full((128,), math.inf if i % 2 else 440.0, device=DEV).to(c.k.dtype)
                c.v[page, :, row] = torch.full((128,), -math.inf if i % 3 else 440.0, device=DEV).to(c.v.dtype)
            assert torch.equal(c.check(), want)
