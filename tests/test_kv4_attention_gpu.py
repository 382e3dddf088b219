"""fmha_sail over a 4-bit cache against 64-bit attention over the values that the cache stands for."""
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
# P is rounded to f16 by the decode kernel (half a step: 2^-11), to bf16 by the prefill kernels (2^-8, and 2^-8 for its sum over a
# different rounding; their exponential is good to 7.5e-5)
P_F16, P_BF16 = 2.0 ** -11, 2.0 ** -7 + 2.0 ** -13


def _gen(seed):
    return torch.Generator().manual_seed(seed)


class Batch:
    """A random batch; scale bytes behind the last key of a sequence are NaN, as if nobody ever wrote there."""

    def __init__(self, seed, qo_lens, kv_lens, hq, hk, extra_pages=2, q_dtype=torch.bfloat16, gap=False, offsets=None):
        g = self.g = _gen(seed)
        self.qo, self.kv, self.hq, self.hk = qo_lens, kv_lens, hq, hk
        need = [-(-n // 128) for n in kv_lens]
        self.indptr = [sum(need[:i]) for i in range(len(need) + 1)]
        P = self.indptr[-1] + extra_pages
        self.k, self.v = ref.random_kv4(g, P, hk), ref.random_kv4(g, P, hk)
        self.table = torch.randperm(P, generator=g)[:self.indptr[-1]].to(torch.int32)
        for b, n in enumerate(kv_lens):
            if n % 128:
                page = int(self.table[self.indptr[b + 1] - 1])
                for c in (self.k, self.v):
                    c.view(P, hk, -1)[page, :, 128 * 64 + 8 * (n % 128):] = 0x7F
        self.T = sum(qo_lens)
        self.q = torch.randn(self.T, hq, 128, generator=g).to(q_dtype)
        self.offsets = offsets if offsets is not None else [k - q for q, k in zip(qo_lens, kv_lens)]
        self.gap = gap

    def cuda(self):
        k, v = self.k.to(DEV), self.v.to(DEV)
        if self.gap:                                            # keys and values of a page in one allocation
            both = torch.empty((k.shape[0], 2) + k.shape[1:], dtype=torch.uint8, device=DEV)
            both[:, 0], both[:, 1] = k, v
            k, v = both[:, 0], both[:, 1]
        return self.q.to(DEV), k, v, self.table.to(DEV)

    def plan(self, **kw):
        import msa_for_sail as msa
        if kw.pop("given", True):
            kw["num_kv_heads"] = self.hk
        off = None if self.offsets == [k - q for q, k in zip(self.qo, self.kv)] else torch.tensor(self.offsets, dtype=torch.int32)
        return msa.fmha_sail_plan(torch.tensor(self.qo, dtype=torch.int32), torch.tensor(self.kv, dtype=torch.int32), self.hq, page_size=128,
                                  qo_offset=off, use_kv4_cache=True, **kw)

    def want(self, **kw):
        return ref.attention(self.q, ref.kv4_values(self.k).nan_to_num(0.0), ref.kv4_values(self.v).nan_to_num(0.0), self.table, self.indptr, self.qo,
                             self.kv, self.offsets, **kw)

    def blocks(self, kbn, pad=0.3):
        """Ascending visible pages per (token, head), -1 behind the last; some rows select nothing at all."""
        out = torch.full((self.T, self.hk, kbn), -1, dtype=torch.int32)
        t = 0
        for b, n in enumerate(self.qo):
            pages = self.indptr[b + 1] - self.indptr[b]
            for i in range(n):
                for h in range(self.hk):
                    most = min(kbn, pages)
                    m = most if torch.rand(1, generator=self.g) > pad else int(torch.randint(0, most + 1, (1,), generator=self.g))
                    out[t, h, :m] = torch.randperm(pages, generator=self.g)[:m].sort().values.to(torch.int32)
                t += 1
        return out


RAGGED = [1, 127, 128, 129, 500, 0, 1300, 255]


@pytest.mark.parametrize("hq,hk", [(8, 1), (16, 1), (16, 2), (64, 4), (4, 4), (12, 2), (3, 1), (20, 1), (40, 1)])
@pytest.mark.parametrize("splits", [-1, 1, 3])
def test_decode_ragged(hq, hk, splits):
    import msa_for_sail as msa
    b = Batch(hq + splits, [1] * len(RAGGED), RAGGED, hq, hk)
    q, k, v, table = b.cuda()
    lse = torch.empty(b.T, hq, device=DEV)
    out, _ = msa.fmha_sail(q, k, v, b.plan(num_kv_splits=splits), kv_indices=table, lse=lse)
    ref.check_attention(out, lse, b.want(), P_F16, f"{hq}/{hk} splits {splits}")
    assert (out[5] == 0).all() and torch.isinf(lse[5]).all()      # a sequence without a key


@pytest.mark.parametrize("n", [2, 3, 8])
@pytest.mark.parametrize("hq,hk", [(16, 2), (16, 1), (8, 8), (6, 2)])
def test_decode_of_several_tokens(n, hq, hk):
    import msa_for_sail as msa
    kv = [n, 130, 700, 128 + n, 2100]
    b = Batch(n * hq, [n, 1, n, 0, n], kv, hq, hk, gap=True)
    q, k, v, table = b.cuda()
    out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table)
    ref.check_attention(out, None, b.want(), P_F16, f"{n} tokens")


def test_offsets_that_leave_rows_empty():
    import msa_for_sail as msa
    b = Batch(3, [4, 4, 4], [300, 5, 200], 8, 2, offsets=[126, 0, 1000])
    b2 = Batch(3, [4, 4, 4], [300, 5, 200], 8, 2)
    q, k, v, table = b.cuda()
    lse = torch.empty(b.T, 8, device=DEV)
    out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table, lse=lse)
    ref.check_attention(out, lse, b.want(), P_F16, "offsets")
    # the same through the override, with rows before the first key
    b2.offsets = [-2, 0, 1000]
    out, _ = msa.fmha_sail(q, k, v, b2.plan(), kv_indices=table, q_offset_override=torch.tensor([-2, 0, 1000], dtype=torch.int32, device=DEV), lse=lse)
    ref.check_attention(out, lse, b2.want(), P_F16, "override")
    assert (out[:2] == 0).all() and torch.isinf(lse[:2]).all()


@pytest.mark.parametrize("q_dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("sm_scale", [None, 0.3, 0.0, -0.1])
def test_scales_and_types(q_dtype, sm_scale):
    import msa_for_sail as msa
    b = Batch(9, [1, 2, 1], [700, 90, 128], 16, 2, q_dtype=q_dtype)
    q, k, v, table = b.cuda()
    ks, vs = torch.tensor([0.7, 1.9], device=DEV), torch.tensor([3.0, 0.01], device=DEV)
    for out_dtype in (torch.bfloat16, torch.float32):
        for splits in (1, 2):
            out = torch.empty(b.T, 16, 136, dtype=out_dtype, device=DEV)[..., :128]
            lse = torch.empty(b.T, 16, device=DEV)
            msa.fmha_sail(q, k, v, b.plan(num_kv_splits=splits), kv_indices=table, k_scale=ks, v_scale=vs, o_scale=2.0, out=out, lse=lse, sm_scale=sm_scale)
            want = b.want(k_scale=ks, v_scale=vs * 2, **({} if sm_scale is None else dict(sm_scale=sm_scale)))
            ref.check_attention(out, lse, want, P_F16, f"{out_dtype} {splits}")


def test_large_and_small_queries():
    """A query row is scaled by a power of two before it becomes f16: neither huge nor tiny rows lose digits."""
    import msa_for_sail as msa
    b = Batch(10, [1] * 4, [300] * 4, 8, 1)
    b.q = b.q * torch.tensor([1e-30, 1e4, 3e-5, 1.0])[:, None, None].to(torch.bfloat16)
    b.q[3, 0] = 0
    q, k, v, table = b.cuda()
    lse = torch.empty(4, 8, device=DEV)
    scale = [1e29, 1e-5, 3e3, 1.0]
    for i in range(4):
        out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table, lse=lse, sm_scale=scale[i])
        want = b.want(sm_scale=scale[i])
        ref.check_attention(out[i:i + 1], lse[i:i + 1], tuple(x[i:i + 1] for x in want), P_F16, f"scale {scale[i]}")


def test_not_a_number_in_a_visible_place_stays_in_its_head():
    import msa_for_sail as msa
    b = Batch(11, [1, 1], [300, 200], 16, 2)
    page = int(b.table[1])
    b.v.view(b.v.shape[0], 2, -1)[page, 1, 128 * 64 + 8 * 5 + 3] = 0x7F          # elements 48..63 of key 133, head 1, sequence 0
    q, k, v, table = b.cuda()
    out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table)
    nan = torch.isnan(out.cpu())
    assert nan[0, 8:, 48:64].all() and nan.sum() == 8 * 16


@pytest.mark.parametrize("hq,hk,kbn", [(16, 2, 4), (16, 1, 16), (8, 4, 1), (24, 1, 7), (64, 8, 40)])
@pytest.mark.parametrize("splits", [-1, 1, 4])
def test_sparse_decode(hq, hk, kbn, splits):
    import msa_for_sail as msa
    b = Batch(kbn, [1, 3, 1, 2], [5600, 900, 60, 129], hq, hk)
    blocks = b.blocks(kbn)
    blocks[0, 0] = -1                                           # a row that selects nothing
    q, k, v, table = b.cuda()
    lse = torch.empty(b.T, hq, device=DEV)
    wide = torch.full((b.T, hk, kbn + 5), 7, dtype=torch.int32, device=DEV)
    wide[..., :kbn] = blocks.to(DEV)
    out, _ = msa.fmha_sail(q, k, v, b.plan(kv_block_num=kbn, num_kv_splits=splits), kv_indices=table, kv_block_indexes=wide[..., :kbn], lse=lse)
    ref.check_attention(out, lse, b.want(blocks=blocks), P_F16, f"{hq}/{hk} top {kbn}")
    assert (out[0, :hq // hk] == 0).all()


@pytest.mark.parametrize("case", ["dense", "mixed", "sparse", "mha"])
def test_prefill_runs_on_the_unpacked_pages(case):
    import msa_for_sail as msa
    qo, kv = ([200, 1, 130], [333, 700, 130]) if case != "sparse" else ([300], [900])
    hq, hk = (4, 4) if case == "mha" else (8, 2)
    b = Batch(21, qo, kv, hq, hk, q_dtype=torch.float8_e4m3fn if case == "dense" else torch.bfloat16)
    q, k, v, table = b.cuda()
    lse = torch.empty(b.T, hq, device=DEV)
    ks = torch.rand(hk, device=DEV) + 0.5
    kw, want = {}, dict(k_scale=ks)
    if case == "sparse":
        blocks = b.blocks(4)
        kw, want = dict(kv_block_indexes=blocks.to(DEV)), dict(k_scale=ks, blocks=blocks)
        plan = b.plan(kv_block_num=4)
        assert plan[3]["sparse_tc_preferred"]
    else:
        plan = b.plan(given=case != "mha")
    # a table that is longer than its use, with entries that are no pages behind the last one
    table = torch.cat([table, torch.tensor([-1, 10 ** 6], dtype=torch.int32, device=DEV)])
    out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table, k_scale=ks, lse=lse, **kw)
    ref.check_attention(out, lse, b.want(**want), P_BF16, case)


def test_decode_first_batches_are_split():
    import msa_for_sail as msa
    b = Batch(22, [1, 1, 1, 300], [400, 129, 77, 500], 16, 2)
    q, k, v, table = b.cuda()
    plan = b.plan(split_prefill_decode=True)
    assert plan[0]
    out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table)
    ref.check_attention(out, None, b.want(), P_BF16, "split")


@pytest.mark.parametrize("qo,kv,output_o", [([1, 1], [300, 900], False), ([2, 40], [300, 450], True)])
def test_scores_of_pages(qo, kv, output_o):
    import msa_for_sail as msa
    b = Batch(23, qo, kv, 4, 2)
    q, k, v, table = b.cuda()
    out, ms = msa.fmha_sail(q, k, v if output_o else None, b.plan(output_maxscore=True), kv_indices=table, output_o=output_o) if output_o else \
        msa.fmha_sail(q, k, k, b.plan(output_maxscore=True), kv_indices=table, output_o=False)
    values = ref.kv4_values(b.k).nan_to_num(0.0)
    t = 0
    for i, (n, keys) in enumerate(zip(qo, kv)):
        pages = b.table[b.indptr[i]:b.indptr[i + 1]].long()
        for j in range(n):
            see = min(keys, j + b.offsets[i] + 1)
            for h in range(4):
                x = values[pages, h // 2].reshape(-1, 128)[:see] @ b.q[t, h].double()
                for pg in range(ms.shape[1]):
                    part = x[pg * 128:(pg + 1) * 128]
                    got = float(ms[h, pg, t])
                    assert got == -float("inf") if not len(part) else abs(got - float(part.max())) <= 1e-3 * max(1.0, abs(float(part.max())))
            t += 1
    if output_o:
        ref.check_attention(out, None, b.want(), P_BF16, "with scores")


def test_scales_of_one_head_in_a_graph():
    """Scales stay on the device, also where there is one KV head or one value for all heads: nothing is read back."""
    import msa_for_sail as msa
    for hk in (1, 2):
        b = Batch(61, [1, 1], [300, 200], 8 * hk, hk)
        q, k, v, table = b.cuda()
        plan, ks, vs = b.plan(num_kv_splits=2), torch.tensor([0.5], device=DEV), torch.tensor([3.0], device=DEV)
        msa.fmha_sail(q, k, v, plan, kv_indices=table, k_scale=ks, v_scale=vs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table, k_scale=ks, v_scale=vs)
        vs.fill_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        ref.check_attention(out, None, b.want(k_scale=ks.expand(hk), v_scale=vs.expand(hk)), P_F16, f"{hk} heads")


@pytest.mark.parametrize("rows", [1, 4])
def test_a_reported_timeout_stops_the_tensor_core_kernel(rows):
    """While the status word is set, the kernel with waits does not start; once it is cleared it gives the right result."""
    import msa_for_sail as msa
    from msa_for_sail import api
    b = Batch(62, [rows, rows], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    plan = b.plan(num_kv_splits=1)
    out = torch.full((b.T, 16, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    api._status_word(q.device).fill_(1)
    msa.fmha_sail(q, k, v, plan, kv_indices=table, out=out)
    torch.cuda.synchronize()
    if rows * 8 > 16:
        assert (out == 7.0).all()
    assert api.last_status() == 1 and api.last_status() == 0
    msa.fmha_sail(q, k, v, plan, kv_indices=table, out=out)
    ref.check_attention(out, None, b.want(), P_F16, "after the status was cleared")


@pytest.mark.parametrize("sparse", [False, True])
def test_planned_and_run_in_a_graph(sparse):
    """graph_safe plan and call in one graph; lengths, table and selection change between replays; padded rows are left alone by nobody."""
    import msa_for_sail as msa
    hq, hk, B, most = 16, 2, 4, 1000
    b = Batch(31, [1] * B, [most] * B, hq, hk)
    q, k, v, table = b.cuda()
    ql, kl, off = (torch.full((B,), x, dtype=torch.int32, device=DEV) for x in (1, most, -1))
    kbn = 3
    ws = msa.allocate_graph_workspace(B, hq, num_kv_heads=hk, page_size=128, num_kv_splits=2, kv_block_num=kbn if sparse else -1)
    sel = torch.zeros(B, hk, kbn, dtype=torch.int32, device=DEV)
    lse = torch.empty(B, hq, device=DEV)

    def step():
        plan = msa.fmha_sail_plan(ql, kl, hq, num_kv_heads=hk, page_size=128, kv_block_num=kbn if sparse else -1, num_kv_splits=2, graph_safe=True,
                                  max_total_q=B, max_qo_len_override=1, qo_len_uniform_override=True, max_kv_len_override=most, qo_offset=off,
                                  given_workspace=ws, use_kv4_cache=True)
        return msa.fmha_sail(q, k, v, plan, kv_indices=table, lse=lse, **(dict(kv_block_indexes=sel) if sparse else {}))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed, kv in ((1, [1, 128, 555, 1000]), (2, [1000, 999, 130, 0]), (3, [127, 129, 1, 256])):
        n = Batch(31 + seed, [1] * B, kv, hq, hk, extra_pages=32 - sum(-(-x // 128) for x in kv) + 2)
        n.q = b.q
        blocks = n.blocks(kbn)
        k.copy_(n.k.to(DEV)); v.copy_(n.v.to(DEV)); kl.copy_(torch.tensor(kv, dtype=torch.int32)); sel.copy_(blocks.to(DEV))
        table[:len(n.table)] = n.table.to(DEV)
        graph.replay()
        torch.cuda.synchronize()
        ref.check_attention(out, lse, n.want(blocks=blocks) if sparse else n.want(), P_F16, f"replay {seed}")


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("n", [1, 3])
def test_rows_behind_the_last_sequence(sparse, splits, n):
    """A padded batch of a graph-safe plan: the rows behind the last sequence stay as they were, or become empty rows in the merge of splits."""
    import msa_for_sail as msa
    qo, pad = [n, 1, 0], 4
    b = Batch(72, qo, [500, 130, 0], 16, 2)
    q, k, v, table = b.cuda()
    T = b.T + pad
    q = torch.cat([q, torch.ones(pad, 16, 128, dtype=torch.bfloat16, device=DEV)])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    blocks = torch.cat([b.blocks(3), torch.zeros(pad, 2, 3, dtype=torch.int32)])
    ws = msa.allocate_graph_workspace(3, 16, num_kv_heads=2, page_size=128, num_kv_splits=2, kv_block_num=3 if sparse else -1, max_qo_len=n + 2)
    plan = msa.fmha_sail_plan(i32(qo), i32(b.kv), 16, num_kv_heads=2, page_size=128, kv_block_num=3 if sparse else -1, num_kv_splits=splits,
                              graph_safe=True, max_total_q=T, max_qo_len_override=n, qo_len_uniform_override=False, max_kv_len_override=600,
                              qo_offset=i32([-1] * 3), given_workspace=ws, use_kv4_cache=True)
    out, lse = torch.full((T, 16, 128), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((T, 16), 7.0, device=DEV)
    msa.fmha_sail(q, k, v, plan, kv_indices=table, out=out, lse=lse, **(dict(kv_block_indexes=blocks.to(DEV)) if sparse else {}))
    ref.check_attention(out[:b.T], lse[:b.T], b.want(**(dict(blocks=blocks[:b.T]) if sparse else {})), P_F16, "real rows")
    if plan[3]["num_kv_splits"] == 1:
        assert (out[b.T:] == 7).all() and (lse[b.T:] == 7).all()
    else:
        assert (out[b.T:] == 0).all() and torch.isinf(lse[b.T:]).all()


def test_two_streams_share_a_plan():
    """The partials of a call are its own: one plan may run on two streams at the same time."""
    import msa_for_sail as msa
    b = Batch(41, [1] * 6, [4000] * 6, 16, 2)
    q, k, v, table = b.cuda()
    q2 = q.flip(0).contiguous()
    plan = b.plan(num_kv_splits=6)
    want = [msa.fmha_sail(x, k, v, plan, kv_indices=table)[0].clone() for x in (q, q2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for s, x in zip(streams, (q, q2)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(msa.fmha_sail(x, k, v, plan, kv_indices=table)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_runs_are_repeatable():
    import msa_for_sail as msa
    b = Batch(42, [2] * 8, [1500, 3, 700, 128, 129, 2000, 999, 40], 64, 4)
    q, k, v, table = b.cuda()
    plan = b.plan()
    first = msa.fmha_sail(q, k, v, plan, kv_indices=table)[0]
    for _ in range(10):
        assert torch.equal(msa.fmha_sail(q, k, v, plan, kv_indices=table)[0], first)


def test_step_of_a_serving_engine():
    """Page tables, norm, rotation and append, page selection and attention of growing sequences, in one graph: prompts first, then tokens
    one by one, against attention over what the cache should hold."""
    import msa_for_sail as msa
    hq, hk, B, most = 16, 2, 3, 700
    g = _gen(77)
    rope = msa.rope_plan(64, base=5e5)
    inv = [5e5 ** (-2 * i / 64) for i in range(32)]
    kc, vc = msa.allocate_kv4_cache(24, hk)
    width = -(-most // 128)
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    held, free, num_free = i32([0] * B), torch.randperm(24, generator=g).to(torch.int32).to(DEV), i32([24])
    w = (torch.rand(128, generator=g) + 0.5).to(DEV)
    scales = dict(k_scale=torch.full((hk,), 0.5, device=DEV), v_scale=torch.full((hk,), 0.25, device=DEV))
    history = [[] for _ in range(B)]                            # (k, v) of each sequence as bf16

    def append(x, tabs, T):
        q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        return msa.qk_norm_rope(q, k, tabs["positions"][:T], rope, v=v, q_weight=w, k_weight=w, k_cache=kc, v_cache=vc, slot_map=tabs["slot_map"][:T], **scales)[0]

    def remember(x, pos, lens):
        k, _ = ref.norm_rope(x[:, hq:hq + hk], pos[None], inv, [32], False, w)
        t = 0
        for b, n in enumerate(lens):
            history[b].append((k[t:t + n].float().to(torch.bfloat16), x[t:t + n, hq + hk:].cpu()))
            t += n

    def held_values(which):
        """What 4 bits hold of every sequence, as pages in order."""
        pages = []
        for b in range(B):
            x = torch.cat([h[which] for h in history[b]])
            codes, sb = ref.kv4_encode(x, scales["v_scale" if which else "k_scale"].cpu())
            n = -(-len(x) // 128)
            tile = torch.zeros(n, hk, 128 * 72, dtype=torch.uint8)
            at = torch.arange(len(x))
            tile[:, :, :8192].view(n, hk, 128, 64)[at // 128, :, at % 128] = codes
            tile[:, :, 8192:].view(n, hk, 128, 8)[at // 128, :, at % 128] = sb
            pages.append(ref.kv4_values(tile.view(n, hk, 128, 72)))
        return torch.cat(pages)

    def check(out, q, ql, kl, p_rounding, what):
        need = [-(-n // 128) for n in kl]
        want = ref.attention(q, held_values(0), held_values(1), torch.arange(sum(need)), [sum(need[:i]) for i in range(B + 1)], ql, kl,
                             [a - b for a, b in zip(kl, ql)], k_scale=scales["k_scale"], v_scale=scales["v_scale"])
        ref.check_attention(out, None, want, p_rounding, what)

    # prompts
    ql = kl = [300, 128, 77]
    T = sum(ql)
    x = torch.randn(T, hq + 2 * hk, 128, generator=g).to(torch.bfloat16).to(DEV)
    tabs = msa.paged_kv_tables(i32(ql), i32(kl), table, held, free, num_free, max_total_q=T, num_held_out=held, num_free_out=num_free)
    q = append(x, tabs, T)
    plan = msa.fmha_sail_plan(torch.tensor(ql), torch.tensor(kl), hq, num_kv_heads=hk, page_size=128, use_kv4_cache=True)
    out, _ = msa.fmha_sail(q, kc, vc, plan, kv_indices=tabs["kv_indices"], **scales)
    remember(x, tabs["positions"], ql)
    assert int(tabs["num_missing"]) == 0
    check(out, q, ql, kl, P_BF16, "prompts")

    # tokens: one graph for every step
    ql_d, kl_d, off = i32([1] * B), i32(kl), i32([-1] * B)
    x_d = torch.empty(B, hq + 2 * hk, 128, dtype=torch.bfloat16, device=DEV)
    ws = msa.allocate_graph_workspace(B, hq, num_kv_heads=hk, page_size=128, num_kv_splits=3)

    def step():
        kl_d.add_(1)
        tabs = msa.paged_kv_tables(ql_d, kl_d, table, held, free, num_free, max_total_q=B, num_held_out=held, num_free_out=num_free)
        q = append(x_d, tabs, B)
        plan = msa.fmha_sail_plan(ql_d, kl_d, hq, num_kv_heads=hk, page_size=128, num_kv_splits=3, graph_safe=True, max_total_q=B, max_qo_len_override=1,
                                  qo_len_uniform_override=True, max_kv_len_override=most, qo_offset=off, given_workspace=ws, use_kv4_cache=True)
        return msa.fmha_sail(q, kc, vc, plan, kv_indices=tabs["kv_indices"], **scales)[0], q, tabs

    x_d.zero_()
    state = [t.clone() for t in (kl_d, held, num_free, table, kc, vc)]
    step()                                                      # warm up, and put everything back
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, q, tabs = step()
    for t, was in zip((kl_d, held, num_free, table, kc, vc), state):
        t.copy_(was)
    for i in range(60):
        x = torch.randn(B, hq + 2 * hk, 128, generator=g).to(torch.bfloat16)
        x_d.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        kl = [n + 1 for n in kl]
        assert tabs["positions"].tolist() == [n - 1 for n in kl]
        remember(x, tabs["positions"], [1] * B)
        if i % 20 == 19 or i == 0:
            check(out, q, [1] * B, kl, P_F16, f"token {i}")
    assert num_free.tolist() == [24 - sum(-(-n // 128) for n in kl)]


def _poison(b, seq, key, head, block, which=("k", "v")):
    page = int(b.table[b.indptr[seq] + key // 128])
    for c in which:
        getattr(b, c).view(b.k.shape[0], b.hk, -1)[page, head, 128 * 64 + 8 * (key % 128) + block] = 0x7F


@pytest.mark.parametrize("n,hq,hk", [(1, 16, 2), (1, 32, 2), (2, 8, 2), (4, 8, 2), (4, 16, 2), (16, 8, 2), (16, 16, 2)])
@pytest.mark.parametrize("splits", [1, 2])
def test_not_a_number_in_places_that_rows_do_not_see(n, hq, hk, splits):
    """Keys behind a row's last one may be NaN, behind the last row's (stale places below the sequence's length) and between the rows'
    (tokens of the same step): only rows that see such a key have it, in the 16 elements that share its scale."""
    import msa_for_sail as msa
    kv = [300, 128 + n // 2, 500]
    b = Batch(70 + n, [n] * 3, kv, hq, hk, offsets=[300 - n - 90, 128 + n // 2 - n, 500 - n])
    q, k, v, table = b.cuda()
    lse = torch.empty(b.T, hq, device=DEV)
    want = b.want()
    for key in range(210, 300):
        for block in range(8):
            _poison(b, 0, key, 0, block)
            _poison(b, 0, key, 1, block)
    hit = {1: kv[1] - 1, 2: 500 - max(1, n // 2)}               # the last token, and one in the middle
    for seq, key in hit.items():
        _poison(b, seq, key, 1, 3, "v")
    q, k, v, table = b.cuda()
    out, _ = msa.fmha_sail(q, k, v, b.plan(num_kv_splits=splits), kv_indices=table, lse=lse)
    nan = torch.zeros(b.T, hq, 128, dtype=torch.bool)
    for seq, key in hit.items():
        for i in range(n):
            if i + b.offsets[seq] >= key:
                nan[seq * n + i, hq // hk:, 48:64] = True
    assert nan.any() and torch.equal(torch.isnan(out.cpu()), nan)
    ref.check_attention(torch.where(nan.to(DEV), 0.0, out), lse, (torch.where(nan, 0.0, want[0]),) + tuple(want[1:]), P_F16, f"{n} tokens")


def test_offsets_past_every_key():
    """An offset that no sum may add to: every row sees every key."""
    import msa_for_sail as msa
    for n, hq in ((1, 16), (4, 32)):
        b = Batch(71, [n, n], [300, 200], hq, 2, offsets=[1000, 1000])
        q, k, v, table = b.cuda()
        far = torch.full((2,), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
        out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table, q_offset_override=far)
        ref.check_attention(out, None, b.want(), P_F16, f"{n} tokens")


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("sparse", [False, True])
def test_a_table_shorter_than_the_lengths(rows, sparse):
    """Lengths on the device may outgrow a table: the places behind its end are its last page, nothing behind it is read.  An empty one has
    no keys."""
    import msa_for_sail as msa
    from msa_for_sail import api
    b = Batch(63, [rows], [600], 16, 2)
    q, k, v, table = b.cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    sel = i32([0, 2, 4]).expand(rows, 2, 3).contiguous()
    ws = msa.allocate_graph_workspace(1, 16, num_kv_heads=2, page_size=128, num_kv_splits=2, kv_block_num=3 if sparse else -1, max_qo_len=rows)
    plan = msa.fmha_sail_plan(i32([rows]), i32([600]), 16, num_kv_heads=2, page_size=128, kv_block_num=3 if sparse else -1, num_kv_splits=2,
                              graph_safe=True, max_total_q=rows, max_qo_len_override=rows, qo_len_uniform_override=True, max_kv_len_override=700,
                              qo_offset=i32([600 - rows]), given_workspace=ws, use_kv4_cache=True)
    blocks = dict(kv_block_indexes=sel) if sparse else {}
    short = table[:2].clone()
    got = msa.fmha_sail(q, k, v, plan, kv_indices=short, **blocks)[0].clone()
    api.last_status()                                           # (the build with bounds checks reports the places past the end)
    b.table[2:] = b.table[1]
    lse = torch.empty(rows, 16, device=DEV)
    again, _ = msa.fmha_sail(q, k, v, plan, kv_indices=b.table.to(DEV), lse=lse, **blocks)
    assert torch.equal(got, again)
    ref.check_attention(got, lse, b.want(**(dict(blocks=sel.cpu()) if sparse else {})), P_F16, "short table")
    none, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table[:0].clone(), lse=lse, **blocks)
    assert (none == 0).all() and torch.isinf(lse).all()


def test_a_plan_keeps_no_pointer():
    """The tensors of a plan may be replaced between calls."""
    import msa_for_sail as msa
    b = Batch(64, [1, 1], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    plan = b.plan(num_kv_splits=1)
    msa.fmha_sail(q, k, v, plan, kv_indices=table)
    b.kv = [300, 140]
    b.offsets = [299, 139]
    for name, value in (("kv_segment_lens", b.kv), ("qo_offset", b.offsets)):
        plan[3][name] = torch.tensor(value, dtype=torch.int32, device=DEV)
    out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table)
    ref.check_attention(out, None, b.want(), P_F16, "replaced")


def test_two_streams_share_a_plan_of_a_prompt():
    """The copies and workspaces of the path over unpacked pages belong to the call."""
    import msa_for_sail as msa
    b = Batch(65, [300], [900], 8, 2)
    q, k, v, table = b.cuda()
    q2, blocks = q.flip(0).contiguous(), b.blocks(4).to(DEV)
    plan = b.plan(kv_block_num=4)
    want = [msa.fmha_sail(x, k, v, plan, kv_indices=table, kv_block_indexes=blocks)[0].clone() for x in (q, q2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for s, x in zip(streams, (q, q2)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(msa.fmha_sail(x, k, v, plan, kv_indices=table, kv_block_indexes=blocks)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_first_call_of_a_process_inside_a_capture(monkeypatch):
    """The word that kernels report to is not made inside a capture, where it would belong to the graph's memory."""
    import msa_for_sail as msa
    from msa_for_sail import api
    b = Batch(66, [1, 1], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    plan = b.plan(num_kv_splits=1)
    msa.fmha_sail(q, k, v, plan, kv_indices=table)
    torch.cuda.synchronize()
    monkeypatch.setattr(api, "_STATUS", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table)
    assert not api._STATUS
    graph.replay()
    torch.cuda.synchronize()
    ref.check_attention(out, None, b.want(), P_F16, "captured")


def test_checked_inputs_and_the_line_of_a_call(monkeypatch, capfd):
    import msa_for_sail as msa
    from msa_for_sail import api
    monkeypatch.setattr(api, "_SHOW_PARAMS", True)
    b = Batch(68, [1, 2], [300, 700], 16, 2)
    q, k, v, table = b.cuda()
    out, _ = msa.fmha_sail(q, k, v, b.plan(), kv_indices=table, check_input_valid=True)
    ref.check_attention(out, None, b.want(), P_F16, "checked")
    assert "[MSA] --format=" in capfd.readouterr().out
    bad = table.clone()
    bad[1] = 10 ** 6
    with pytest.raises(AssertionError, match="outside"):
        msa.fmha_sail(q, k, v, b.plan(), kv_indices=bad, check_input_valid=True)
    blocks = b.blocks(3)
    out, _ = msa.fmha_sail(q, k, v, b.plan(kv_block_num=3), kv_indices=table, kv_block_indexes=blocks.to(DEV), check_input_valid=True)
    ref.check_attention(out, None, b.want(blocks=blocks), P_F16, "checked selection")


@pytest.mark.parametrize("hq,hk", [(256, 1), (130, 1), (144, 1)])
def test_more_than_128_heads_to_a_kv_head(hq, hk):
    """A dense plan has no items for a token of so many heads, whatever the cache; where pages are selected they are groups of 16 rows."""
    import msa_for_sail as msa
    b = Batch(69, [1, 1], [300, 200], hq, hk)
    q, k, v, table = b.cuda()
    with pytest.raises(RuntimeError, match="bad argument"):
        b.plan()
    blocks = b.blocks(2)
    out, _ = msa.fmha_sail(q, k, v, b.plan(kv_block_num=2), kv_indices=table, kv_block_indexes=blocks.to(DEV))
    ref.check_attention(out, None, b.want(blocks=blocks), P_F16, f"{hq} heads, selected")


def test_strides_the_kernels_read():
    """Queries inside a wider buffer, a selection whose rows are apart, a cache whose pages hold more than keys and values."""
    import msa_for_sail as msa
    for n, hq in ((1, 16), (2, 32)):
        b = Batch(70, [n] * 3, [300, 129, 700], hq, 2)
        q, k, v, table = b.cuda()
        wide = torch.full((b.T, hq + 5, 128), torch.nan, dtype=torch.bfloat16, device=DEV)
        wide[:, 2:2 + hq] = q
        big = torch.full((k.shape[0], 5, 128, 72), 0x7F, dtype=torch.uint8, device=DEV)
        big[:, 1:3], big[:, 3:5] = k, v
        out = torch.full((b.T, hq + 3, 128), 7.0, dtype=torch.bfloat16, device=DEV)
        msa.fmha_sail(wide[:, 2:2 + hq], big[:, 1:3], big[:, 3:5], b.plan(), kv_indices=table, out=out[:, 1:1 + hq])
        ref.check_attention(out[:, 1:1 + hq], None, b.want(), P_F16, f"{n} tokens")
        assert (out[:, 0] == 7).all() and (out[:, 1 + hq:] == 7).all()


def test_refusals_of_tables_and_offsets():
    import msa_for_sail as msa
    b = Batch(67, [1, 1], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    plan = b.plan()
    with pytest.raises(ValueError, match="kv_indices must have the 5 pages"):
        msa.fmha_sail(q, k, v, plan, kv_indices=table[:4].clone())
    with pytest.raises(ValueError, match="q_offset_override must be"):
        msa.fmha_sail(q, k, v, plan, kv_indices=table, q_offset_override=torch.zeros(1, dtype=torch.int32, device=DEV))


def test_refusals():
    import msa_for_sail as msa
    b = Batch(51, [1, 1], [300, 200], 16, 2)
    q, k, v, table = b.cuda()
    plan = b.plan()
    run = lambda q=q, k=k, v=v, plan=plan, table=table, **kw: msa.fmha_sail(q, k, v, plan, kv_indices=table, **kw)
    run()
    with pytest.raises(RuntimeError):
        run(q=b.q)
    lens = torch.tensor([1, 1], dtype=torch.int32), torch.tensor([300, 200], dtype=torch.int32)
    bad = [lambda: run(table=None), lambda: run(table=table.long()), lambda: run(table=table.cpu()), lambda: run(k=k.cpu()),
           lambda: run(k=k.view(k.shape[0], 2, 9216)), lambda: run(k=k[:, :, :64]), lambda: run(v=v[:3]), lambda: run(v=None),
           lambda: run(v=v.view(torch.int8)), lambda: run(q=q.half()), lambda: run(q=q[..., :64]), lambda: run(q=q[:1]), lambda: run(k=k[:0], v=v[:0]),
           lambda: run(k=k[:, :1], v=v[:, :1]), lambda: run(q=q[:, :5]),
           lambda: run(kv_block_indexes=torch.zeros(2, 2, 4, dtype=torch.int32, device=DEV)),
           lambda: run(plan=b.plan(kv_block_num=4)), lambda: run(plan=b.plan(kv_block_num=4), kv_block_indexes=torch.zeros(2, 1, 4, dtype=torch.int32, device=DEV)),
           lambda: run(plan=msa.fmha_sail_plan(*lens, 16, num_kv_heads=2, page_size=64)),
           lambda: run(k=torch.empty(k.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(k.shape))]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, AssertionError)):
            f()
            print("not refused:", i)


@pytest.mark.parametrize("hq", [8, 16])
def test_lists_of_fewer_pages_than_stages(hq):
    """One to three pages an item, pages that are not in a cache of the device, many items at once."""
    import msa_for_sail as msa
    kv = [1 + 37 * i % 384 for i in range(600)]
    b = Batch(81, [1] * len(kv), kv, hq, 1)
    q, k, v, table = b.cuda()
    plan, want = b.plan(num_kv_splits=1), b.want()
    flush = torch.zeros(1 << 28, dtype=torch.uint8, device=DEV)
    for _ in range(8):
        flush.add_(1)
        out, _ = msa.fmha_sail(q, k, v, plan, kv_indices=table)
        ref.check_attention(out, None, want, P_F16, f"{hq} rows")
