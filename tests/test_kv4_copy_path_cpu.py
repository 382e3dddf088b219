"""Arguments of attention over a 4-bit cache where it runs on bf16 copies (longer queries, page scores, pages that many tokens share): what is
refused, is refused before a page is copied.  CPU tensors stand in for those of a GPU; nothing is launched."""
import contextlib

import pytest
import torch


class Copied(Exception):
    """The call came as far as copying pages."""


@pytest.fixture
def api(monkeypatch):
    from msa_for_sail import api, cache

    def copied(*a, **kw):
        raise Copied
    monkeypatch.setattr(api, "_num_sms", lambda dev: 148)
    monkeypatch.setattr(cache, "_same_device", lambda *a, **kw: None)
    monkeypatch.setattr(cache, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(cache, "unpack_pages", copied)
    return api


# query tokens, keys, options of the plan, what the call adds
PATHS = {"prompt": ([200, 1], [300, 200], {}, {}), "scores": ([1, 1], [300, 200], dict(output_maxscore=True), dict(output_o=False)),
         "shared pages": ([300], [600], dict(kv_block_num=2), {}), "prompt of 9 tokens": ([9], [600], {}, {})}


def _call(api, path, table=None, **kw):
    qo, kv, opts, extra = PATHS[path]
    hq, hk = (64, 4) if path == "prompt of 9 tokens" else (16, 2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    plan = api._fmha_sail_plan(i32(qo), i32(kv), hq, hk, page_size=128, device="cpu", use_kv4_cache=True, **opts)
    q = torch.zeros(sum(qo), hq, 128, dtype=torch.bfloat16)
    k, v = (torch.zeros(9, hk, 128, 72, dtype=torch.uint8) for _ in range(2))
    table = torch.arange(5, dtype=torch.int32) if table is None else table
    args = dict(kv_block_indexes=None, q_offset_override=None, out=None, max_score=None, sm_scale=None, q_scale=None, k_scale=None, v_scale=None,
                o_scale=None, output_maxscore=True, output_o=True, check_input_valid=False, max_score_dtype=None, lse=None)
    if "kv_block_num" in opts:
        args["kv_block_indexes"] = torch.arange(opts["kv_block_num"], dtype=torch.int32).expand(sum(qo), hk, -1)
    return api._fmha_sail_kv4(q, k, v, plan, table, **{**args, **extra, **kw})


@pytest.mark.parametrize("path", list(PATHS))
def test_a_table_shorter_than_the_plan_is_refused(api, path):
    with pytest.raises(Copied):
        _call(api, path)
    for n in (4, 1, 0):
        with pytest.raises(ValueError, match="kv_indices must have the 5 pages"):
            _call(api, path, table=torch.arange(n, dtype=torch.int32))


def test_a_call_without_tokens_needs_no_table(api):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    plan = api._fmha_sail_plan(i32([0, 0]), i32([300, 200]), 16, 2, page_size=128, device="cpu", use_kv4_cache=True)
    k = torch.zeros(9, 2, 128, 72, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="needs CUDA tensors"):         # as far as the attention over the copies
        api._fmha_sail_kv4(torch.zeros(0, 16, 128, dtype=torch.bfloat16), k, k, plan, i32([]), *[None] * 9, True, True, False, None, None)


@pytest.mark.parametrize("path", list(PATHS))
def test_offsets_of_another_batch_are_refused(api, path):
    with pytest.raises(Copied):
        _call(api, path, q_offset_override=torch.zeros(len(PATHS[path][0]), dtype=torch.int32))
    for shape in [(len(PATHS[path][0]) + 1,), (0,), (len(PATHS[path][0]), 1)]:
        with pytest.raises(ValueError, match="q_offset_override must be"):
            _call(api, path, q_offset_override=torch.zeros(shape, dtype=torch.int32))


@pytest.mark.parametrize("path", list(PATHS))
def test_checked_inputs_are_those_of_the_caller(api, path):
    with pytest.raises(Copied):
        _call(api, path, check_input_valid=True)
    for bad in (9, -1, 10 ** 6):
        with pytest.raises(AssertionError, match="outside"):
            _call(api, path, table=torch.tensor([0, 1, bad, 3, 4], dtype=torch.int32), check_input_valid=True)


def test_an_empty_table_copies_nothing(api, monkeypatch):
    """Lengths of a device-made plan that an empty table cannot hold: the call goes on with sequences that have no keys."""
    seen = {}

    def run(q, k, v, plan, kv_indices, *a, **kw):
        seen.update(k=k, v=v, lens=plan["kv_segment_lens"], table=kv_indices)
        return None, None
    monkeypatch.setattr(api, "_fmha_sail", run)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    plan = api._fmha_sail_plan(i32([200]), i32([600]), 16, 2, page_size=128, device="cpu", use_kv4_cache=True)
    plan["_host"] = None                                        # as if the lengths had stayed on the device
    k = torch.zeros(9, 2, 128, 72, dtype=torch.uint8)
    api._fmha_sail_kv4(torch.zeros(200, 16, 128, dtype=torch.bfloat16), k, k, plan, i32([]), *[None] * 9, True, True, False, None, None)
    assert seen["k"].shape == seen["v"].shape == (1, 2, 128, 128) and seen["table"].tolist() == [0] and seen["lens"].tolist() == [0]
    assert plan["kv_segment_lens"].tolist() == [600]


@pytest.mark.parametrize("qo,kv,hq,hk", [([1] * 24, [20000] * 23 + [60000], 64, 4), ([1], [1 << 20], 64, 8), ([4] * 8, [20000] * 8, 64, 8), ([20] * 2, [9000] * 2, 16, 4)])
def test_plans_of_a_4_bit_cache_reserve_no_partials(api, qo, kv, hq, hk):
    """Its calls allocate their own: a plan holds none, and a workspace without room for any still gets the finer cut."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    make = lambda **kw: api._fmha_sail_plan(i32(qo), i32(kv), hq, hk, page_size=128, device="cpu", use_kv4_cache=True, **kw)
    free = make()
    assert free["num_kv_splits"] > 1 and free["workspace_o"] is None and free["workspace_lse"] is None
    last = max((t for t in free.values() if isinstance(t, torch.Tensor)), key=lambda t: t.data_ptr() + t.numel() * 4)
    first = min(t.data_ptr() for t in free.values() if isinstance(t, torch.Tensor))
    ws = torch.empty(last.data_ptr() + last.numel() * 4 - first, dtype=torch.uint8)
    given = make(given_workspace=ws)
    assert given["num_kv_splits"] == free["num_kv_splits"] and torch.equal(given["work"], free["work"])
    with pytest.raises(ValueError, match="too small"):
        make(given_workspace=ws[:1000])
