"""paged_kv_tables against a plain loop over the requests."""
import random

import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _case(seed, batch, longest, page_size, tokens, pool_extra=5, width_extra=0):
    rng = random.Random(seed)
    kv = [rng.choice([0, 1, page_size - 1, page_size, page_size + 1, rng.randint(0, longest), longest]) for _ in range(batch)]
    kv = [min(n, longest) for n in kv]
    ql = [rng.choice([0, min(n, 1), min(n, tokens), n if rng.random() < 0.1 else min(n, tokens)]) for n in kv]
    need = [-(-n // page_size) for n in kv]
    held = [-(-(n - t) // page_size) for t, n in zip(ql, kv)]
    pool = list(range(sum(need) + pool_extra))
    rng.shuffle(pool)
    width = max(1, -(-longest // page_size) + width_extra)
    table, at = [], 0
    for h in held:
        table.append([pool[at + i] if i < h else -7 for i in range(width)])
        at += h
    return ql, kv, table, held, pool[at:]


def _run(ql, kv, table, held, free, num_free, max_q, max_pages, page_size, **kw):
    import msa_for_sail as msa
    t = _i32(table).reshape(len(ql), -1)
    more = {} if held is None else dict(num_held=_i32(held), free_pages=_i32(free), num_free=_i32([num_free]))
    r = msa.paged_kv_tables(_i32(ql), _i32(kv), t, max_total_q=max_q, max_total_pages=max_pages, page_size=page_size, **more, **kw)
    torch.cuda.synchronize()
    return r, t


def _check(ql, kv, table, held, free, num_free, max_q, max_pages, page_size):
    r, t = _run(ql, kv, table, held, free, num_free, max_q, max_pages, page_size)
    want = [list(row) for row in table]
    flat, indptr, slots, pos, new_held, left, missing = ref.page_tables(ql, kv, want, held, free, num_free, max_q, max_pages, page_size)
    assert t.tolist() == want
    assert r["kv_indices"].tolist() == flat
    assert r["kv_page_indptr"].tolist() == indptr
    assert r["slot_map"].tolist() == slots
    assert r["positions"].tolist() == pos
    assert r["num_missing"].tolist() == [missing]
    if held is not None:
        assert r["num_held"].tolist() == new_held and r["num_free"].tolist() == [left]
    else:
        assert "num_held" not in r


@pytest.mark.parametrize("batch,longest,page_size,tokens", [
    (1, 1, 128, 1), (1, 100000, 128, 1), (7, 700, 128, 3), (33, 300, 16, 5), (1023, 900, 128, 2), (1024, 40, 1, 2), (1025, 900, 64, 4),
    (2500, 5000, 128, 3), (3, 20000, 7, 20000)])
@pytest.mark.parametrize("alloc", [True, False])
def test_against_a_loop(batch, longest, page_size, tokens, alloc):
    ql, kv, table, held, free = _case(batch + longest, batch, longest, page_size, tokens)
    total = sum(-(-n // page_size) for n in kv)
    if not alloc:
        r = random.Random(1)
        table = [[r.randrange(1000) for _ in row] for row in table]
    _check(ql, kv, table, held if alloc else None, free if alloc else None, len(free) if alloc else 0, sum(ql) + 3, total + 2, page_size)


@pytest.mark.parametrize("short", ["stack", "row", "pages", "tokens", "count"])
@pytest.mark.parametrize("batch", [5, 600])
def test_what_does_not_fit_is_counted(short, batch):
    ql, kv, table, held, free = _case(11, batch, 900, 128, 200)
    total, num_free = sum(-(-n // 128) for n in kv), len(free)
    max_q, max_pages = sum(ql), total
    if short == "stack":
        num_free = 2
    elif short == "row":
        table = [row[:4] for row in table]
    elif short == "pages":
        max_pages = total // 2
    elif short == "tokens":
        max_q = sum(ql) // 2
    else:
        num_free, free = 5000, free[:3]                          # a count above the stack's size is cut to it
    r, t = _run(ql, kv, table, held, free, num_free, max_q, max_pages, 128)
    want = [list(row) for row in table]
    flat, indptr, slots, pos, new_held, left, missing = ref.page_tables(ql, kv, want, held, free, min(num_free, len(free)), max_q, max_pages, 128)
    assert missing > 0 and r["num_missing"].tolist() == [missing]
    assert t.tolist() == want and r["kv_indices"].tolist() == flat and r["slot_map"].tolist() == slots and r["positions"].tolist() == pos
    assert r["num_held"].tolist() == new_held and r["num_free"].tolist() == [left]


def test_empty_batch_and_sizes_of_zero():
    import msa_for_sail as msa
    r = msa.paged_kv_tables(_i32([]), _i32([]), torch.empty(0, 4, dtype=torch.int32, device="cuda"), max_total_q=3, max_total_pages=2)
    assert r["kv_page_indptr"].tolist() == [0] and r["slot_map"].tolist() == [-1] * 3 and r["kv_indices"].tolist() == [-1] * 2
    r = msa.paged_kv_tables(_i32([0, 0]), _i32([0, 0]), torch.empty(2, 0, dtype=torch.int32, device="cuda"), max_total_q=0)
    assert r["kv_page_indptr"].tolist() == [0, 0, 0] and r["kv_indices"].numel() == 0 and r["num_missing"].tolist() == [0]


def test_steps_in_place_inside_a_graph():
    """Counts updated in place, outputs at fixed addresses: every replay is one more step of growing requests."""
    import msa_for_sail as msa
    B, width = 40, 9
    kv, ql = [100 + 20 * i for i in range(B)], [0] * B
    table = torch.full((B, 16), -7, dtype=torch.int32, device="cuda")[:, :width]          # rows that lie apart
    held, free, num_free = _i32([0] * B), torch.randperm(B * width, device="cuda").to(torch.int32), _i32([B * width])
    q_dev, k_dev = _i32(ql), _i32(kv)
    a = dict(max_total_q=200, num_held_out=held, num_free_out=num_free)
    first = msa.paged_kv_tables(q_dev, k_dev, table, held, free, num_free, **a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = msa.paged_kv_tables(q_dev, k_dev, table, held, free, num_free, out=first, **a)
    want, h, n = [[-7] * width for _ in range(B)], [0] * B, B * width
    stack = free.tolist()
    _, _, _, _, h, n, _ = ref.page_tables(ql, kv, want, h, stack, n, 200, B * width, 128)
    assert held.tolist() == h and num_free.tolist() == [n]
    rng = random.Random(3)
    for _ in range(5):
        ql = [rng.randint(0, 5) for _ in range(B)]
        kv = [min(k + q, width * 128) for k, q in zip(kv, ql)]
        q_dev.copy_(_i32(ql)); k_dev.copy_(_i32(kv))
        graph.replay()
        torch.cuda.synchronize()
        flat, indptr, slots, pos, h, n, missing = ref.page_tables(ql, kv, want, h, stack, n, 200, B * width, 128)
        assert missing == 0 and table.tolist() == want and held.tolist() == h and num_free.tolist() == [n]
        assert r["kv_indices"].tolist() == flat and r["kv_page_indptr"].tolist() == indptr
        assert r["slot_map"].tolist() == slots and r["positions"].tolist() == pos


def test_slots_that_pass_32_bits():
    """A page whose tokens have no 32-bit slot gives -1, which nothing is written to."""
    edge = 2 ** 31 // 128
    r, _ = _run([3, 2], [3, 130], [[edge, 0], [edge - 1, 7]], None, None, 0, 6, 4, 128)
    assert r["slot_map"].tolist() == [-1, -1, -1, 7 * 128, 7 * 128 + 1, -1]
    r, _ = _run([2], [128], [[edge - 1]], None, None, 0, 2, 1, 128)
    assert r["slot_map"].tolist() == [2 ** 31 - 2, 2 ** 31 - 1]


def test_refusals():
    import msa_for_sail as msa
    q, k, t = _i32([1, 1]), _i32([5, 6]), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    ok = dict(max_total_q=2)
    msa.paged_kv_tables(q, k, t, **ok)
    for bad in [lambda: msa.paged_kv_tables(q.cpu(), k, t, **ok)]:
        with pytest.raises(RuntimeError):
            bad()
    for bad in [lambda: msa.paged_kv_tables(q.long(), k, t, **ok),
                lambda: msa.paged_kv_tables(q, k.cpu(), t, **ok),
                lambda: msa.paged_kv_tables(q, k[:1], t, **ok),
                lambda: msa.paged_kv_tables(q, k, t[:1], **ok),
                lambda: msa.paged_kv_tables(q, k, t.t(), **ok),
                lambda: msa.paged_kv_tables(q, k, t[:1].expand(2, 4), **ok),
                lambda: msa.paged_kv_tables(q, k, t, max_total_q=-1),
                lambda: msa.paged_kv_tables(q, k, t, page_size=0, **ok),
                lambda: msa.paged_kv_tables(q, k, t, num_held=q, **ok),
                lambda: msa.paged_kv_tables(q, k, t, num_held_out=q, **ok),
                lambda: msa.paged_kv_tables(q, k, t, q, _i32([1]), _i32([1, 2]), **ok),
                lambda: msa.paged_kv_tables(q, k, t, out=msa.paged_kv_tables(q, k, t, max_total_q=3), **ok)]:
        with pytest.raises(ValueError):
            bad()
