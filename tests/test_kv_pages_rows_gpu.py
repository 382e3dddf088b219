"""Rows of the block table that calls on pages name twice, or share."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _msa():
    import msa_for_sail
    return msa_for_sail


@pytest.mark.parametrize("parents,children,made,missing", [
    ([-1, 2], [5, 5], {5: 2}, 0),                               # a stale row number behind an entry that does nothing
    ([-1, -7, 2, -1, 0], [4, 5, 5, 5, 4], {5: 2, 4: 0}, 0),
    ([2, -1], [5, 5], {5: 2}, 0),
    ([2, -1, 0], [5, 5, 5], {5: 2}, 1),                         # named twice: the first has it
    ([-1], [5], {}, 0)])
def test_an_entry_without_a_parent_takes_no_child(parents, children, made, missing):
    P, page, width = 40, 16, 4
    kv = [20, 64, 41, 0, 0, 0]
    table = [[-1] * width for _ in kv]
    at = 0
    for b, n in enumerate(kv):
        for c in range(-(-n // page)):
            table[b][c] = at
            at += 1
    held = [-(-n // page) for n in kv]
    free = list(range(P - 1, at - 1, -1))
    num_free = len(free)
    shares = [0] * P
    want_table, want_held, want_kv = [list(r) for r in table], list(held), list(kv)
    for p, c in zip(parents, children):                         # in the order of the entries
        if made.get(c) == p and want_held[c] == 0:
            full, part = divmod(kv[p], page)
            for i in range(full):
                want_table[c][i] = table[p][i]
                shares[table[p][i]] += 1
            if part:
                num_free -= 1
                want_table[c][full] = free[num_free]
            want_held[c], want_kv[c] = held[p], kv[p]
    cache = torch.randint(0, 256, (P, page, 24), dtype=torch.uint8, device=DEV)
    want_cache = cache.clone()
    for c, p in made.items():
        if kv[p] % page:
            want_cache[want_table[c][kv[p] // page]] = cache[table[p][kv[p] // page]]
    t = dict(block_table=_i32(table), num_held=_i32(held), kv_lens=_i32(kv))
    stack, count, sh = _i32(free), _i32([len(free)]), _i32([0] * P)
    got = _msa().kv_pages_fork(*t.values(), _i32(parents), _i32(children), stack, count, sh, [cache], page)
    assert got.item() == missing and count.item() == num_free and sh.tolist() == shares
    assert t["block_table"].tolist() == want_table and t["num_held"].tolist() == want_held and t["kv_lens"].tolist() == want_kv
    assert torch.equal(cache, want_cache)
