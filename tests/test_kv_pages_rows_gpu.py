"""Rows of the block table that calls on pages name twice, or share."""
import random

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


def _cut(table, held, kv, free, num_free, shares, page, moving):
    """Rows cut back into a page that others hold, one after the other, after the pages behind them went back.  Returns (moves, num_free, left)."""
    P = len(shares)

    def into(b):
        col = max(kv[b], 0) // page
        return table[b][col] if kv[b] > 0 and kv[b] % page and col < held[b] else -1
    cut = [b for b in range(len(table)) if 0 <= into(b) < P and shares[into(b)] > 0]
    moves = []
    if moving:
        for b in cut:
            p = into(b)
            if shares[p] > 0 and num_free > 0:
                num_free -= 1
                shares[p] -= 1
                table[b][kv[b] // page] = free[num_free]
                moves.append((p, free[num_free], kv[b] % page))
    left = sum(0 <= into(b) < P and shares[into(b)] > 0 for b in cut)
    return moves, num_free, left


def _holders(rng, rows, width, page):
    """Rows that hold the same pages up to some column, each with more of its own: (table, held, lengths, free, shares, pages)."""
    table, held, kv, shares, at = [], [], [], {}, 0
    for b in range(rows):
        n = rng.randint(0, width)
        row = []
        if table and rng.random() < 0.7:
            other = rng.choice(table[-5:])
            row = [p for p in other if p >= 0][:rng.randint(0, n)]
            for p in row:
                shares[p] = shares.get(p, 0) + 1
        for _ in range(n - len(row)):
            row.append(at)
            at += 1
        table.append(row + [-1] * (width - n))
        held.append(n)
        kv.append(n * page)
    P = at + rows + 2
    order = list(range(P))
    rng.shuffle(order)
    table = [[order[p] if p >= 0 else -1 for p in row] for row in table]
    sh = [0] * P
    for p, n in shares.items():
        sh[order[p]] = n
    return table, held, kv, [order[p] for p in range(at, P)], sh, P


@pytest.mark.parametrize("rows,width,page", [(1, 3, 16), (4, 3, 16), (60, 5, 16), (3000, 3, 16), (40, 9, 128), (3, 90000, 16)])
@pytest.mark.parametrize("moving", [True, False])
@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("window,sinks,seed", [(-1, 0, 1), (-1, 0, 2), (20, 5, 3)])
def test_rows_cut_back_into_a_shared_page(rows, width, page, moving, short, window, sinks, seed):
    import pages_ref as ref
    rng = random.Random(seed * 100 + rows)
    table, held, kv, free, shares, P = _holders(rng, rows, width, page)
    num_free = len(free)
    if short:
        num_free = 0                                            # what is on the stack then is what the call itself gives back
    kv = [rng.choice([n, max(0, n - 1), max(0, n - rng.randint(0, 2 * page)), n - n % page // 2 - 1, 0]) for n in kv]
    free += [-9] * (P - len(free))
    d = dict(block_table=_i32(table), num_held=_i32(held), kv_lens=_i32(kv), free_pages=_i32(free), num_free=_i32([num_free]), shares=_i32(shares))
    caches = [torch.randint(0, 256, (P, 2, page, 8), dtype=torch.uint8, device=DEV), torch.randint(0, 256, (P, page, 3, 16), dtype=torch.uint8, device=DEV),
              torch.randint(0, 256, (P, 5), dtype=torch.uint8, device=DEV)]
    want = [c.clone() for c in caches]
    left = _i32([-3])
    freed = _msa().kv_pages_free(**d, window_size=window, num_sink_tokens=sinks, page_size=page, caches=caches if moving else (), num_shared=left)
    num_free, n = ref.free_pages(table, held, kv, free, num_free, shares, window, sinks, page)
    moves, num_free, still = _cut(table, held, kv, free, num_free, shares, page, moving)
    assert freed.item() == n and left.item() == still and d["num_free"].item() == num_free
    assert d["block_table"].tolist() == table and d["num_held"].tolist() == held and d["shares"].tolist() == shares and d["kv_lens"].tolist() == kv
    assert d["free_pages"].tolist() == free
    for a, b, tokens in moves:
        want[0][b, :, :tokens] = want[0][a, :, :tokens]
        want[1][b, :tokens] = want[1][a, :tokens]
        want[2][b] = want[2][a]
    assert all(torch.equal(a, b) for a, b in zip(caches, want))
    if rows == 3000:                                            # the tables have such rows
        assert len(moves) + still > 100


@pytest.mark.parametrize("captured", [False, True])
def test_a_rollback_below_the_fork_leaves_the_other_rows_tokens_alone(captured):
    """Fork, reject tokens of one row back into a page that both hold, append: the other row reads what it read before."""
    msa = _msa()
    P, page, hk, width = 12, 128, 2, 4
    b16 = lambda *s: torch.randn(*s, device=DEV).bfloat16()
    kc, vc = b16(P, hk, page, 128), b16(P, hk, page, 128)
    k0, v0 = kc.clone(), vc.clone()
    table0, held0, kv0 = _i32([[0, 1, 2, -1], [-1] * width]), _i32([3, 0]), _i32([300, 0])
    table, held, kv, free, num_free, shares = table0.clone(), held0.clone(), kv0.clone(), _i32(list(range(P - 1, 2, -1)) + [-1] * 3), _i32([P - 3]), _i32([0] * P)
    left, newk, newv = _i32([7]), b16(3, hk, 128), b16(3, hk, 128)

    def step():
        msa.kv_pages_fork(table, held, kv, _i32_0, _i32_1, free, num_free, shares, [kc, vc])
        kv[:1] -= 100                                           # 200 tokens: inside page 1, which row 1 holds too
        msa.kv_pages_free(table, held, kv, free, num_free, shares, caches=[kc, vc], num_shared=left)
        kv.add_(ql)
        tabs = msa.paged_kv_tables(ql, kv, table, held, free, num_free, max_total_q=3, num_held_out=held, num_free_out=num_free)
        msa.kv_cache_append(newk, newv, kc, vc, tabs["slot_map"])

    _i32_0, _i32_1, ql = _i32([0]), _i32([1]), _i32([3, 0])
    if captured:
        keep = [t.clone() for t in (table, held, kv, free, num_free, shares, kc, vc)]
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for t, was in zip((table, held, kv, free, num_free, shares, kc, vc), keep):
            t.copy_(was)
        graph.replay()
    else:
        step()
    t = table.tolist()
    assert left.item() == 0 and kv.tolist() == [203, 300] and t[1][:2] == [0, 1] and t[0][0] == 0 and t[0][1] not in (0, 1, t[1][2])
    assert shares.tolist() == [1] + [0] * (P - 1)
    for c, was, new in ((kc, k0, newk), (vc, v0, newv)):
        assert torch.equal(c[0], was[0]) and torch.equal(c[1], was[1]) and torch.equal(c[t[1][2]][:, :44], was[2][:, :44])      # row 1's 300 tokens
        assert torch.equal(c[t[0][1]][:, :72], was[1][:, :72]) and torch.equal(c[t[0][1]][:, 72:75], new.transpose(0, 1))


def test_rows_cut_back_needs_shares():
    msa = _msa()
    t = [_i32([[0, 1]]), _i32([2]), _i32([20]), _i32([3, 2]), _i32([2])]
    cache = torch.zeros(4, 1, 16, 8, device=DEV)
    for kw in (dict(caches=[cache]), dict(num_shared=_i32([0]))):
        with pytest.raises(ValueError, match="shares"):
            msa.kv_pages_free(*t, page_size=16, **kw)
    for kw in (dict(caches=[cache[:3]]), dict(num_shared=_i32([0, 0])), dict(num_shared=torch.zeros(1, device=DEV))):
        with pytest.raises(ValueError):
            msa.kv_pages_free(*t, _i32([0] * 4), page_size=16, **kw)
    assert t[0].tolist() == [[0, 1]] and t[2].tolist() == [20]


def test_forks_copy_whole_pages_where_the_tokens_could_be_either_dimension():
    P, page = 6, 16
    both = torch.randint(0, 256, (P, page, page, 8), dtype=torch.uint8, device=DEV)              # heads or tokens
    last = torch.randint(0, 256, (P, 3, page, page), dtype=torch.uint8, device=DEV)              # tokens last: given as a view
    want = [both.clone(), last.clone()]
    table, free = _i32([[2], [-1]]), _i32([4])
    _msa().kv_pages_fork(table, _i32([1, 0]), _i32([5, 0]), _i32([0]), _i32([1]), free, _i32([1]), _i32([0] * P), [both, last.flatten(1)], page)
    for t, w in zip((both, last), want):
        w[4] = w[2]
        assert torch.equal(t, w)
    assert table.tolist() == [[2], [4]]


@pytest.mark.parametrize("rows,width,seed", [(2, 3, 1), (5, 6, 2), (5, 3, 3), (20, 3, 4), (20, 6, 5), (20, 6, 6)])
def test_requests_keep_their_tokens(rows, width, seed):
    """Requests that grow, fork, are cut back anywhere, end and move: each reads its own tokens throughout, and no page is lost or held twice."""
    msa, rng, page, P = _msa(), random.Random(seed), 16, rows * width + 4
    table, held, kv = torch.full((rows, width), -1, dtype=torch.int32, device=DEV), _i32([0] * rows), _i32([0] * rows)
    free, num_free, shares, left = _i32(rng.sample(range(P), P)), _i32([P]), _i32([0] * P), _i32([0])
    cache = torch.zeros(P, 1, page, 1, dtype=torch.int32, device=DEV)          # a number for each token
    tokens, last = [[] for _ in range(rows)], 0
    for _ in range(60):
        op = rng.choice(["grow", "grow", "fork", "cut", "end", "compact"])
        if op == "grow":
            ql = [min(rng.randint(0, 20), width * page - len(t)) if t or rng.random() < 0.5 else 0 for t in tokens]
            if sum(-(-(len(t) + q) // page) - -(-len(t) // page) for t, q in zip(tokens, ql)) > num_free.item():
                continue
            kv += _i32(ql)
            slots = msa.paged_kv_tables(_i32(ql), kv, table, held, free, num_free, max_total_q=max(1, sum(ql)), page_size=page, num_held_out=held,
                                        num_free_out=num_free)["slot_map"][:sum(ql)]
            cache.view(-1)[slots.long()] = torch.arange(last, last + sum(ql), dtype=torch.int32, device=DEV)
            for t, q in zip(tokens, ql):
                t += range(last, last + q)
                last += q
        elif op == "fork":
            empty, full = [b for b in range(rows) if not tokens[b]], [b for b in range(rows) if tokens[b]]
            if not empty or not full:
                continue
            children = rng.sample(empty, rng.randint(1, len(empty)))
            parents = [rng.choice(full) for _ in children]
            if sum(len(tokens[p]) % page > 0 for p in parents) > num_free.item():
                continue
            at = rng.randint(0, len(children))
            entries = children[:at] + [rng.randrange(rows)] + children[at:], parents[:at] + [-1] + parents[at:]      # one that does nothing
            assert msa.kv_pages_fork(table, held, kv, _i32(entries[1]), _i32(entries[0]), free, num_free, shares, cache, page).item() == 0
            for p, c in zip(parents, children):
                tokens[c] = list(tokens[p])
        elif op == "compact":
            msa.kv_pages_compact(table, held, free, num_free, cache, shares)
        else:
            tokens = [t if rng.random() < 0.4 else t[:0 if op == "end" else rng.randint(0, len(t))] for t in tokens]
            kv.copy_(_i32([len(t) for t in tokens]))
            msa.kv_pages_free(table, held, kv, free, num_free, shares, page_size=page, caches=cache, num_shared=left)
            assert left.item() == 0                             # (the pool has a page for every entry of the table)
        rows_of, used, data, holders = table.tolist(), held.tolist(), cache.view(P, page).tolist(), {}
        for b, t in enumerate(tokens):
            pages = rows_of[b][:used[b]]
            assert len(pages) == -(-len(t) // page) and [x for p in pages for x in data[p]][:len(t)] == t, op
            for p in pages:
                holders[p] = holders.get(p, 0) + 1
            assert len(t) % page == 0 or shares[pages[-1]].item() == 0, op
        stack = free.tolist()[:num_free.item()]
        assert sorted(stack + list(holders)) == list(range(P)) and shares.tolist() == [holders.get(p, 1) - 1 for p in range(P)], op
