"""Pages of a cache (copy, fork, free, compact) against loops over the tables."""
import random

import pytest
import torch

import pages_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _msa():
    import msa_for_sail
    return msa_for_sail


def _ok():
    from msa_for_sail import api
    torch.cuda.synchronize()
    assert api.last_status() == 0


def _bytes(seed, *shape, dtype=torch.uint8):
    g = torch.Generator(device=DEV).manual_seed(seed)
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * size), dtype=torch.uint8, device=DEV, generator=g).view(dtype)


def _raw(t):
    """Bytes of a tensor of any strides."""
    return t.contiguous().view(torch.uint8)


KINDS = ["hnd", "nhd", "e4m3", "kv4", "sliced", "interleaved", "scales", "odd", "nhd_heads", "vector"]


def _cache(kind, P, seed=0, page=128):
    b = torch.bfloat16
    return {
        "hnd": lambda: _bytes(seed, P, 3, page, 128, dtype=b),
        "nhd": lambda: _bytes(seed, P, page, 3, 128, dtype=b),
        "e4m3": lambda: _bytes(seed, P, 2, page, 128, dtype=torch.float8_e4m3fn),
        "kv4": lambda: _bytes(seed, P, 2, 128, 72),
        "sliced": lambda: _bytes(seed, P, 5, page, 128, dtype=b)[:, 1:3],
        "interleaved": lambda: _bytes(seed, P, 2, 2, page, 128, dtype=b)[:, 1],
        "scales": lambda: _bytes(seed, P, 3, 4, dtype=torch.float32),
        "odd": lambda: _bytes(seed, P, 37),
        "nhd_heads": lambda: _bytes(seed, P, page, 5, 128, dtype=b)[:, :, 2:4],
        "vector": lambda: _bytes(seed, P, 1, dtype=torch.float32)[:, 0],
    }[kind]()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [0, 1, 5, 40])
def test_copy(kind, n):
    P = 97
    c = _cache(kind, P, n)
    order = random.Random(n).sample(range(P), 2 * n)
    src, dst = order[:n], order[n:]
    if n >= 5:
        src[1], dst[2], src[3], dst[4] = -1, -5, P, P + 1000    # no page, on either side
    want = c.clone()
    for a, b in zip(src, dst):
        if 0 <= a < P and 0 <= b < P:
            want[b] = c[a]
    _msa().kv_pages_copy(c, _i32(src), _i32(dst))
    _ok()
    assert torch.equal(_raw(c), _raw(want))


def test_copy_of_many_caches_at_once():
    P = 23
    caches = [_cache(KINDS[i % len(KINDS)], P, i) for i in range(150)]
    want = [c.clone() for c in caches]
    for w in want:
        w[3], w[0] = w[5].clone(), w[22].clone()
    _msa().kv_pages_copy(caches, _i32([5, 22]), _i32([3, 0]))
    _ok()
    assert all(torch.equal(_raw(a), _raw(b)) for a, b in zip(caches, want))


def test_copy_past_four_gigabytes():
    """Offsets of 64 bits: pages at both ends of a cache of 5 GB."""
    P, page = 40, 1 << 27
    c = torch.empty(P, page, dtype=torch.uint8, device=DEV)
    c[P - 1] = _bytes(1, page)
    c[2] = _bytes(2, page)
    _msa().kv_pages_copy(c, _i32([P - 1, 2]), _i32([0, P - 2]))
    _ok()
    assert torch.equal(c[0], c[P - 1]) and torch.equal(c[P - 2], c[2])


def _pool(rng, rows, width, page_size, spare=7, kids=0, sharing=True, longest=None):
    """Tables of a pool in use: (table, held, kv, free, shares, P)."""
    longest = width * page_size if longest is None else longest
    kv = [rng.choice([0, 1, page_size, page_size + 1, longest, rng.randint(0, longest)]) for _ in range(rows)]
    kv = [min(n, longest) for n in kv]
    need = [-(-n // page_size) for n in kv]
    P = sum(need) + kids + spare
    order = rng.sample(range(P), P)
    table, held, shares, at = [], [], [0] * P, 0
    for b in range(rows):
        row = []
        if sharing and b and rng.random() < 0.5:
            row = [p for p in table[rng.randrange(b)][:rng.randint(0, need[b])]][:need[b]]
            row = row[:row.index(-1)] if -1 in row else row
            for p in row:
                shares[p] += 1
        more = order[at:at + need[b] - len(row)]
        at += len(more)
        row += more
        table.append(row + [-1] * (width - need[b]))
        held.append(need[b])
    table += [[-1] * width for _ in range(kids)]
    held += [0] * kids
    kv += [0] * kids
    return table, held, kv, order[at:] + [-9] * at, P - at, shares, P


@pytest.mark.parametrize("rows,kids,width,page_size", [(1, 1, 1, 128), (3, 5, 9, 128), (40, 200, 5, 16), (7, 3000, 4, 64), (2, 3, 3000, 128), (5, 9, 40, 1)])
@pytest.mark.parametrize("short", [False, True])
def test_fork(rows, kids, width, page_size, short):
    rng = random.Random(rows * kids + width + short)
    table, held, kv, free, num_free, shares, P = _pool(rng, rows, width, page_size, kids=kids)
    parents = [rng.randrange(rows) for _ in range(kids)]
    children = list(range(rows, rows + kids))
    if short:
        num_free = min(num_free, kids // 2)
    if kids >= 5:                                               # entries that are not made, or not meant
        parents[1], children[2] = -1, -1
        parents[3] = rows + kids + 3
        children[4] = children[0]
    if kids >= 9:
        children[5], parents[6], children[7] = 0, children[6], rows + kids
        parents[8] = children[0]                                # a parent that is a child in the same call had nothing
    pad = 3
    t = torch.full((rows + kids, width + pad), -77, dtype=torch.int32, device=DEV)
    t[:, :width] = _i32(table)
    d = dict(held=_i32(held), kv=_i32(kv), free=_i32(free), num_free=_i32([num_free]), shares=_i32(shares))
    kinds = KINDS if page_size == 128 else ["hnd", "nhd", "e4m3", "sliced", "nhd_heads", "odd"]
    caches = [_cache(k, P, i, page_size) for i, k in enumerate(kinds)] if P < 3500 else []
    before = [c.clone() for c in caches]
    missing = _msa().kv_pages_fork(t[:, :width], d["held"], d["kv"], _i32(parents), _i32(children), d["free"], d["num_free"], d["shares"], caches, page_size)
    _ok()
    moves, left, missed = ref.fork(table, held, kv, parents, children, free, num_free, shares, page_size)
    assert t[:, :width].tolist() == table and (t[:, width:] == -77).all()
    assert d["held"].tolist() == held and d["kv"].tolist() == kv and d["shares"].tolist() == shares
    assert d["num_free"].tolist() == [left] and missing.tolist() == [missed] and d["free"].tolist() == free
    for kind, c, want in zip(kinds, caches, before):
        for a, b, n in moves:
            if kind in ("hnd", "e4m3", "sliced", "interleaved"):
                want[b, :, :n] = want[a, :, :n].clone()
            elif kind in ("nhd", "nhd_heads"):
                want[b, :n] = want[a, :n].clone()
            elif kind == "kv4":
                f = want.flatten(2)
                for lo, size in ((0, 64), (128 * 64, 8)):
                    f[b, :, lo:lo + n * size] = f[a, :, lo:lo + n * size].clone()
            else:
                want[b] = want[a].clone()
        assert torch.equal(_raw(c), _raw(want)), kind


def test_fork_of_requests_whose_pages_behind_the_window_are_gone():
    table = [[-1, -1, 4, 2, -1], [-1] * 5, [-1] * 5]
    d = [_i32(table), _i32([4, 0, 0]), _i32([500, 0, 0])]
    shares = torch.zeros(9, dtype=torch.int32, device=DEV)
    free, num_free = _i32([8, 7, 6]), _i32([3])
    missing = _msa().kv_pages_fork(*d, _i32([0, 0]), _i32([1, 2]), free, num_free, shares)
    assert d[0].tolist() == [[-1, -1, 4, 2, -1], [-1, -1, 4, 6, -1], [-1, -1, 4, 7, -1]]
    assert shares.tolist() == [0, 0, 0, 0, 2, 0, 0, 0, 0] and num_free.tolist() == [1] and missing.tolist() == [0]
    assert d[1].tolist() == [4, 4, 4] and d[2].tolist() == [500] * 3
    # a parent whose last page is gone: the child has none either
    d = [_i32([[3, -1], [-1, -1]]), _i32([2, 0]), _i32([200, 0])]
    num_free = _i32([3])
    _msa().kv_pages_fork(*d, _i32([0]), _i32([1]), free, num_free, shares)
    assert d[0].tolist() == [[3, -1], [3, -1]] and num_free.tolist() == [3] and d[1].tolist() == [2, 2]


@pytest.mark.parametrize("rows,width,page_size", [(1, 1, 128), (5, 9, 128), (100, 60, 16), (300, 70, 128), (3, 9000, 16), (20, 1025, 4), (2000, 17, 128), (0, 4, 128)])
@pytest.mark.parametrize("window,sinks", [(-1, 0), (1, 0), (300, 4), (1000, 200), (5, 1 << 30)])
@pytest.mark.parametrize("sharing", [True, False])
def test_free(rows, width, page_size, window, sinks, sharing):
    rng = random.Random(rows + width + window + sinks)
    table, held, kv, free, num_free, shares, P = _pool(rng, rows, width, page_size, sharing=sharing)
    now = [rng.choice([0, n, n, max(0, n - 3), rng.randint(0, n), n + 5]) for n in kv]
    if rows > 4:
        now[2] = -4
        for c in range(0, min(width, held[1]), 3):              # entries given back before
            if table[1][c] >= 0:
                p, table[1][c] = table[1][c], -1
                if sharing:
                    shares[p] = max(0, shares[p] - 1)
    t = torch.full((rows, width + 2), -77, dtype=torch.int32, device=DEV)
    t[:, :width] = _i32(table).view(rows, width)
    d = dict(held=_i32(held), kv=_i32(now), free=_i32(free), num_free=_i32([num_free]), shares=_i32(shares) if sharing else None)
    freed = _msa().kv_pages_free(t[:, :width], d["held"], d["kv"], d["free"], d["num_free"], d["shares"], window_size=window, num_sink_tokens=sinks,
                                 page_size=page_size)
    _ok()
    left, count = ref.free_pages(table, held, now, free, num_free, shares if sharing else None, window, sinks, page_size)
    assert t[:, :width].tolist() == table and (t[:, width:] == -77).all()
    assert d["held"].tolist() == held and d["num_free"].tolist() == [left] and freed.tolist() == [count] and d["free"].tolist() == free
    if sharing:
        assert d["shares"].tolist() == shares


def test_free_keeps_what_a_windowed_query_sees():
    """The next query stands at kv_len and sees the keys from kv_len - window + 1 on, its own among them."""
    for n in range(1, 700, 13):
        for window, sinks in ((1, 0), (128, 4), (129, 128), (200, 130)):
            t, held, num_free = _i32([[0, 1, 2, 3, 4, 5]]), _i32([-(-n // 128)]), _i32([0])
            free = torch.zeros(6, dtype=torch.int32, device=DEV)
            _msa().kv_pages_free(t, held, _i32([n]), free, num_free, window_size=window, num_sink_tokens=sinks)
            pages = -(-n // 128)
            need = {j // 128 for j in range(n + 1) if j > n - window or j < sinks} & set(range(pages))
            assert {i for i, p in enumerate(t.tolist()[0][:pages]) if p >= 0} == need, (n, window, sinks)


@pytest.mark.parametrize("rows,width,spare", [(1, 1, 0), (4, 9, 40), (50, 30, 0), (200, 20, 3000), (3, 2000, 100), (900, 130, 40000), (40, 30, 200000), (1300, 130, 500)])
@pytest.mark.parametrize("sharing", [True, False])
def test_compact(rows, width, spare, sharing):
    rng = random.Random(rows + width)
    table, held, kv, free, num_free, shares, P = _pool(rng, rows, width, 128, spare=spare, sharing=sharing)
    if num_free > 3:                                            # pages that are kept for something else
        num_free -= 2
    kinds = [k for k in KINDS] if P < 3000 else ["vector", "odd"]
    caches = [_cache(k, P, i) for i, k in enumerate(kinds)]
    before = [c.clone() for c in caches]
    d = dict(t=_i32(table), held=_i32(held), free=_i32(free), num_free=_i32([num_free]), shares=_i32(shares) if sharing else None)
    r = _msa().kv_pages_compact(d["t"], d["held"], d["free"], d["num_free"], caches, d["shares"])
    _ok()
    moves, left = ref.compact(table, held, free, num_free, shares if sharing else None, P)
    n = len(moves)
    assert r.num_moved.tolist() == [n]
    assert list(zip(r.src.tolist(), r.dst.tolist())) == moves + [(-1, -1)] * (P - n)
    assert d["t"].tolist() == table and d["num_free"].tolist() == [left] and d["free"].tolist() == free
    if sharing:
        assert d["shares"].tolist() == shares
    for c, want in zip(caches, before):
        for a, b in moves:
            want[b] = want[a].clone()
        assert torch.equal(_raw(c), _raw(want))


def test_compact_twice_moves_nothing_and_numbers_that_are_no_pages_stay():
    t, held = _i32([[7, -1, 5, 900, 3]]), _i32([4])
    free, num_free = _i32([6, 1, 1, -3, 0, 77]), _i32([5])
    r = _msa().kv_pages_compact(t, held, free, num_free, num_pages=8)
    assert t.tolist() == [[1, -1, 0, 900, 3]] and r.num_moved.tolist() == [2]
    assert r.src.tolist()[:3] == [5, 7, -1] and r.dst.tolist()[:3] == [0, 1, -1]
    assert num_free.tolist() == [3] and free.tolist()[:3] == [7, 6, 5]
    r = _msa().kv_pages_compact(t, held, free, num_free, num_pages=8)
    assert t.tolist() == [[1, -1, 0, 900, 3]] and r.num_moved.tolist() == [0] and free.tolist()[:3] == [7, 6, 5]


def test_an_empty_pool():
    t, held, free, num_free = torch.zeros(0, 4, dtype=torch.int32, device=DEV), _i32([]), _i32([]), _i32([0])
    m = _msa()
    m.kv_pages_free(t, held, held, free, num_free)
    m.kv_pages_fork(t, held, held.clone(), _i32([]), _i32([]), free, num_free, _i32([]))
    r = m.kv_pages_compact(t, held, free, num_free, num_pages=0)
    m.kv_pages_copy(torch.zeros(0, 5, device=DEV), _i32([]), _i32([]))
    m.kv_pages_copy([], _i32([0]), _i32([1]))
    _ok()
    assert r.num_moved.tolist() == [0] and num_free.tolist() == [0]
    # a stack whose count is nonsense stays in bounds
    t, held, free, num_free = _i32([[0, 1]]), _i32([2]), _i32([5, 4]), _i32([1000])
    m.kv_pages_free(t, held, _i32([0]), free, num_free)
    _ok()
    assert num_free.tolist() == [2] and free.tolist() == [5, 4] and t.tolist() == [[-1, -1]]


def test_a_captured_beam_step():
    """Free what ended, fork what goes on, page tables of the next token, compact: captured once, replayed on changing lists."""
    m = _msa()
    rng = random.Random(3)
    B, width, ps, P = 12, 6, 128, 60
    table, held, kv, free, num_free, shares = [[-1] * width for _ in range(B)], [0] * B, [0] * B, list(range(P - 1, -1, -1)), P, [0] * P
    d = dict(t=_i32(table), held=_i32(held), kv=_i32(kv), free=_i32(free), num_free=_i32([num_free]), shares=_i32(shares), ql=_i32([0] * B),
             par=_i32([-1] * 4), kid=_i32([-1] * 4))
    cache = _cache("hnd", P, 1)

    def step():
        m.kv_pages_free(d["t"], d["held"], d["kv"], d["free"], d["num_free"], d["shares"], window_size=300, num_sink_tokens=10)
        m.kv_pages_fork(d["t"], d["held"], d["kv"], d["par"], d["kid"], d["free"], d["num_free"], d["shares"], cache)
        d["kv"].add_(d["ql"])
        m.paged_kv_tables(d["ql"], d["kv"], d["t"], d["held"], d["free"], d["num_free"], max_total_q=B, num_held_out=d["held"], num_free_out=d["num_free"])
        m.kv_pages_compact(d["t"], d["held"], d["free"], d["num_free"], cache, d["shares"])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    for it in range(25):
        kv = [0 if rng.random() < 0.15 else n for n in kv]
        ql = [rng.choice([1, 1, 40]) if n or rng.random() < 0.2 else 0 for n in kv]
        live = [b for b in range(B) if kv[b]]
        dead = [b for b in range(B) if not kv[b] and not ql[b]]
        pairs = [(rng.choice(live), c) for c in dead[:4]] if live else []
        pairs += [(-1, -1)] * (4 - len(pairs))
        # tokens that would outgrow the row are not asked for
        ql = [n if kv[b] + n <= width * ps else 0 for b, n in enumerate(ql)]
        d["kv"].copy_(_i32(kv)), d["ql"].copy_(_i32(ql)), d["par"].copy_(_i32([p for p, _ in pairs])), d["kid"].copy_(_i32([c for _, c in pairs]))
        graph.replay()
        num_free, _ = ref.free_pages(table, held, kv, free, num_free, shares, 300, 10, ps)
        _, num_free, missing = ref.fork(table, held, kv, *zip(*pairs), free, num_free, shares, ps)
        assert missing == 0
        kv = [n + q for n, q in zip(kv, ql)]
        for b in range(B):
            while held[b] < -(-kv[b] // ps):
                num_free -= 1
                table[b][held[b]] = free[num_free]
                held[b] += 1
        _, num_free = ref.compact(table, held, free, num_free, shares, P)
        assert d["t"].tolist() == table and d["held"].tolist() == held and d["num_free"].tolist() == [num_free] and d["shares"].tolist() == shares
        assert d["free"].tolist()[:num_free] == free[:num_free]
        # every page is held as often as its shares say, or free
        count = [0] * P
        for row, n in zip(table, held):
            for p in row[:n]:
                if p >= 0:
                    count[p] += 1
        assert all((c - 1 if c else 0) == s for c, s in zip(count, shares))
        assert sorted(free[:num_free]) == [p for p in range(P) if not count[p]]
    _ok()


def test_refused_calls():
    m = _msa()
    P, B, width = 8, 2, 4
    t, held, kv, free, num_free, shares = torch.zeros(B, width, dtype=torch.int32, device=DEV), _i32([2, 1]), _i32([200, 100]), _i32([7] * 8), _i32([5]), _i32([0] * P)
    cache = _cache("hnd", P)
    one = _i32([0])
    other = torch.zeros(8, P, 4, 4, device=DEV).transpose(0, 1)[:, ::2, ::3, ::2]         # no even steps
    bad = [
        lambda: m.kv_pages_copy(cache, one, _i32([0, 1])), lambda: m.kv_pages_copy(cache, one.long(), one), lambda: m.kv_pages_copy(cache, one.cpu(), one),
        lambda: m.kv_pages_copy([cache, cache[:4]], one, one), lambda: m.kv_pages_copy([cache, cache.cpu()], one, one), lambda: m.kv_pages_copy(other, one, one),
        lambda: m.kv_pages_copy(cache[:1].expand(P, -1, -1, -1), one, one), lambda: m.kv_pages_copy(cache, one[0], one),
        lambda: m.kv_pages_fork(t, held, kv, one, _i32([0, 1]), free, num_free, shares), lambda: m.kv_pages_fork(t, held[:1], kv, one, one, free, num_free, shares),
        lambda: m.kv_pages_fork(t, held, kv.long(), one, one, free, num_free, shares), lambda: m.kv_pages_fork(t, held, kv, one, one, free, held, shares),
        lambda: m.kv_pages_fork(t, held, kv, one, one, free, num_free, shares[:4], cache), lambda: m.kv_pages_fork(t, held, kv, one, one, free, num_free, shares, page_size=0),
        lambda: m.kv_pages_fork(t.T, held, kv, one, one, free, num_free, shares), lambda: m.kv_pages_fork(t[:1].expand(2, -1), held, kv, one, one, free, num_free, shares),
        lambda: m.kv_pages_fork(t.long(), held, kv, one, one, free, num_free, shares),
        lambda: m.kv_pages_free(t, held, kv, free, num_free, window_size=0), lambda: m.kv_pages_free(t, held, kv, free, num_free, window_size=-3),
        lambda: m.kv_pages_free(t, held, kv, free, num_free, window_size=3, num_sink_tokens=-1), lambda: m.kv_pages_free(t, held, kv, free.cpu(), num_free),
        lambda: m.kv_pages_free(t, held, kv, free, num_free, shares.float()), lambda: m.kv_pages_free(t, held, kv, free, num_free, page_size=1 << 31),
        lambda: m.kv_pages_free(t[0], held, kv, free, num_free),
        lambda: m.kv_pages_compact(t, held, free, num_free), lambda: m.kv_pages_compact(t, held, free, num_free, num_pages=-1),
        lambda: m.kv_pages_compact(t, held, free, num_free, cache, shares[:4]), lambda: m.kv_pages_compact(t, held, free, num_free, cache, num_pages=4),
        lambda: m.kv_pages_compact(t, held, free, num_free, shares=shares, num_pages=9)]
    before = [x.clone() for x in (t, held, kv, free, num_free, shares, cache.view(torch.int16))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")
    _ok()
    for x, y in zip(before, (t, held, kv, free, num_free, shares, cache.view(torch.int16))):
        assert torch.equal(x, y)


def test_two_streams():
    """Two pools on two streams at once; workspaces are each call's own."""
    m = _msa()
    P = 3000
    streams, pools = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        table = torch.randperm(P, generator=torch.Generator().manual_seed(i))[:2000].view(20, 100).int().to(DEV)
        rest = torch.tensor(sorted(set(range(P)) - set(table.flatten().tolist())), dtype=torch.int32, device=DEV)
        free = torch.cat([rest, torch.zeros(2000, dtype=torch.int32, device=DEV)])
        cache = _cache("e4m3", P, i, 16)
        pools.append((table, _i32([100] * 20), free, _i32([P - 2000]), cache, cache[table.flatten().long()].clone()))
    torch.cuda.synchronize()
    for r in range(3):
        for s, (t, held, free, num_free, cache, _) in zip(streams, pools):
            with torch.cuda.stream(s):
                m.kv_pages_compact(t, held, free, num_free, cache)
    _ok()
    for t, held, free, num_free, cache, was in pools:
        assert sorted(t.flatten().tolist()) == list(range(2000)) and num_free.item() == P - 2000
        assert torch.equal(_raw(cache[t.flatten().long()]), _raw(was)) and sorted(free[:1000].tolist()) == list(range(2000, P))
