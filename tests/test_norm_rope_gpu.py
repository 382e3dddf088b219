"""qk_norm_rope, kv_cache_append and kv4_read against 64-bit forms."""
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(seed, T, hq, hk, spread=2.0):
    """q, k, v side by side in one buffer, as a projection leaves them."""
    g = _gen(seed)
    x = torch.randn(T, hq + 2 * hk, 128, generator=g) * (torch.rand(T, hq + 2 * hk, 1, generator=g) * spread + 0.1)
    x = x.to(torch.bfloat16).to(DEV)
    return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], g


def _check_bf16(got, want, size, what):
    """Half a step of bf16, and 2^-19 of the magnitudes in between (a sum of 128 squares, an inverse root, three products, a sum: under 32
    roundings of 2^-24)."""
    got = got.double().cpu()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -18 * size
    assert ((got - want).abs() <= tol).all(), f"{what}: {((got - want).abs() / tol).max():.3g} of the tolerance"


def _positions(g, axes, T, far=3_000_000):
    return torch.randint(0, far, (axes, T), generator=g)


SECTIONS = {1: lambda n: [n], 2: lambda n: [n // 4, n - n // 4], 3: lambda n: [n - 2 * (n // 3), n // 3, n // 3], 4: lambda n: [0, 1, n - 3, 2]}


@pytest.mark.parametrize("T,hq,hk", [(1, 1, 1), (1, 64, 8), (3, 5, 2), (2, 16, 1), (70, 12, 3), (5, 33, 4), (2500, 8, 4)])
@pytest.mark.parametrize("rotary,interleaved,axes", [(128, False, 1), (64, False, 3), (32, True, 2), (96, False, 4), (128, True, 1), (0, False, 1)])
def test_norm_and_rotation(T, hq, hk, rotary, interleaved, axes):
    import msa_for_sail as msa
    q, k, _, g = _inputs(T * 7 + hq, T, hq, hk)
    wq, wk = torch.rand(128, generator=g) + 0.5, torch.rand(hk, 128, generator=g) - 0.5
    if hq % 2:
        wq = (torch.rand(hq, 128, generator=g) + 0.5)
        wk = wk[0].clone()
    inv = [1e6 ** (-i / max(1, rotary // 2)) for i in range(rotary // 2)]
    sections = SECTIONS[axes](rotary // 2)
    pos = _positions(g, axes, T)
    rope = msa.rope_plan(rotary, inv_freq=inv, sections=sections, interleaved=interleaved) if rotary else None
    p = pos.to(DEV) if T % 2 else pos.to(torch.int32).to(DEV)
    qo, ko = msa.qk_norm_rope(q, k, p, rope, q_weight=wq.to(DEV), k_weight=wk.to(DEV), eps=1e-5)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        want, size = ref.norm_rope(x, pos, inv, sections if rotary else [], interleaved, w, eps=1e-5)
        _check_bf16(got, want, size, f"{T} {hq}/{hk} rotary {rotary}")


def test_rotation_alone_in_place_and_bf16_weights():
    import msa_for_sail as msa
    q, k, _, g = _inputs(3, 40, 6, 2)
    pos = torch.tensor([0, 1, 2, 2 ** 31 - 1] * 10)
    inv = [10000.0 ** (-2 * i / 128) for i in range(64)]
    rope = msa.rope_plan(128)
    q0, k0 = q.clone(), k.clone()
    qo, ko = msa.qk_norm_rope(q, k, pos.to(DEV), rope, norm=False, q_out=q, k_out=k)
    assert qo is q and ko is k
    for got, x in ((q, q0), (k, k0)):
        # the angle of position 2^31 - 1 in 64 bits is good to 2^31 x 2^-53: 3e-7
        want, size = ref.norm_rope(x, pos[None], inv, [64], False, norm=False)
        _check_bf16(got, want, size, "in place")
    w = (torch.rand(128, generator=g) + 0.5).to(torch.bfloat16)
    qo, _ = msa.qk_norm_rope(q0, k0, None, None, q_weight=w.to(DEV))
    want, size = ref.norm_rope(q0, None, [], [], False, w)
    _check_bf16(qo, want, size, "bf16 weight")
    # weights of one only; zeros; no tokens
    z = torch.zeros_like(q0)
    qo, ko = msa.qk_norm_rope(z, k0, None, None, k_weight=w.to(DEV))
    assert (qo == 0).all()
    want, size = ref.norm_rope(k0, None, [], [], False, w)
    _check_bf16(ko, want, size, "bf16 weight of k")
    qo, ko = msa.qk_norm_rope(q0[:0], k0[:0], pos.to(DEV)[:0], rope)
    assert qo.shape[0] == ko.shape[0] == 0


def test_negative_positions_turn_the_other_way():
    import msa_for_sail as msa
    q, k, _, _ = _inputs(4, 9, 2, 1)
    pos = torch.arange(9) * -1000
    inv = [10000.0 ** (-2 * i / 64) for i in range(32)]
    qo, ko = msa.qk_norm_rope(q, k, pos.to(DEV), msa.rope_plan(64))
    want, size = ref.norm_rope(q, pos[None], inv, [32], False)
    _check_bf16(qo, want, size, "negative")


def _cache(kind, P, hk, nhd=False, gap=False):
    shape = (P, hk, 128, 72) if kind == "kv4" else (P, 128, hk, 128) if nhd else (P, hk, 128, 128)
    dt = {"kv4": torch.uint8, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}[kind]
    both = torch.full((P, 2) + shape[1:], 0x55, dtype=torch.uint8 if kind != "bf16" else torch.int16, device=DEV)
    both = both if kind == "kv4" else both.view(dt)
    if gap:                                                     # keys and values of a page side by side
        return both[:, 0], both[:, 1]
    return both[:, 0].contiguous(), both[:, 1].contiguous()


def _rows(cache, slots, kind, nhd):
    c = cache.cpu()
    s = slots.long()
    if kind == "kv4":
        a, b = ref.kv4_parts(cache)
        return a[s // 128, :, s % 128], b[s // 128, :, s % 128]
    return c[s // 128, s % 128] if nhd else c[s // 128, :, s % 128]


@pytest.mark.parametrize("kind,nhd,gap", [("bf16", False, False), ("bf16", True, True), ("e4m3", False, True), ("e4m3", True, False), ("kv4", False, False),
                                          ("kv4", False, True)])
@pytest.mark.parametrize("T,hq,hk,rotary,interleaved", [(1, 8, 1, 64, False), (37, 5, 3, 128, False), (300, 16, 4, 32, True), (64, 4, 2, 96, False), (1, 64, 8, 0, False)])
@pytest.mark.parametrize("two", [True, False])
def test_written_rows(kind, nhd, gap, T, hq, hk, rotary, interleaved, two):
    """Rows of the cache: keys normed, rotated and rounded to bf16, then to the cache's type; everything else left as it was."""
    import msa_for_sail as msa
    q, k, v, g = _inputs(T + hq, T, hq, hk)
    P = -(-T // 128) + 2
    kc, vc = _cache(kind, P, hk, nhd, gap)
    kc0, vc0 = kc.clone(), vc.clone()
    slots = torch.randperm(P * 128, generator=g)[:T].to(torch.int32)
    if T > 5:
        slots[2], slots[4] = -1, P * 128 + 3                    # padding, and a slot past the cache: nothing is written
    real = (slots >= 0) & (slots < P * 128)
    inv = [1e4 ** (-i / max(1, rotary // 2)) for i in range(rotary // 2)]
    rope = msa.rope_plan(rotary, inv_freq=inv, interleaved=interleaved) if rotary else None
    pos = _positions(g, 1, T)
    ks = vs = None
    if kind != "bf16":
        ks, vs = (0.25, 0.03125) if two else ([0.3, 0.0123], 0.7)
        ks, vs = (torch.tensor((x * hk)[:hk] if isinstance(x, list) else [x] * hk) for x in (ks, vs))
    k_out = torch.empty(T, hk, 128, dtype=torch.bfloat16, device=DEV) if two else None
    scales = {} if ks is None else dict(k_scale=ks.to(DEV), v_scale=float(vs[0]))
    _, ko = msa.qk_norm_rope(q, k, pos.to(DEV), rope, v=v, k_cache=kc, v_cache=vc, slot_map=slots.to(DEV), k_out=k_out, **scales)
    assert ko is k_out
    torch.cuda.synchronize()
    want, size = ref.norm_rope(k, pos, inv, [rotary // 2] if rotary else [], interleaved)
    at = slots[real]
    if kind == "bf16":
        _check_bf16(_rows(kc, at, kind, nhd), want[real], size[real], "keys")
        assert torch.equal(_rows(vc, at, kind, nhd), v.cpu()[real])
    else:
        kb, vb = want.float().to(torch.bfloat16)[real], v.cpu()[real]
        if k_out is not None:
            assert torch.equal(k_out.cpu()[real], kb)            # keys that are quantised are computed in 64 bits: the same bf16
        for c, x, s, name in ((kc, kb, ks, "keys"), (vc, vb, vs, "values")):
            if kind == "e4m3":
                y = (x.float() / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                assert torch.equal(_rows(c, at, kind, nhd).view(torch.uint8), y.view(torch.uint8)), name
            else:
                codes, sb = _rows(c, at, kind, nhd)
                want_codes, want_sb = ref.kv4_encode(x, s)
                assert torch.equal(sb, want_sb), name
                assert torch.equal(codes, want_codes), name
    # what was not written is as it was
    for c, c0 in ((kc, kc0), (vc, vc0)):
        if kind == "kv4":
            for a, b in zip(ref.kv4_parts(c), ref.kv4_parts(c0)):
                keep = torch.ones(P, 128, dtype=torch.bool)
                keep[at.long() // 128, at.long() % 128] = False
                assert torch.equal(a.transpose(1, 2)[keep], b.transpose(1, 2)[keep])
        else:
            a, b = (x.cpu().view(torch.uint8 if kind == "e4m3" else torch.int16) for x in (c, c0))
            if not nhd:
                a, b = a.transpose(1, 2), b.transpose(1, 2)
            keep = torch.ones(P, 128, dtype=torch.bool)
            keep[at.long() // 128, at.long() % 128] = False
            assert torch.equal(a[keep], b[keep])


def test_borders_ties_and_special_values_in_4_bits():
    """Ties go to the even code for every scale; zeros, tiny and huge blocks; infinities saturate, a NaN takes its block along."""
    import msa_for_sail as msa
    rows = []
    for m in range(8, 16):                                      # every significand of a scale
        s = m / 8
        edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]) * s
        for sign in (1, -1):
            rows.append(torch.cat([edge * sign, edge.flip(0) * -sign]))
            up = torch.cat([edge, edge]).to(torch.bfloat16).view(torch.int16)
            rows.append(((up + torch.tensor([1, -1] * 8, dtype=torch.int16)).view(torch.bfloat16).float() * sign).clamp(-6 * s, 6 * s))
    x = torch.stack(rows)                                       # 32 blocks of 16
    e = torch.tensor([2.0 ** -16, 2.0 ** -9, 1.0, 2.0 ** 6, 2.0 ** 30]).repeat_interleave(32)[:, None]
    x = (x.repeat(5, 1) * e).reshape(-1, 128)
    inf, nan = float("inf"), float("nan")
    special = torch.zeros(8, 128)
    special[0, 5], special[1, 3], special[2, 17], special[3] = inf, -inf, nan, 0.0
    special[4], special[5, 0], special[6] = 3e38, 1e-38, -0.0
    x = torch.cat([x, special]).to(torch.bfloat16)[:, None]     # [T, 1, 128]
    T = x.shape[0]
    kc, vc = msa.allocate_kv4_cache(-(-T // 128), 1, device=DEV)
    slots = torch.arange(T, dtype=torch.int32)
    for scale in (1.0, 0.5, 0.37):
        msa.kv_cache_append(x.to(DEV), x.to(DEV), kc, vc, slots.to(DEV), k_scale=scale, v_scale=1.0)
        codes, sb = _rows(kc, slots, "kv4", False)
        want, want_sb = ref.kv4_encode(x, torch.tensor([scale]))
        ok = want_sb != 0x7F                                    # the codes of a NaN block mean nothing
        assert torch.equal(sb & 0x7F, want_sb & 0x7F)
        each = ok.repeat_interleave(8, -1)
        assert torch.equal(codes[each], want[each])
        got = msa.kv4_read(kc, slots.to(DEV)).double().cpu()
        want_v = ref.kv4_values(kc)[slots.long() // 128, :, slots.long() % 128]
        assert torch.equal(torch.isnan(got), torch.isnan(want_v)) and torch.isnan(got[-6, 0, 16:32]).all()
        assert torch.equal(got.nan_to_num(7.0), want_v.nan_to_num(7.0))


def test_read_of_padding_and_pages_outside():
    import msa_for_sail as msa
    from msa_for_sail import cache
    g = _gen(5)
    c = ref.random_kv4(g, 7, 3).to(DEV)
    slots = torch.tensor([5, -1, 7 * 128, 130, -100, 7 * 128 - 1], dtype=torch.int32)
    got = msa.kv4_read(c, slots.to(DEV)).double().cpu()
    v = ref.kv4_values(c)
    assert torch.equal(got[0], v[0, :, 5]) and torch.equal(got[3], v[1, :, 2]) and torch.equal(got[5], v[6, :, 127])
    assert (got[[1, 2, 4]] == 0).all()
    pages = torch.tensor([6, -1, 2, 7], dtype=torch.int32, device=DEV)
    got = cache.unpack_pages(c, pages).double().cpu()
    assert torch.equal(got[0], v[6]) and torch.equal(got[2], v[2])
    big = torch.zeros(7, 2, 3, 128, 72, dtype=torch.uint8, device=DEV)
    big[:, 1] = c
    assert torch.equal(msa.kv4_read(big[:, 1], slots.to(DEV)), msa.kv4_read(c, slots.to(DEV)))


def test_e4m3_queries():
    import msa_for_sail as msa
    q, k, _, g = _inputs(8, 50, 7, 1)
    out = torch.empty(50, 7, 128, dtype=torch.float8_e4m3fn, device=DEV)
    qo, _ = msa.qk_norm_rope(q, k, None, None, q_out=out, q_scale=0.02)
    want, size = ref.norm_rope(q, None, [], [], False)
    y = (want / 0.02).clamp(-448, 448)
    # e4m3 rounds by at most 2^-4 of the value or half of its smallest step, bf16 before it by 2^-8
    tol = (2.0 ** -4 + 2.0 ** -8) * y.abs() * 1.01 + 2.0 ** -10 + 2.0 ** -18 * size / 0.02
    assert ((qo.double().cpu() - y).abs() <= tol).all()


def test_capture_and_another_stream():
    import msa_for_sail as msa
    q, k, v, g = _inputs(9, 6, 8, 2)
    rope = msa.rope_plan(128)
    pos, slots = torch.arange(6, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV)
    kc, vc = msa.allocate_kv4_cache(3, 2)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        msa.qk_norm_rope(q, k, pos, rope, v=v, q_out=qo, k_cache=kc, v_cache=vc, slot_map=slots)
    torch.cuda.current_stream().wait_stream(side)
    first, rows = qo.clone(), msa.kv4_read(kc, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        msa.qk_norm_rope(q, k, pos, rope, v=v, q_out=qo, k_cache=kc, v_cache=vc, slot_map=slots)
        r = msa.kv4_read(kc, slots)
    pos += 5
    slots += 7
    graph.replay()
    torch.cuda.synchronize()
    want, size = ref.norm_rope(q, pos.cpu()[None], [1e4 ** (-i / 64) for i in range(64)], [64], False)
    _check_bf16(qo, want, size, "replayed")
    assert not torch.equal(qo, first) and not torch.equal(r, rows)
    assert torch.equal(msa.kv4_read(kc, slots), r)


def test_refusals():
    import msa_for_sail as msa
    q, k, v, _ = _inputs(1, 4, 4, 2)
    pos, rope = torch.arange(4, device=DEV), msa.rope_plan(64)
    kc, vc = msa.allocate_kv4_cache(2, 2)
    sl = torch.arange(4, dtype=torch.int32, device=DEV)
    c = dict(v=v, k_cache=kc, v_cache=vc, slot_map=sl)
    msa.qk_norm_rope(q, k, pos, rope, **c)
    with pytest.raises(RuntimeError):
        msa.qk_norm_rope(q.cpu(), k, pos, rope)
    w = torch.ones(128, device=DEV)
    bad = [lambda: msa.qk_norm_rope(q[..., :64], k, pos, rope), lambda: msa.qk_norm_rope(q.float(), k, pos, rope),
           lambda: msa.qk_norm_rope(q, k[:3], pos, rope), lambda: msa.qk_norm_rope(q, k, pos[:3], rope), lambda: msa.qk_norm_rope(q, k, None, rope),
           lambda: msa.qk_norm_rope(q, k, pos.float(), rope), lambda: msa.qk_norm_rope(q, k, torch.stack([pos, pos]), rope),
           lambda: msa.qk_norm_rope(q, k, pos.cpu(), rope), lambda: msa.qk_norm_rope(q, k.cpu(), pos, rope),
           lambda: msa.qk_norm_rope(q, k, pos, rope, v=v), lambda: msa.qk_norm_rope(q, k, pos, rope, **{**c, "v_cache": None}),
           lambda: msa.qk_norm_rope(q, k, pos, rope, **{**c, "slot_map": None}), lambda: msa.qk_norm_rope(q, k, pos, rope, **{**c, "slot_map": sl.long()}),
           lambda: msa.qk_norm_rope(q, k, pos, rope, **{**c, "slot_map": sl[:3]}), lambda: msa.qk_norm_rope(q, k, pos, rope, page_size=64, **c),
           lambda: msa.qk_norm_rope(q, k, pos, rope, **{**c, "k_cache": kc[:, :1], "v_cache": vc[:, :1]}),
           lambda: msa.qk_norm_rope(q, k, pos, rope, **{**c, "k_cache": kc[:1]}),
           lambda: msa.qk_norm_rope(q, k, pos, rope, k_scale=torch.ones(3, device=DEV), **c),
           lambda: msa.qk_norm_rope(q, k, pos, rope, k_scale=1.0), lambda: msa.qk_norm_rope(q, k, pos, rope, slot_map=sl),
           lambda: msa.qk_norm_rope(q, k, pos, rope, norm=False, q_weight=w), lambda: msa.qk_norm_rope(q, k, pos, rope, q_weight=w[:64]),
           lambda: msa.qk_norm_rope(q, k, pos, rope, q_weight=w, k_weight=w.to(torch.bfloat16)),
           lambda: msa.qk_norm_rope(q, k, pos, rope, q_scale=2.0), lambda: msa.qk_norm_rope(q, k, pos, rope, q_out=q[:3]),
           lambda: msa.qk_norm_rope(q, k, pos, rope, q_out=torch.empty(4, 4, 129, dtype=torch.bfloat16, device=DEV)[..., 1:]),
           lambda: msa.kv4_read(kc.view(2, 2, 9216), sl), lambda: msa.kv4_read(kc, sl.long()), lambda: msa.kv4_read(kc, sl, out=q),
           lambda: msa.kv_cache_append(k, v, kc, vc.to(torch.bfloat16), sl), lambda: msa.kv_cache_append(k, v, kc[:0], vc[:0], sl),
           lambda: msa.allocate_kv4_cache(4, 2, page_size=64)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
    bf = torch.zeros(2, 2, 128, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        msa.kv_cache_append(k, v, bf, bf.clone(), sl, k_scale=0.5)


def test_keys_of_a_bf16_cache_are_rounded_once():
    """Cached keys are computed in 64 bits: they are the nearest bf16 numbers, also where 32 bits would fall on the other side of a border."""
    import msa_for_sail as msa
    T, hk = 900, 4
    q, k, v, g = _inputs(91, T, 4, hk)
    w = torch.rand(128, generator=g) + 0.5
    pos, inv = torch.randint(0, 100_000, (1, T), generator=g), [1e4 ** (-2 * i / 128) for i in range(64)]
    kc, vc = _cache("bf16", 8, hk)
    slots = torch.randperm(1024, generator=g)[:T].to(torch.int32)
    msa.qk_norm_rope(q, k, pos.to(DEV), msa.rope_plan(128), v=v, q_weight=w.to(DEV), k_weight=w.to(DEV), k_cache=kc, v_cache=vc, slot_map=slots.to(DEV))
    want, _ = ref.norm_rope(k, pos, inv, [64], False, w)
    # 64-bit angles of the reference are good to 1e5 x 2^-53: borders that close are left out
    near = (want.float().to(torch.bfloat16).double() - want).abs()
    step = 2.0 ** (torch.floor(torch.log2(want.abs().clamp(min=1e-30))) - 7)
    clear = (near / step - 0.5).abs() > 1e-7
    got = _rows(kc, slots, "bf16", False)
    assert clear.float().mean() > 0.999 and torch.equal(got[clear], want.float().to(torch.bfloat16)[clear])
